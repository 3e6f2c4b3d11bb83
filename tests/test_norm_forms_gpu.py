"""Every form of the norms' kernels, by the sizes and offsets that take it and
the verification hook that says so, through the C entries."""

import ctypes

import pytest
import torch

from layer_checks import check_rows, norm_error
from oracle import layer_ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
DIRECT, RING, LONG = 0, 1, 2
ALIGNED, SHIFTED, LOOSE = 0, 1, 2


@pytest.fixture(scope="module")
def abi():
    from sgl_glm53_ascend_ops import abi as _abi
    return _abi


def rows(T, N, dtype, seed, offset=0, extra=0):
    """Random rows, each `extra` elements apart from the next, the first `offset` elements in."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.zeros(T * (N + extra) + offset, dtype=dtype, device="cuda")
    v = buf[offset:].view(T, N + extra)[:, :N]
    v.copy_(torch.randn(T, N, generator=g, device="cuda"))
    return v


def code(abi, dtype):
    return abi.KDA_DTYPE_FP16 if dtype == torch.float16 else abi.KDA_DTYPE_BF16


def form(abi, hook, args):
    """(kernel, rows, units) on 148 SMs."""
    f = abi.KdaNormForm()
    assert hook(ctypes.byref(args), 148, ctypes.byref(f)) == abi.KDA_OK
    return f.kernel, f.rows, f.units


def rmsnorm(abi, x, w, residual, residual_out, fp8, want_form):
    """(out, scale) of one launch."""
    T, N = x.shape
    out = torch.empty(T, N, dtype=torch.float8_e4m3fn if fp8 else x.dtype, device="cuda")
    scale = torch.empty(T, device="cuda") if fp8 else None
    given = residual is not None
    a = abi.KdaNormArgs(
        x=x.data_ptr(), x_row_stride=x.stride(0), residual=residual.data_ptr() if given else None,
        residual_row_stride=residual.stride(0) if given else 0, residual_out=residual_out.data_ptr() if given else None,
        residual_out_row_stride=residual_out.stride(0) if given else 0, weight=w.data_ptr(),
        out=out.data_ptr(), out_row_stride=N, scale=scale.data_ptr() if fp8 else None, num_tokens=T, hidden=N,
        dtype=code(abi, x.dtype), weight_fp32=int(w.dtype == torch.float32), eps=1e-6)
    assert form(abi, abi.lib().kda_rmsnorm_form, a) == want_form
    assert abi.lib().kda_rmsnorm_launch(ctypes.byref(a), abi.stream_handle()) == abi.KDA_OK
    torch.cuda.synchronize()
    return out, scale


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# T, N, offset and extra of x and of the residual, and the form: each kernel's kinds of rows and units a thread.
FORMS = [(3, 512, 0, 0, 0, 0, (DIRECT, ALIGNED, 1)), (400, 4096, 0, 8, 0, 0, (DIRECT, ALIGNED, 2)),
         (600, 4096, 0, 0, 0, 0, (DIRECT, ALIGNED, 4)), (300, 32768, 0, 0, 0, 0, (DIRECT, ALIGNED, 4)),
         (37, 1001, 0, 0, 0, 0, (DIRECT, SHIFTED, 1)), (1300, 1001, 0, 0, 0, 0, (DIRECT, SHIFTED, 2)),
         (5, 20001, 0, 0, 0, 0, (DIRECT, SHIFTED, 4)), (37, 515, 1, 2, 0, 5, (DIRECT, LOOSE, 1)),
         (900, 2050, 3, 1, 1, 0, (DIRECT, LOOSE, 2)), (5, 20002, 1, 1, 0, 3, (DIRECT, LOOSE, 4)),
         (11000, 200, 0, 0, 0, 8, (RING, ALIGNED, 1)), (11000, 512, 0, 0, 0, 0, (RING, ALIGNED, 2)),
         (4000, 4096, 0, 0, 0, 0, (RING, ALIGNED, 4)), (11000, 520, 0, 8, 8, 0, (RING, ALIGNED, 4)),
         (3, 40960, 0, 0, 0, 0, (LONG, LOOSE, 0)), (3, 40961, 1, 0, 0, 2, (LONG, LOOSE, 0))]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,offset,extra,res_offset,res_extra,kind", FORMS)
def test_rmsnorm_forms(abi, T, N, offset, extra, res_offset, res_extra, kind, dtype, fp8):
    """Both types, with and without a residual, weights of either type, against the definition."""
    x, res = rows(T, N, dtype, 1, offset, extra), rows(T, N, dtype, 2, res_offset, res_extra)
    w = 1 + 0.1 * torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    total = rows(T, N, dtype, 4, res_offset, res_extra)
    for weight in (w, w.to(dtype)):
        out, scale = rmsnorm(abi, x, weight, res, total, fp8, kind)
        y, _ = layer_ref.rmsnorm(x, weight, res)
        check_rows(out, scale, y, dtype, norm_error(N))
        assert torch.equal(total, (x.float() + res.float()).to(dtype))
    out, scale = rmsnorm(abi, x, w, None, None, fp8, kind)
    check_rows(out, scale, layer_ref.rmsnorm(x, w)[0], dtype, norm_error(N))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,offset,extra,res_offset,res_extra,kind", FORMS)
def test_sum_written_over_an_input(abi, T, N, offset, extra, res_offset, res_extra, kind, dtype, fp8):
    """residual_out may be residual or x: the bits of a launch that writes the sum to rows laid out alike elsewhere."""
    x, res = rows(T, N, dtype, 1, offset, extra), rows(T, N, dtype, 2, res_offset, res_extra)
    w = 1 + 0.1 * torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    total = (x.float() + res.float()).to(dtype)
    apart = rows(T, N, dtype, 4, res_offset, res_extra)
    out, scale = rmsnorm(abi, x, w, res, apart, fp8, kind)
    assert torch.equal(apart, total)
    keep = res.clone()
    got, got_scale = rmsnorm(abi, x, w, res, res, fp8, kind)
    assert same(res, total) and same(got, out) and (not fp8 or same(got_scale, scale))
    res.copy_(keep)
    apart = rows(T, N, dtype, 4, offset, extra)
    out, scale = rmsnorm(abi, x, w, res, apart, fp8, kind)
    got, got_scale = rmsnorm(abi, x, w, res, x, fp8, kind)
    assert same(x, total) and same(got, out) and (not fp8 or same(got_scale, scale))


# T, H, D, head stride beyond D, gate offset, and the form.
GATED = [(3, 2, 64, 0, 0, (DIRECT, ALIGNED, 1)), (400, 32, 128, 0, 0, (DIRECT, ALIGNED, 2)), (600, 32, 128, 8, 0, (DIRECT, ALIGNED, 4)),
         (19, 5, 64, 0, 3, (DIRECT, LOOSE, 1)), (400, 33, 128, 3, 0, (DIRECT, LOOSE, 2)), (600, 40, 128, 0, 1, (DIRECT, LOOSE, 4)),
         (11000, 1, 64, 0, 0, (RING, ALIGNED, 1)), (11000, 4, 128, 0, 0, (RING, ALIGNED, 2)), (4000, 32, 128, 0, 0, (RING, ALIGNED, 4)),
         (11000, 16, 64, 0, 8, (RING, ALIGNED, 4)), (2, 300, 128, 0, 0, (LONG, ALIGNED, 0)), (2, 301, 128, 0, 5, (LONG, LOOSE, 0))]


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,D,gap,offset,kind", GATED)
def test_gated_rmsnorm_forms(abi, T, H, D, gap, offset, kind, dtype, fp8, act):
    """Both types, gates and outputs, weights of either type, against the definition."""
    heads = rows(T, H * (D + gap), dtype, 5)
    o = heads.as_strided((T, H, D), (H * (D + gap), D + gap, 1))
    gate = rows(T, H * D, dtype, 6, offset, 0)
    w = 1 + 0.1 * torch.randn(D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    for weight in (w, w.to(dtype)):
        out = torch.empty(T, H * D, dtype=torch.float8_e4m3fn if fp8 else dtype, device="cuda")
        scale = torch.empty(T, device="cuda") if fp8 else None
        a = abi.KdaGatedNormArgs(
            o=o.data_ptr(), gate=gate.data_ptr(), gate_row_stride=gate.stride(0), weight=weight.data_ptr(), out=out.data_ptr(),
            out_row_stride=H * D, scale=scale.data_ptr() if fp8 else None, num_tokens=T, num_heads=H, head_dim=D,
            dtype=code(abi, dtype), weight_fp32=int(weight.dtype == torch.float32),
            activation=abi.KDA_ACT_SILU if act == "silu" else abi.KDA_ACT_SIGMOID, eps=1e-6)
        a.o_stride[0], a.o_stride[1] = o.stride(0), o.stride(1)
        assert form(abi, abi.lib().kda_gated_rmsnorm_form, a) == kind
        assert abi.lib().kda_gated_rmsnorm_launch(ctypes.byref(a), abi.stream_handle()) == abi.KDA_OK
        torch.cuda.synchronize()
        check_rows(out, scale, layer_ref.gated_rmsnorm(o, gate, weight, act=act), dtype, norm_error(D))
