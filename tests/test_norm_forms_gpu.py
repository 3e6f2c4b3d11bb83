"""rmsnorm's forms by their lengths, offsets and row counts, through the C
entry: the sum written over one of its own inputs."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


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


def rmsnorm(abi, x, w, residual, residual_out, fp8):
    """(out, scale) of one launch."""
    T, N = x.shape
    out = torch.empty(T, N, dtype=torch.float8_e4m3fn if fp8 else x.dtype, device="cuda")
    scale = torch.empty(T, device="cuda") if fp8 else None
    a = abi.KdaNormArgs(
        x=x.data_ptr(), x_row_stride=x.stride(0), residual=residual.data_ptr(), residual_row_stride=residual.stride(0),
        residual_out=residual_out.data_ptr(), residual_out_row_stride=residual_out.stride(0), weight=w.data_ptr(),
        out=out.data_ptr(), out_row_stride=N, scale=scale.data_ptr() if fp8 else None, num_tokens=T, hidden=N,
        dtype=abi.KDA_DTYPE_FP16 if x.dtype == torch.float16 else abi.KDA_DTYPE_BF16,
        weight_fp32=int(w.dtype == torch.float32), eps=1e-6)
    assert abi.lib().kda_rmsnorm_launch(ctypes.byref(a), abi.stream_handle()) == abi.KDA_OK
    torch.cuda.synchronize()
    return out, scale


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# Lengths, offsets and row counts of each form: vectors (1, 2 and 4 a thread), rows at odd offsets alike and
# unlike, the ring, and rows read twice.
FORMS = [(3, 512, 0, 0, 0, 0), (600, 4096, 0, 0, 0, 0), (300, 32768, 0, 0, 0, 0), (37, 1001, 0, 0, 0, 0),
         (1200, 1001, 0, 0, 0, 0), (5, 20001, 0, 0, 0, 0), (37, 515, 1, 2, 0, 5), (900, 2050, 3, 1, 1, 0),
         (5, 20002, 1, 1, 0, 3), (4000, 4096, 0, 0, 0, 0), (9000, 520, 0, 8, 8, 0), (3, 40960, 0, 0, 0, 0),
         (3, 40961, 1, 0, 0, 2)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,offset,extra,res_offset,res_extra", FORMS)
def test_sum_written_over_an_input(abi, T, N, offset, extra, res_offset, res_extra, dtype, fp8):
    """residual_out may be residual or x: the bits of a launch that writes the sum to rows laid out alike elsewhere."""
    x, res = rows(T, N, dtype, 1, offset, extra), rows(T, N, dtype, 2, res_offset, res_extra)
    w = 1 + 0.1 * torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    total = (x.float() + res.float()).to(dtype)
    apart = rows(T, N, dtype, 4, res_offset, res_extra)
    out, scale = rmsnorm(abi, x, w, res, apart, fp8)
    assert torch.equal(apart, total)
    keep = res.clone()
    got, got_scale = rmsnorm(abi, x, w, res, res, fp8)
    assert same(res, total) and same(got, out) and (not fp8 or same(got_scale, scale))
    res.copy_(keep)
    apart = rows(T, N, dtype, 4, offset, extra)
    out, scale = rmsnorm(abi, x, w, res, apart, fp8)
    got, got_scale = rmsnorm(abi, x, w, res, x, fp8)
    assert same(x, total) and same(got, out) and (not fp8 or same(got_scale, scale))
