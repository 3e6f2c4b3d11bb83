"""Chains of overlapped launches over the same few buffers, each written by one
kernel right before the next reads it: the bits of the chain with a wait after
every launch."""

import ctypes

import pytest
import torch

from linear_abi import linear_args

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def abi():
    from sgl_glm53_ascend_ops import abi as _abi
    return _abi


@pytest.mark.parametrize("T", [1, 40, 700, 4000])
def test_chain_over_shared_buffers(abi, T):
    """norm (sum over its residual) -> projection -> gated norm -> projection (over its residual), 12 times around: every
    tensor, the norms' weights, the bias and the gate among them, is written while the kernel that reads it may already run."""
    H, D = 4, 128
    N = H * D
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w1, w2 = (rnd(N, N) * N ** -0.5).to(BF16), (rnd(N, N) * N ** -0.5).to(BF16)
    start = [rnd(T, N).to(BF16), rnd(T, N).to(BF16), torch.ones(N, dtype=BF16, device="cuda"), torch.zeros(N, device="cuda")]
    stream = abi.stream_handle()
    lib = abi.lib()

    def chain(wait):
        x, res, weight, bias = (t.clone() for t in start)
        normed, gate, gated = (torch.zeros_like(x) for _ in range(3))
        a = abi.KdaNormArgs(x=x.data_ptr(), x_row_stride=N, residual=res.data_ptr(), residual_row_stride=N,
                            residual_out=res.data_ptr(), residual_out_row_stride=N, weight=weight.data_ptr(),
                            out=normed.data_ptr(), out_row_stride=N, num_tokens=T, hidden=N, eps=1e-6)
        b = linear_args(normed, w1, gate, bias=bias)
        c = abi.KdaGatedNormArgs(o=normed.data_ptr(), gate=gate.data_ptr(), gate_row_stride=N, weight=weight.data_ptr(),
                                 out=gated.data_ptr(), out_row_stride=N, num_tokens=T, num_heads=H, head_dim=D,
                                 activation=abi.KDA_ACT_SIGMOID, eps=1e-6)
        c.o_stride[0], c.o_stride[1] = N, D
        d = linear_args(gated, w2, x, residual=x)
        # The gated norm's row 0, normalised, becomes the norms' weights.
        e = abi.KdaNormArgs(x=gated.data_ptr(), x_row_stride=N, weight=weight.data_ptr(), out=weight.data_ptr(),
                            out_row_stride=N, num_tokens=1, hidden=N, eps=1.0)
        torch.cuda.synchronize()
        for _ in range(12):
            for rc in (lambda: lib.kda_rmsnorm_launch(ctypes.byref(a), stream),
                       lambda: lib.kda_linear_launch(ctypes.byref(b), None, 0, stream),
                       lambda: lib.kda_gated_rmsnorm_launch(ctypes.byref(c), stream),
                       lambda: lib.kda_linear_launch(ctypes.byref(d), None, 0, stream),
                       lambda: lib.kda_rmsnorm_launch(ctypes.byref(e), stream)):
                assert rc() == abi.KDA_OK
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return x, res, weight, normed, gate, gated

    want = chain(True)
    assert all(t.isfinite().all() for t in want)
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(chain(False), want))
