"""Finite rows whose factors reach far: the norms' products must pass through no
infinity on the way to a finite value."""

import pytest
import torch

from layer_checks import check_rows, norm_error
from oracle import layer_ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from sgl_glm53_ascend_ops import ops as o
    return o


# One launch form each: few rows, the ring, rows read twice.
@pytest.mark.parametrize("T,H", [(6, 4), (6000, 9), (2, 300)])
@pytest.mark.parametrize("fp8", [False, True])
def test_gated_rmsnorm_of_large_gates(ops, T, H, fp8):
    """A SiLU gate near the type's largest value with a weight above 1, on heads of zeros and of tiny values."""
    D = 128
    g = torch.Generator().manual_seed(1)
    o, gate = torch.randn(T, H, D, generator=g).to(BF16), torch.randn(T, H * D, generator=g).to(BF16)
    w = torch.linspace(1.5, 4, D)
    o[0, 0], gate[0, :D] = 0, 3e38
    o[1, 0], gate[1, :D] = o[1, 0] * 1e-30, 3e38      # y = 1e-27 w 3e38
    y = layer_ref.gated_rmsnorm(o, gate, w, act="silu")
    assert y.isfinite().all() and y.abs().max() < 1e13
    r = ops.gated_rmsnorm(o.cuda(), gate.cuda(), w.cuda(), activation="silu", fp8=fp8)
    check_rows(r.out.cpu(), r.scale.cpu() if fp8 else None, y, BF16, norm_error(D))


# Vectors, odd rows (the second operand's rows start elsewhere), the ring, rows read twice.
@pytest.mark.parametrize("T,N,extra", [(9, 512, 0), (600, 4096, 0), (9, 515, 0), (9, 515, 1), (40, 20002, 1),
                                       (9000, 520, 0), (4000, 4096, 0), (3, 40960, 0), (3, 40961, 0)])
@pytest.mark.parametrize("fp8", [False, True])
def test_rmsnorm_of_large_rows_and_weights(ops, T, N, extra, fp8):
    """s w passes fp32's range where y = s w / rms does not; a sum of squares beyond it gives a row of zeros."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, N, generator=g).to(BF16)
    res = torch.randn(T, N, generator=g).to(BF16)
    w = (1 + 0.1 * torch.randn(N, generator=g)) * 1e25
    x[0] = (x[0].float() * 1e15).to(BF16)                     # s w of 1e40, y of 1e25
    x[1] = torch.finfo(BF16).max
    res[1] = 0
    if extra:   # x and residual whose rows start differently
        x = torch.cat([x, torch.zeros(T, extra, dtype=BF16)], dim=1).cuda()[:, :N]
    weights = [w, torch.full((N,), 2.0)]
    for wt, zero_rows in zip(weights, ([], [1])):
        keep = [i for i in range(T) if i != 1]
        r = ops.rmsnorm(x.cuda(), wt.cuda(), residual=res.cuda(), fp8=fp8)
        y, _ = layer_ref.rmsnorm(x.cpu(), wt, res)
        scale = r.scale.cpu() if fp8 else None
        check_rows(r.out.cpu()[keep], scale[keep] if fp8 else None, y[keep], BF16, norm_error(N))
        for i in zero_rows:
            assert (r.out[i].float() == 0).all() and (not fp8 or scale[i].item() == pytest.approx(1e-12))
