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
