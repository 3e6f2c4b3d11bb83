"""Projections whose factors reach far: scales whose product passes fp32's range."""

import pytest
import torch

from layer_checks import ROUND, assert_within
from oracle import layer_ref

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from sgl_glm53_ascend_ops import ops as o
    return o


# Both kernels: few tokens, and products of more tiles than the GPU has SMs.
@pytest.mark.parametrize("T,N", [(5, 96), (1300, 1024)])
@pytest.mark.parametrize("x_scale,weight_scale,size", [(1e20, 1e20, 2.0 ** -8), (1e25, 1e25, 0.0), (1e33, 1e-4, 400.0),
                                                       (1e-20, 1e-20, 400.0)])
def test_scales_far_apart_or_large(ops, T, N, x_scale, weight_scale, size):
    """x and weight of `size`, one term a sum, tokens without a value beside them. The product is exact and
    the two scales round once each, then the output does."""
    K = 64
    x, w = torch.zeros(T, K, device="cuda"), torch.zeros(N, K, device="cuda")
    x[::2, 0], w[:, 0] = size, size
    x, w = x.to(FP8), w.to(FP8)
    sx, sw = torch.full((T,), x_scale, device="cuda"), torch.full((N,), weight_scale, device="cuda")
    want = layer_ref.linear(x, w, x_scale=sx, weight_scale=sw)[0]
    assert want.abs().max() < 3e38
    got = ops.linear(x, w, x_scale=sx, weight_scale=sw)
    assert_within(got, want, want.abs() * (ROUND[torch.bfloat16] + 2.0 ** -22))
    assert (got[1::2] == 0).all()
