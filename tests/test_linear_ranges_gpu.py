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


def activated(act, y):
    """(value, the exponential's argument) in 64 bits, without cancellation in the negative tail."""
    z = (2 / torch.pi) ** 0.5 * 2 * (y + 0.044715 * y ** 3) if act == "gelu_tanh" else y
    logistic = torch.where(z < 0, torch.exp(z) / (1 + torch.exp(z)), 1 / (1 + torch.exp(-z)))
    return {"silu": y * logistic, "sigmoid": logistic, "gelu_tanh": y * logistic}[act], z


@pytest.mark.parametrize("T,N", [(5, 700), (1300, 1400)])
@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activation_tails(ops, dtype, act, T, N):
    """Arguments that are exact (one term a sum), from one end of the exponential's range to the other, relatively:
    2^-21 of the value for the hardware's two functions and the products, 2^-24 |z| for each of five roundings of
    the exponential's argument z, and the output's rounding. Logistics below fp32's smallest normal value are zero."""
    x, w = torch.zeros(T, 64, dtype=dtype, device="cuda"), torch.zeros(N, 64, dtype=dtype, device="cuda")
    x[:, 0] = 1
    w[:, 0] = torch.cat([torch.linspace(-100, 100, N - 300), torch.linspace(-12, 12, 200), torch.logspace(-6, 0, 50),
                         -torch.logspace(-6, 0, 50)]).to(dtype)
    want, z = activated(act, w[:, 0].double())
    half_step = 2.0 ** -25 if dtype == torch.float16 else 0.0
    tol = want.abs() * (ROUND[dtype] + 2.0 ** -21 + 5 * 2.0 ** -24 * z.abs().clamp(max=100)) + 100 * 2.0 ** -126 + half_step
    got = ops.linear(x, w, activation=act)
    assert_within(got, want.expand(T, N), tol.expand(T, N), act)
