"""The attention layer's projections: a matrix product with its epilogue.

The reference's op starts after the layer's projections, which sglang's model
code owns (the arguments ``q, k, v, a, b`` of
``sgl-glm53-ascend-ops/csrc/kda/recurrent/kda_varlen_recurrent.cpp:257-264``).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

_linear = torch.ops.sgl_glm53_ascend.kda_linear.default


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    x_scale: Optional[torch.Tensor] = None,
    weight_scale: Optional[torch.Tensor] = None,
    activation: str = "none",
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``activation(x @ weight.T * weight_scale * x_scale[:, None] + bias) + residual``.

    x [T, K] or [1, T, K] and weight [N, K], both bf16, both fp16, or both
    float8_e4m3fn with fp32 scales per token and per output (see
    :func:`quantize_weight`); columns contiguous, any row stride. bias fp32
    [N]; residual [T, N] in the output's type; activation "none", "silu",
    "sigmoid", "relu" or "gelu_tanh". Sums are fp32. The output has the type
    of 16-bit operands; of e4m3 ones it is ``out_dtype`` (bf16 by default, or
    fp16). T may be 0.

    Operands are read in place where each row starts on a 16-byte boundary
    (base and row stride); others are copied to such rows first, on every
    call, so keep odd-width weights in padded rows.
    """
    return _linear(x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype)


def quantize_weight(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weights laid out once for e4m3 products: ([N, K] float8_e4m3fn, fp32 scale [N]),
    scale = max(max|w[n]| / 448, 1e-12) of each output's row."""
    if weight.dim() != 2:
        raise ValueError(f"quantize_weight expects [N, K], got {list(weight.shape)}")
    w = weight.float()
    scale = torch.clamp_min(w.abs().amax(dim=1) / 448.0, 1e-12)
    return (w / scale[:, None]).to(torch.float8_e4m3fn), scale
