"""One KDA attention layer on the package's operators: input norm, projections,
conv front end, KDA op, gated output norm and output projection.

The steps between the projections are those of sglang's attention backend
(``AscendKDAAttnBackend.forward_extend``, exercised by
``sgl-glm53-ascend-ops/tests/integration/test_glm53_kda_prefix_ascendc.py:325-387``);
the layer around them is the model's. :func:`pack_kda_layer` lays the weights
out once, :func:`kda_layer_extend` and :func:`kda_layer_decode` run a step.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .conv import kda_forward_decode, kda_forward_extend
from .linear import linear, quantize_weight
from .norm import gated_rmsnorm, rmsnorm


class KDALayerWeights(NamedTuple):
    """A layer's weights as the steps read them (see :func:`pack_kda_layer`)."""

    norm: torch.Tensor                    # [N]
    in_proj: torch.Tensor                 # [3 H D + 2 R + H, rounded up to 16; N]: q | k | v | decay and gate factors | beta
    in_scale: Optional[torch.Tensor]      # scales of an e4m3 in_proj
    decay_up: torch.Tensor                # [H D, R]: the decay's second factor
    gate_up: torch.Tensor                 # [H D, R]: the output gate's second factor
    gate_bias: Optional[torch.Tensor]     # [H D] fp32
    conv_weight: torch.Tensor             # [3 H D, W]
    conv_bias: Optional[torch.Tensor]
    A_log: torch.Tensor                   # [H] fp32
    dt_bias: torch.Tensor                 # [H D] fp32
    out_norm: torch.Tensor                # [D]
    out_proj: torch.Tensor                # [N, H D]
    out_scale: Optional[torch.Tensor]     # scales of an e4m3 out_proj
    lower_bound: float
    eps: float


def pack_kda_layer(
    *,
    norm: torch.Tensor,
    qkv_proj: torch.Tensor,
    decay_down: torch.Tensor,
    decay_up: torch.Tensor,
    gate_down: torch.Tensor,
    gate_up: torch.Tensor,
    gate_bias: Optional[torch.Tensor],
    beta_proj: torch.Tensor,
    conv_weight: torch.Tensor,
    conv_bias: Optional[torch.Tensor],
    A_log: torch.Tensor,
    dt_bias: torch.Tensor,
    out_norm: torch.Tensor,
    out_proj: torch.Tensor,
    lower_bound: float,
    eps: float = 1e-6,
    fp8: bool = False,
) -> KDALayerWeights:
    """Lays a layer's weights out once. All projections are [outputs, inputs]
    bf16: qkv_proj [3 H D, N], decay_down and gate_down [R, N], decay_up and
    gate_up [H D, R], beta_proj [H, N], out_proj [N, H D]. The five that read
    the normalised hidden row become one matrix, padded with zero rows so that
    its output's rows start on 16 bytes; with ``fp8`` it and out_proj are
    rounded to e4m3 with a scale per output."""
    rows = torch.cat([qkv_proj, decay_down, gate_down, beta_proj])
    pad = -rows.shape[0] % 16
    if pad:
        rows = torch.cat([rows, rows.new_zeros(pad, rows.shape[1])])
    in_scale = out_scale = None
    if fp8:
        rows, in_scale = quantize_weight(rows)
        out_proj, out_scale = quantize_weight(out_proj)
    return KDALayerWeights(norm, rows, in_scale, decay_up, gate_up, gate_bias, conv_weight, conv_bias, A_log, dt_bias,
                           out_norm, out_proj, out_scale, lower_bound, eps)


def _layer(step, hidden, w, residual, head_dim, **kwargs):
    T = hidden.shape[-2]
    H, R = w.A_log.numel(), w.decay_up.shape[1]
    C = 3 * H * head_dim
    stream = hidden.reshape(T, hidden.shape[-1])   # T may be 0
    x = rmsnorm(stream, w.norm, None if residual is None else residual.reshape(stream.shape), w.eps,
                fp8=w.in_scale is not None)
    p = linear(x.out, w.in_proj, x_scale=x.scale, weight_scale=w.in_scale)
    a = linear(p[:, C:C + R], w.decay_up)
    gate = linear(p[:, C + R:C + 2 * R], w.gate_up, bias=w.gate_bias)
    b = p[:, C + 2 * R:C + 2 * R + H].contiguous()
    o = step(mixed=p[:, :C], a=a, b=b, conv_weights=w.conv_weight, conv_bias=w.conv_bias, A_log=w.A_log,
             dt_bias=w.dt_bias, lower_bound=w.lower_bound, head_dim=head_dim, **kwargs)
    y = gated_rmsnorm(o[0], gate, w.out_norm, w.eps, fp8=w.out_scale is not None)
    if residual is not None:
        stream = x.residual
    return linear(y.out, w.out_proj, residual=stream, x_scale=y.scale, weight_scale=w.out_scale).view(hidden.shape)


def kda_layer_extend(
    hidden: torch.Tensor,
    weights: KDALayerWeights,
    *,
    conv_state: torch.Tensor,
    temporal_state: torch.Tensor,
    cache_indices: torch.Tensor,
    query_start_loc: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    head_dim: int = 128,
    scale: Optional[float] = None,
    has_initial_state: Optional[torch.Tensor] = None,
    track_indices: Optional[torch.Tensor] = None,
    track_lens: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One layer's extend (prefill) step over a varlen batch: the residual
    stream hidden [T, N] (or [1, T, N]) bf16, plus ``residual`` where the block
    before hands over two parts, to the stream after the layer. The pools and
    the other arguments are those of :func:`kda_forward_extend`. The output
    projection adds the stream, so the weights hold all of the layer's heads:
    results over parts of the heads cannot be summed (each has the stream)."""
    return _layer(kda_forward_extend, hidden, weights, residual, head_dim, conv_state=conv_state,
                  temporal_state=temporal_state, cache_indices=cache_indices, query_start_loc=query_start_loc,
                  scale=scale, has_initial_state=has_initial_state, track_indices=track_indices, track_lens=track_lens)


def kda_layer_decode(
    hidden: torch.Tensor,
    weights: KDALayerWeights,
    *,
    conv_state: torch.Tensor,
    temporal_state: torch.Tensor,
    cache_indices: torch.Tensor,
    query_start_loc: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    head_dim: int = 128,
    scale: Optional[float] = None,
    intermediate_state: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One layer's decode (or verify) step; see :func:`kda_layer_extend` and
    :func:`kda_forward_decode`."""
    return _layer(kda_forward_decode, hidden, weights, residual, head_dim, conv_state=conv_state,
                  temporal_state=temporal_state, cache_indices=cache_indices, query_start_loc=query_start_loc,
                  scale=scale, intermediate_state=intermediate_state)
