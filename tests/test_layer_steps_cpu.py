"""The layer steps' own wiring on the CPU: the operators they call replaced by
plain forms of the same shapes."""

import pytest
import torch

from oracle import layer_ref

BF16 = torch.bfloat16


@pytest.fixture
def layer(monkeypatch):
    from sgl_glm53_ascend_ops.ops import layer as m
    from sgl_glm53_ascend_ops.ops.norm import NormOutput

    def rmsnorm(x, weight, residual=None, eps=1e-6, fp8=False):
        y, s = layer_ref.rmsnorm(x, weight, residual, eps)
        return NormOutput(y.to(x.dtype), None, None if residual is None else s.to(x.dtype))

    def gated_rmsnorm(o, gate, weight, eps=1e-6, activation="sigmoid", fp8=False):
        return NormOutput(o.flatten(1) * gate)

    def linear(x, weight, bias=None, residual=None, x_scale=None, weight_scale=None):
        return layer_ref.linear(x, weight, bias, residual)[0].to(x.dtype)

    def step(*, mixed, a, b, head_dim, A_log, **kw):
        T, H = mixed.shape[0], A_log.numel()
        assert mixed.shape == (T, 3 * H * head_dim) and a.shape == (T, H * head_dim) and b.shape == (T, H)
        return mixed[:, :H * head_dim].reshape(1, T, H, head_dim)

    for name, f in (("rmsnorm", rmsnorm), ("gated_rmsnorm", gated_rmsnorm), ("linear", linear),
                    ("kda_forward_extend", step), ("kda_forward_decode", step)):
        monkeypatch.setattr(m, name, f)
    return m


def weights(layer, N=48, H=2, D=64, R=16):
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF16)  # noqa: E731
    HD = H * D
    return layer.pack_kda_layer(
        norm=rnd(N), qkv_proj=rnd(3 * HD, N), decay_down=rnd(R, N), decay_up=rnd(HD, R), gate_down=rnd(R, N),
        gate_up=rnd(HD, R), gate_bias=None, beta_proj=rnd(H, N), conv_weight=rnd(3 * HD, 4).float(), conv_bias=None,
        A_log=torch.zeros(H), dt_bias=torch.zeros(HD), out_norm=rnd(D), out_proj=rnd(N, HD), lower_bound=-5.0)


@pytest.mark.parametrize("shape", [(0, 48), (1, 0, 48), (3, 48), (1, 3, 48)])
@pytest.mark.parametrize("residual", [False, True])
def test_steps_keep_the_stream_s_shape(layer, shape, residual):
    """No tokens are a batch like any other: a rank without requests runs its step."""
    w = weights(layer)
    hidden = torch.ones(shape, dtype=BF16)
    tokens = shape[-2]
    for step in (layer.kda_layer_extend, layer.kda_layer_decode):
        out = step(hidden, w, residual=hidden if residual else None, head_dim=64, conv_state=None, temporal_state=None,
                   cache_indices=torch.zeros(tokens, dtype=torch.int32),
                   query_start_loc=torch.arange(tokens + 1, dtype=torch.int32))
        assert out.shape == hidden.shape and out.dtype == BF16
