"""The layer steps at the edges of their use: a batch without tokens."""

import pytest
import torch

from test_layer_gpu import make, pools, to_gpu

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from sgl_glm53_ascend_ops import ops as o
    return o


def packed(ops, N, H, D, fp8=False, seed=5):
    return ops.pack_kda_layer(**{k: v.cuda() if torch.is_tensor(v) else v for k, v in make(N, H, D, 64, seed).items()},
                              fp8=fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(0, 256), (1, 0, 256)])
def test_no_requests(ops, shape, residual, fp8):
    """A rank without requests in a step: an empty stream, the pools as they were."""
    w = packed(ops, 256, 2, 128, fp8)
    conv, temporal = (to_gpu(t) for t in pools(4, 2, 128))
    keep = conv.clone(), temporal.clone()
    hidden = torch.empty(shape, dtype=BF16, device="cuda")
    for step in (ops.kda_layer_extend, ops.kda_layer_decode):
        out = step(hidden, w, residual=hidden if residual else None, conv_state=conv, temporal_state=temporal,
                   cache_indices=torch.empty(0, dtype=torch.int32, device="cuda"),
                   query_start_loc=torch.zeros(1, dtype=torch.int32, device="cuda"))
        assert out.shape == shape and out.dtype == BF16
    torch.cuda.synchronize()
    assert torch.equal(conv, keep[0]) and torch.equal(temporal, keep[1])
