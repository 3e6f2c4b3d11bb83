"""The layer steps at the edges of their use: a batch without tokens, a graph
replayed on new rows."""

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


@pytest.mark.parametrize("fp8", [False, True])
def test_graph_replays_on_new_rows(ops, fp8):
    """A decode step captured once, then replayed step after step on hidden rows that were not there at its capture: the
    outputs and both pools of eager steps on the same rows."""
    N, H, D = 256, 2, 128
    w = packed(ops, N, H, D, fp8, 6)
    idx = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    seed = [to_gpu(t) for t in pools(4, H, D)]
    g = torch.Generator(device="cuda").manual_seed(7)
    steps = torch.randn(4, 2, 3, N, generator=g, device="cuda").to(BF16)

    def run(hidden, residual, state):
        return ops.kda_layer_decode(hidden, w, residual=residual, conv_state=state[0], temporal_state=state[1],
                                    cache_indices=idx, query_start_loc=cu)

    eager = [t.clone() for t in seed]
    want = [run(h, r, eager).clone() for h, r in steps]
    hidden, residual, state = steps[0, 0].clone(), steps[0, 1].clone(), [t.clone() for t in seed]
    run(hidden, residual, state)      # opt-ins and allocations ahead of the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(hidden, residual, state)
    for t, s in zip(state, seed):
        t.copy_(s)
    for i in range(4):
        hidden.copy_(steps[i, 0])
        residual.copy_(steps[i, 1])
        graph.replay()
        assert torch.equal(out, want[i])
    assert all(torch.equal(a, b) for a, b in zip(state, eager))
