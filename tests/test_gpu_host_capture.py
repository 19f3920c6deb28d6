"""The host captures the context's stream itself (torch.cuda.graph): linear attention follows later batches, the others refuse."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype
from memory_rig import Cache
from test_gpu_linear_attend import EPS, Rig, by_definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_linear_attention_in_a_graph_of_the_hosts_own(dtype):
    import torch
    side = torch.cuda.Stream()
    rig = Rig(dtype, 1, 2, 64, 64, slots=4, seed=1, max_tokens=300, stream=side.cuda_stream)
    rig.set_decay(0, [-0.02, -0.5])
    q, k, v = rig.inputs(300)
    out = torch.zeros((300, 2, 64), device="cuda").to(torch_dtype(dtype))
    torch.cuda.synchronize()
    rig.lin.prepare([0], [1], [0, 1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for call, words in [(lambda: rig.lin.prepare([0], [1], [0, 1]), "outside captured graphs"), (lambda: rig.lin.set_decay(0, [0.0, 0.0]), "outside captured graphs")]:
            with pytest.raises(pkg.PsiError, match=words):
                call()
        rig.lin.attend(0, rig.states, q, k, v, out)
    for batch in ([(0, 0, 5, 1)], [(1, 1, 0, 150), (2, 3, 9, 2)], [(0, 0, 6, 300)], [(3, 3, 1, 1), (2, 2, 1, 20), (1, 1, 1, 1)]):
        before = rig.states.cpu().numpy()
        cu = np.concatenate([[0], np.cumsum([n for _, _, _, n in batch])]).astype(np.uint32)
        rig.decay[0] = np.array([-0.02, -0.5], np.float32)
        rig.lin.prepare([s for s, _, _, _ in batch], [i for _, _, i, _ in batch], cu, [d for _, d, _, _ in batch])
        rig.ctx.sync()                                                    # the graph runs on the host's stream
        graph.replay()
        torch.cuda.synchronize()
        n = int(cu[-1])
        want, mag, states, states_mag = by_definition(rig, 0, before, q[:n], k[:n], v[:n], batch)
        assert (np.abs(out.double().cpu().numpy()[:n] - want) <= 2 * EPS[dtype] * mag + mag * 2.0 ** -24 * 1500).all()
        assert (np.abs(rig.states.double().cpu().numpy() - states) <= states_mag * 2.0 ** -24 * 1300 + 1e-30).all()
    assert rig.lin.device_status() == 0
    del graph
    rig.close()


def test_key_weights_eviction_and_positions_refuse_a_capture_of_the_hosts_own():
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = Cache(pkg.BF16, 4, 2, 64, 16, 128, 2, seed=2, max_tokens=8)
        weights, q = torch.zeros((2, 2, cache.capacity), device="cuda"), cache.randn(8, 4, 64)
        kept = torch.zeros((1, 2, 64), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    gqa, rig = cache.rig.gqa, cache.rig
    gqa.set_norm_rope(pkg.NormRopeConfig(64, 1e-6, 1e4, 0, 1, 1, 1, 1, 1, 0), [0x3F80] * 64, [0x3F80] * 64)
    gqa.reserve_replay()
    gqa.prepare([0], [60], [0, 1])
    gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)
    torch.cuda.synchronize()
    before = weights.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(pkg.PsiError, match="psi_ctx_capture_begin"):
            gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)
        with pytest.raises(pkg.PsiError, match="outside captured graphs"):
            gqa.evict(rig.pages, rig.table, 0, [0], [1], [60], [30], 4, weights, weights, cache.capacity, kept, 64)
        with pytest.raises(pkg.PsiError, match="outside captured graphs"):
            gqa.set_positions([7])
        q.add_(0.0)                                                       # (a graph of something)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(weights, before)
    gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)    # and goes on
    cache.rig.ctx.sync()
    del graph
    cache.close()
