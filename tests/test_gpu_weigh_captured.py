"""A captured key-weight launch refuses batches that name a slot twice, for as long as its graph lives."""
import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache, f64

pytestmark = pytest.mark.gpu


def test_a_slot_named_twice_is_refused_until_the_last_graph_is_gone():
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = Cache(pkg.BF16, 4, 2, 64, 16, 128, 3, seed=1, max_tokens=8)
        weights, q, out = torch.zeros((3, 2, cache.capacity), device="cuda"), cache.randn(8, 4, 64), cache.randn(8, 4, 64)
    torch.cuda.synchronize()
    gqa, ctx, rig = cache.rig.gqa, cache.rig.ctx, cache.rig
    weigh = lambda: gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)
    twice = lambda: gqa.prepare([0, 0], [60, 60], [0, 1, 2])              # two rows at one position: attention takes them

    gqa.reserve_replay()
    gqa.prepare([0], [60], [0, 1])
    weigh()
    twice()                                                               # nothing is captured yet
    with pytest.raises(pkg.PsiError, match="appears twice"):
        weigh()
    gqa.prepare([0], [60], [0, 1])
    graphs = []
    for _ in range(2):
        ctx.capture_begin()
        weigh()
        weigh()
        graphs.append(ctx.capture_end())
        with pytest.raises(pkg.PsiError, match="appears twice"):
            twice()
        gqa.prepare([0], [60], [0, 1])
    graphs[0].launch()
    ctx.sync()
    graphs[0].close()
    with pytest.raises(pkg.PsiError, match="appears twice"):
        twice()
    graphs[1].close()
    twice()
    gqa.attend(rig.pages, rig.table, 0, q, out)
    ctx.sync()
    k, v, x = f64(cache.rows(0, 0))[:, :61], f64(cache.rows(0, 1))[:, :61], f64(q)
    for t in range(2):
        for h in range(4):
            s = k[h // 2] @ x[t, h] * cache.scale
            p = np.exp(s - s.max())
            assert np.abs(f64(out)[t, h] - (p / p.sum()) @ v[h // 2]).max() <= 2e-2   # bf16 outputs of about one
    cache.close()


def test_a_capture_that_holds_no_key_weights_refuses_nothing():
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = Cache(pkg.BF16, 4, 2, 64, 16, 128, 3, seed=2, max_tokens=8)
        weights, q, out = torch.zeros((3, 2, cache.capacity), device="cuda"), cache.randn(8, 4, 64), cache.randn(8, 4, 64)
    torch.cuda.synchronize()
    gqa, ctx, rig = cache.rig.gqa, cache.rig.ctx, cache.rig
    gqa.reserve_replay()
    gqa.prepare([0], [60], [0, 1])
    gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)
    ctx.capture_begin()
    gqa.attend(rig.pages, rig.table, 0, q, out)
    graph = ctx.capture_end()
    gqa.prepare([0, 0], [60, 60], [0, 1, 2])
    graph.launch()
    ctx.sync()
    graph.close()
    cache.close()
