"""When key weights are planned: at a component's first call, then with every prepare; never for callers that do not weigh."""
import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache, prepare, weights_by_definition

pytestmark = pytest.mark.gpu


def expect(cache, q, got, before, batches):
    want, bound = before.astype(np.float64), np.zeros(before.shape)
    for batch in batches:
        tokens = sum(n for _, _, n in batch)
        more, off = weights_by_definition(cache, q[:tokens], np.zeros(before.shape, np.float32), batch)
        want, bound = want + more, bound + off + np.abs(want) * 2.0 ** -22
    assert (np.abs(got.cpu().numpy() - want) <= bound + 1e-6).all()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_the_first_call_plans_the_batch_that_is_prepared(dtype):
    import torch
    cache = Cache(dtype, 8, 2, 64, 16, 700, 6, seed=1)
    gqa, weights = cache.rig.gqa, torch.zeros((6, 2, cache.capacity), device="cuda")
    q = cache.randn(300, 8, 64)
    batches = [[(0, 10, 1), (3, 500, 200), (1, 40, 2)], [(2, 699, 1)], [(4, 0, 60), (5, 7, 1)]]
    prepare(cache, [(0, 5, 1), (1, 2, 3)])                              # a step without key weights
    prepare(cache, batches[0])
    before = weights.cpu().numpy()
    for batch in batches:
        if batch is not batches[0]:
            prepare(cache, batch)
        gqa.weigh_keys(cache.rig.pages, cache.rig.table, 0, q, weights, cache.capacity)
    cache.rig.ctx.sync()
    expect(cache, q, weights, before, batches)
    cache.close()


def test_a_first_call_between_attention_calls_leaves_them_as_they_are():
    """The plan of the step lies in the same device block."""
    import torch
    cache = Cache(pkg.BF16, 8, 2, 128, 16, 900, 6, seed=2)
    gqa, weights = cache.rig.gqa, torch.zeros((6, 2, cache.capacity), device="cuda")
    batch = [(0, 800, 2), (1, 100, 70), (2, 1, 1), (5, 899, 1)]
    tokens = prepare(cache, batch)
    q = cache.randn(tokens, 8, 128)
    outs = [torch.zeros_like(q) for _ in range(2)]
    gqa.attend(cache.rig.pages, cache.rig.table, 0, q, outs[0])
    gqa.weigh_keys(cache.rig.pages, cache.rig.table, 0, q, weights, cache.capacity)
    gqa.attend(cache.rig.pages, cache.rig.table, 0, q, outs[1])
    cache.rig.ctx.sync()
    assert torch.equal(outs[0], outs[1])
    expect(cache, q, weights, np.zeros(weights.shape, np.float32), [batch])
    cache.close()


def test_a_replay_of_the_very_batch_that_the_first_call_planned():
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = Cache(pkg.BF16, 4, 2, 64, 16, 300, 4, seed=3, max_tokens=64)
        weights, q = torch.zeros((4, 2, cache.capacity), device="cuda"), cache.randn(64, 4, 64)
    torch.cuda.synchronize()
    gqa, ctx = cache.rig.gqa, cache.rig.ctx
    gqa.reserve_replay()
    call = lambda: gqa.weigh_keys(cache.rig.pages, cache.rig.table, 0, q, weights, cache.capacity)
    batches = [[(0, 200, 1), (2, 30, 40)], [(1, 5, 64)], [(3, 299, 1), (0, 201, 3)]]
    cu = lambda batch: np.concatenate([[0], np.cumsum([n for _, _, n in batch])]).astype(np.uint32)
    prep = lambda batch: gqa.prepare([s for s, _, _ in batch], [f for _, f, _ in batch], cu(batch))
    prep(batches[0])
    call()
    ctx.capture_begin()
    call()
    graph = ctx.capture_end()
    graph.launch()                                                       # no prepare between
    for batch in batches[1:]:
        prep(batch)
        graph.launch()
    ctx.sync()
    assert gqa.device_status() == 0
    expect(cache, q, weights, np.zeros(weights.shape, np.float32), [batches[0], batches[0], *batches[1:]])
    graph.close()
    cache.close()
