"""The attention weight that cached keys gather (GQA.weigh_keys) against its definition in 64 bits."""
import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache, prepare, weights_by_definition

pytestmark = pytest.mark.gpu


def run(cache, batch, stride=None, q=None, weights=None, calls=1):
    import torch
    tokens = prepare(cache, batch)
    q = cache.randn(tokens, cache.hq, cache.d, scale=2.0) if q is None else q
    stride = cache.capacity if stride is None else stride
    if weights is None:
        weights = torch.rand((cache.slots, cache.hkv, stride), generator=cache.gen, device="cuda") * 0.1
    before = weights.cpu().numpy()
    for _ in range(calls):
        cache.rig.gqa.weigh_keys(cache.rig.pages, cache.rig.table, cache.layer, q, weights, stride)
    cache.rig.ctx.sync()
    return q, before, weights.cpu().numpy()


def check(cache, batch, **kw):
    q, before, got = run(cache, batch, **kw)
    want, bound = weights_by_definition(cache, q, before, batch)
    off = np.abs(got - want)
    assert (off <= bound).all(), (float((off / bound).max()), np.unravel_index(np.argmax(off / bound), off.shape))
    untouched = np.ones(got.shape, bool)
    for slot, first, length in batch:
        untouched[slot, :, : first + length] = False
    assert (got[untouched] == before[untouched]).all()
    return got


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [
    (pkg.BF16, 8, 2, 128, 16), (pkg.F16, 16, 2, 256, 16), (pkg.BF16, 5, 1, 64, 8), (pkg.F16, 6, 2, 96, 12), (pkg.BF16, 4, 4, 80, 1),
    (pkg.F16, 3, 3, 8, 5), (pkg.BF16, 8, 1, 136, 16), (pkg.BF16, 32, 2, 64, 16), (pkg.BF16, 17, 1, 64, 16),
    (pkg.F32, 8, 2, 128, 16), (pkg.F32, 3, 1, 33, 7), (pkg.BF16, 4, 2, 36, 16), (pkg.F16, 2, 1, 250, 3),
])
def test_runs_of_every_length(dtype, hq, hkv, d, page):
    cache = Cache(dtype, hq, hkv, d, page, 700, 9, seed=d + hq)
    check(cache, [(3, 0, 1), (1, 699, 1), (0, 30, 1), (5, 31, 2), (2, 62, 3), (7, 0, 8), (8, 500, 70), (4, 0, 131)])
    check(cache, [(6, 63, 1)])
    cache.close()


def test_long_contexts_are_cut_into_pieces_and_joined():
    cache = Cache(pkg.BF16, 4, 1, 64, 16, 40000, 2, seed=1)
    check(cache, [(0, 39990, 2), (1, 20011, 40)])
    cache.close()


def test_a_layer_of_its_own_rows_of_any_stride_and_a_buffer_off_its_boundary():
    import torch
    cache = Cache(pkg.BF16, 4, 2, 64, 16, 100, 3, layers=3, layer=1, seed=2)
    base = torch.zeros(3 * 2 * 77 + 1, device="cuda")
    check(cache, [(2, 40, 1), (0, 76, 1)], stride=77, weights=base[1:].view(3, 2, 77))
    cache.close()


def test_the_same_call_gives_the_same_bits_and_calls_add_up():
    import torch
    cache = Cache(pkg.BF16, 8, 2, 128, 16, 3000, 4, seed=3)
    batch = [(0, 2990, 1), (1, 1500, 20), (2, 7, 1)]
    zero = lambda: torch.zeros((4, 2, cache.capacity), device="cuda")
    q, _, once = run(cache, batch, weights=zero())
    _, _, again = run(cache, batch, q=q, weights=zero())
    assert (once == again).all()
    _, _, twice = run(cache, batch, q=q, weights=zero(), calls=2)
    assert np.array_equal(twice, once + once)
    cache.close()


@pytest.mark.parametrize("dtype,d", [(pkg.BF16, 64), (pkg.F32, 64)])
@pytest.mark.parametrize("tokens", [1, 30])
def test_rows_without_a_softmax_add_nothing_and_masked_values_do_not_count(dtype, d, tokens):
    cache = Cache(dtype, 2, 1, d, 16, 128, 2, seed=4)
    first = 64
    q = cache.randn(tokens, 2, d)
    q[:, 0] = 0
    q[:, 0, 0] = 1.0
    q[:, 1] = q[:, 0]
    q[:, 1, 0] = 0.0
    q[:, 1, 1] = 1.0                                    # head 0 reads column 0 of K, head 1 column 1
    for token in range(cache.capacity):
        row = np.full(d, 0.25, np.float32)
        if token >= first + tokens:
            row[:] = np.nan if token % 2 else np.inf     # behind every row's limit
        cache.set_row(0, 0, 0, token, row)
        cache.set_row(1, 0, 0, token, row)
    batch = [(0, first, tokens)]
    check(cache, batch, q=q)
    row = np.full(d, 0.25, np.float32)
    row[0] = -np.inf                                     # head 0's score of key 3 is -inf: weight 0
    row[1] = np.inf                                      # head 1's is +inf: its rows add nothing
    cache.set_row(0, 0, 0, 3, np.where(np.isinf(row), row, 0.0))
    q[:, 0, 1:] = 1e-3 if dtype == pkg.F32 else 0.0
    got = run(cache, batch, q=q)[2]
    assert np.isfinite(got).all()
    cache.close()


def test_every_score_at_minus_infinity_adds_nothing():
    import torch
    cache = Cache(pkg.BF16, 1, 1, 64, 16, 64, 1, seed=5)
    for token in range(cache.capacity):
        row = np.zeros(64, np.float32)
        row[0] = -np.inf
        cache.set_row(0, 0, 0, token, row)
    q = torch.ones((1, 1, 64), device="cuda").bfloat16()
    _, before, got = run(cache, [(0, 40, 1)], q=q)
    assert (got == before).all()
    cache.close()


def test_a_sharp_softmax_keeps_its_small_weights():
    cache = Cache(pkg.F16, 2, 1, 64, 16, 600, 1, scale=1.0, seed=6)
    check(cache, [(0, 511, 4)])
    cache.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_captured_launches_follow_the_batch(dtype):
    import torch
    cache = Cache(dtype, 4, 2, 64, 16, 300, 6, seed=7, max_tokens=40)
    side = torch.cuda.Stream()
    rig, ctx = cache.rig, pkg.Context(0, stream=side.cuda_stream)
    pages = pkg.PageArena(ctx, rig.num_pages, rig.page_bytes, device_ptr=rig.arena)
    table = pkg.GQARequestPageTable(ctx, rig.layout)
    for s in range(cache.slots):
        table.write_row(s, 0, cache.ids[s, 0])
    gqa = pkg.GQA(ctx, rig.gqa.config)
    q = cache.randn(40, 4, 64)
    weights = torch.zeros((6, 2, cache.capacity), device="cuda")
    torch.cuda.synchronize()
    steps = [[(0, 10, 1), (3, 250, 30)], [(1, 299, 1)], [(5, 0, 40)], [(2, 33, 4), (4, 120, 4)]]

    def prep(batch):
        cu = np.concatenate([[0], np.cumsum([n for _, _, n in batch])]).astype(np.uint32)
        gqa.prepare([s for s, _, _ in batch], [f for _, f, _ in batch], cu)

    gqa.reserve_replay()
    prep(steps[0])
    ctx.capture_begin()
    with pytest.raises(pkg.PsiError, match="once after the replay reservation"):
        gqa.weigh_keys(pages, table, 0, q, weights, cache.capacity)
    ctx.capture_end().close()
    gqa.weigh_keys(pages, table, 0, q, weights, cache.capacity)
    ctx.sync()
    weights.zero_()
    torch.cuda.synchronize()
    ctx.capture_begin()
    with pytest.raises(pkg.PsiError, match="as long as the page table's"):
        gqa.weigh_keys(pages, table, 0, q, weights, cache.capacity - 1)
    gqa.weigh_keys(pages, table, 0, q, weights, cache.capacity)
    graph = ctx.capture_end()
    want = np.zeros((6, 2, cache.capacity))
    bound = np.zeros_like(want)
    for batch in steps:
        prep(batch)
        graph.launch()
        ctx.sync()
        more, off = weights_by_definition(cache, q[: sum(n for _, _, n in batch)], np.zeros_like(want, np.float32), batch)
        want += more
        bound += off + np.abs(want) * 2.0 ** -22
        assert (np.abs(weights.cpu().numpy() - want) <= bound).all()
    with pytest.raises(pkg.PsiError, match="appears twice"):
        prep([(0, 10, 1), (0, 11, 1)])
    graph.close()
    for o in (gqa, table, pages, ctx):
        o.close()
    cache.close()


def test_refusals():
    import torch
    cache = Cache(pkg.BF16, 4, 2, 64, 16, 100, 3, seed=8, max_tokens=16)
    rig = cache.rig
    q = cache.randn(16, 4, 64)
    weights = torch.zeros((3, 2, cache.capacity), device="cuda")
    call = lambda q=q, weights=weights, layer=0, stride=cache.capacity: rig.gqa.weigh_keys(rig.pages, rig.table, layer, q, weights, stride)
    with pytest.raises(pkg.PsiError, match="must be updated before"):
        call()
    prepare(cache, [(0, 50, 2), (1, 60, 1)])
    for kw, words in [(dict(q=None), "not be null"), (dict(weights=None), "not be null"), (dict(layer=1), "exceeds layer count"),
                      (dict(stride=60), "hold every key"), (dict(q=q.data_ptr() + 2), "16-byte aligned"),
                      (dict(weights=weights.data_ptr() + 2), "4-byte aligned")]:
        with pytest.raises(pkg.PsiError, match=words):
            call(**kw)
    prepare(cache, [(0, 50, 1), (1, 60, 1), (0, 50, 1)])
    with pytest.raises(pkg.PsiError, match="appears twice"):
        call()
    rig.ctx.sync()
    assert not weights.any()
    cache.close()
