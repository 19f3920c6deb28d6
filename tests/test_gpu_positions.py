"""Rotary positions apart from the token indices (GQA.set_positions): the front stage of requests whose caches were cut."""
import numpy as np
import pytest

from gpuharness import bits_of, pkg
from memory_rig import Cache, evict_by_definition, f64

pytestmark = pytest.mark.gpu

ONES = lambda d: [0x3F80] * d                                            # bf16 1.0
CONFIG = lambda rope_dim, theta=1e4: pkg.NormRopeConfig(rope_dim, 1e-6, theta, 0, 1, 1, 1, 1, 1, 0)


def stored(cache, slot, first, run):
    """Bits of the K and V rows [first, first + run) of a slot."""
    return [bits_of(cache.rows(slot, w)[:, first:first + run].contiguous()) for w in (0, 1)]


def stage(cache, form, q, k, v):
    """Rotated queries (bits) of the prepared batch by one of the two calls."""
    torch = cache.torch
    out = torch.zeros_like(q)
    if form == "rows":
        cache.rig.gqa.norm_rope_append(cache.rig.pages, cache.rig.table, 0, q, k, v, out)
    else:
        t = q.shape[0]
        pairs = torch.stack([q, -q], 2).reshape(t, -1)                    # (q, gate) of every head
        projection = torch.cat([pairs, k.reshape(t, -1), v.reshape(t, -1)], 1).contiguous()
        gates = torch.zeros_like(q)
        cache.rig.gqa.projection_norm_rope_append(cache.rig.pages, cache.rig.table, 0, projection, True, out, gates)
        assert torch.equal(gates, -q)
    cache.rig.ctx.sync()
    return bits_of(out)


@pytest.mark.parametrize("dtype,hq,hkv,d,page,rope_dim", [(pkg.BF16, 8, 2, 128, 16, 64), (pkg.F16, 4, 1, 256, 8, 256), (pkg.F32, 3, 3, 64, 16, 32),
                                                         (pkg.BF16, 4, 2, 80, 12, 40), (pkg.F32, 2, 1, 6, 5, 4)])
@pytest.mark.parametrize("form", ["rows", "projection"])
def test_a_token_is_stored_at_its_index_and_rotated_by_its_position(dtype, hq, hkv, d, page, rope_dim, form):
    """The same rows at their true places of a long cache: every bit is the same."""
    far, near = Cache(dtype, hq, hkv, d, page, 1200, 4, seed=d), Cache(dtype, hq, hkv, d, page, 1200, 4, seed=d)
    slots, indices, positions, runs = [2, 0, 3], [30, 0, 97], [1100, 7, 97], [1, 5, 3]
    cu = np.concatenate([[0], np.cumsum(runs)]).astype(np.uint32)
    q, k, v = far.randn(9, hq, d), far.randn(9, hkv, d), far.randn(9, hkv, d)
    for c in (far, near):
        c.rig.gqa.set_norm_rope(CONFIG(rope_dim), ONES(d), ONES(d))
    far.rig.gqa.prepare(slots, positions, cu)
    near.rig.gqa.prepare(slots, indices, cu)
    near.rig.gqa.set_positions([5, 5, 5])
    near.rig.gqa.set_positions(positions)                                  # the later call counts
    assert np.array_equal(stage(far, form, q, k, v), stage(near, form, q, k, v))
    for slot, index, position, run in zip(slots, indices, positions, runs):
        for a, b in zip(stored(far, slot, position, run), stored(near, slot, index, run)):
            assert np.array_equal(a, b)
    # the next step has none: token indices again
    far.rig.gqa.prepare(slots, indices, cu)
    near.rig.gqa.prepare(slots, indices, cu)
    assert np.array_equal(stage(far, form, q, k, v), stage(near, form, q, k, v))
    far.close()
    near.close()


def test_decoding_goes_on_behind_a_cut_with_the_front_stage():
    """Steps of one request through norm + RoPE + append, attention, weights and cuts; the reference holds rotated rows itself."""
    import torch
    hq, hkv, d, page, budget, recent, rope_dim = 4, 2, 64, 16, 48, 6, 32
    cache = Cache(pkg.F32, hq, hkv, d, page, 160, 2, seed=3)
    gqa, rig, scale = cache.rig.gqa, cache.rig, d ** -0.5
    gqa.set_norm_rope(CONFIG(rope_dim), ONES(d), ONES(d))
    inv = np.array(pkg.rope_parameters(CONFIG(rope_dim))[0], np.float32)
    weights = torch.zeros((2, hkv, cache.capacity), device="cuda")
    kept = torch.zeros((1, hkv, cache.capacity), dtype=torch.int32, device="cuda")
    held, length, seen, cuts = [[] for _ in range(hkv)], 0, 0, 0

    def turned(x, position):                                              # [heads][d], as the stage does it, in 64 bits
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
        angle = (np.float32(position) * inv).astype(np.float64)           # the product in f32 is the stage's own
        a, b = x[:, :rope_dim // 2], x[:, rope_dim // 2:rope_dim]
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle), x[:, rope_dim:]], 1)

    for step in range(50):
        run = 70 if step == 0 else 2
        q, k, v = cache.randn(run, hq, d), cache.randn(run, hkv, d), cache.randn(run, hkv, d)
        out, turned_q = torch.zeros_like(q), torch.zeros_like(q)
        gqa.prepare([1], [length], [0, run])
        if cuts:
            gqa.set_positions([seen])
        gqa.norm_rope_append(rig.pages, rig.table, 0, q, k, v, turned_q)
        gqa.attend(rig.pages, rig.table, 0, turned_q, out)
        gqa.weigh_keys(rig.pages, rig.table, 0, turned_q, weights, cache.capacity)
        rig.ctx.sync()
        qn, kn, vn, on = f64(q), f64(k), f64(v), f64(out)
        for i in range(run):
            rows, queries = turned(kn[i], seen + i), turned(qn[i], seen + i)
            for h in range(hkv):
                held[h].append((rows[h], vn[i, h]))
                ks, vs = np.stack([x[0] for x in held[h]]), np.stack([x[1] for x in held[h]])
                for g in range(2):
                    s = ks @ queries[h * 2 + g] * scale
                    p = np.exp(s - s.max())
                    # scores of 8 at most from 64 products, each row off by a few 2^-24: 1e-5 of a weight; ten times that
                    assert np.abs(on[i, h * 2 + g] - (p / p.sum()) @ vs).max() <= 1e-4, (step, i)
        length += run
        seen += run
        if length >= budget + page:
            cuts += 1
            chosen = evict_by_definition(weights.cpu().numpy()[1:], [length], [budget], recent)[0]
            gqa.evict(rig.pages, rig.table, 0, [1], [1], [length], [budget], recent, weights, weights, cache.capacity, kept, cache.capacity)
            held = [[held[h][i] for i in chosen[h]] for h in range(hkv)]
            length = budget
    assert cuts >= 4
    cache.close()


def test_replayed_steps_follow_the_positions():
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = Cache(pkg.BF16, 4, 2, 128, 16, 256, 3, seed=4, max_tokens=8)
        eager = Cache(pkg.BF16, 4, 2, 128, 16, 256, 3, seed=4, max_tokens=8)
        q, k, v, out = cache.randn(8, 4, 128), cache.randn(8, 2, 128), cache.randn(8, 2, 128), cache.randn(8, 4, 128)
    torch.cuda.synchronize()
    gqa, ctx, graph = cache.rig.gqa, cache.rig.ctx, None
    for c in (cache, eager):
        c.rig.gqa.set_norm_rope(CONFIG(128), ONES(128), ONES(128))
    gqa.reserve_replay()
    for slots, indices, positions, cu in [([0, 2], [9, 100], [200, 150], [0, 1, 8]), ([0, 2], [10, 107], None, [0, 3, 8]), ([1], [0], [240], [0, 8]),
                                          ([1, 0], [8, 20], [8, 20], [0, 4, 8])]:
        gqa.prepare(slots, indices, cu)
        if positions is not None:
            gqa.set_positions(positions)
        if graph is None:
            ctx.capture_begin()
            with pytest.raises(pkg.PsiError, match="stays outside captured graphs"):
                gqa.set_positions([200, 150])
            gqa.norm_rope_append(cache.rig.pages, cache.rig.table, 0, q, k, v, out)
            graph = ctx.capture_end()
        graph.launch()
        ctx.sync()
        want = torch.zeros_like(q)
        torch.cuda.synchronize()
        eager.rig.gqa.prepare(slots, indices if positions is None else positions, cu)
        eager.rig.gqa.norm_rope_append(eager.rig.pages, eager.rig.table, 0, q, k, v, want)
        eager.rig.ctx.sync()
        assert torch.equal(out, want)
    graph.close()
    cache.close()
    eager.close()


def test_refusals():
    cache = Cache(pkg.BF16, 2, 1, 64, 16, 64, 2, seed=5)
    gqa = cache.rig.gqa
    with pytest.raises(pkg.PsiError, match="must be updated before"):
        gqa.set_positions([0])
    gqa.prepare([0, 1], [3, 4], [0, 1, 3])
    with pytest.raises(pkg.PsiError, match="set_norm_rope must be called"):
        gqa.set_positions([3, 4])
    gqa.set_norm_rope(CONFIG(64), ONES(64), ONES(64))
    for positions, words in [([3], "every request"), ([3, 4, 5], "every request"), ([1 << 24, 0], "below 2\\^24"), ([0, (1 << 24) - 1], "below 2\\^24"),
                             ([0, 0xFFFFFFFF], "below 2\\^24")]:
        with pytest.raises(pkg.PsiError, match=words):
            gqa.set_positions(positions)
    gqa.set_positions([(1 << 24) - 1, (1 << 24) - 2])
    cache.close()
