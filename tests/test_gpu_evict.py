"""Eviction from the paged cache by accumulated attention weight (GQA.evict) against its definition."""
import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache, evict_by_definition

pytestmark = pytest.mark.gpu


def check(cache, src, dst, lengths, keeps, recent, weights=None, same_buffer=False, extra=3):
    import torch
    b, heads, most = len(src), cache.hkv, max(max(keeps), 1) + extra
    if weights is None:
        weights = torch.rand((cache.slots, heads, cache.capacity), generator=cache.gen, device="cuda")
    before = weights.cpu().numpy()
    out = weights if same_buffer else torch.full_like(weights, -7.0)
    out_before = out.cpu().numpy()
    kept = torch.full((b, heads, most), -1, dtype=torch.int32, device="cuda")
    k0, v0 = [torch.stack([cache.rows(s, w) for s in range(cache.slots)]).view(cache.slots, heads, cache.capacity, cache.d) for w in (0, 1)]
    cache.rig.gqa.evict(cache.rig.pages, cache.rig.table, cache.layer, src, dst, lengths, keeps, recent, weights, out, cache.capacity,
                        kept, most)
    cache.rig.ctx.sync()
    k1, v1 = [torch.stack([cache.rows(s, w) for s in range(cache.slots)]) for w in (0, 1)]
    chosen = evict_by_definition(before[src], lengths, keeps, recent)
    got_kept, got_out = kept.cpu().numpy(), out.cpu().numpy()
    want_k, want_v, want_out = k0.clone(), v0.clone(), out_before.copy()
    for r in range(b):
        for h in range(heads):
            rows = chosen[r][h]
            n = len(rows)
            assert (got_kept[r, h, :n] == rows).all() and (got_kept[r, h, n:] == -1).all(), (r, h)
            at = torch.from_numpy(rows).cuda()
            want_k[dst[r], h, :n] = k0[src[r], h, at]
            want_v[dst[r], h, :n] = v0[src[r], h, at]
            want_out[dst[r], h, :n] = before[src[r], h, rows]
            want_out[dst[r], h, n:lengths[r]] = 0.0
    bits = lambda t: t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)
    assert torch.equal(bits(k1), bits(want_k)) and torch.equal(bits(v1), bits(want_v))
    assert np.array_equal(got_out, want_out, equal_nan=True)
    if not same_buffer:
        assert np.array_equal(weights.cpu().numpy(), before, equal_nan=True)


PROFILES = [(pkg.BF16, 2, 128, 16), (pkg.F16, 1, 256, 8), (pkg.F32, 3, 64, 16), (pkg.BF16, 8, 80, 12), (pkg.F16, 2, 33, 7), (pkg.F32, 1, 5, 1),
            (pkg.BF16, 5, 6, 16)]


@pytest.mark.parametrize("dtype,heads,d,page", PROFILES)
@pytest.mark.parametrize("in_place", [False, True])
def test_lengths_and_shares(dtype, heads, d, page, in_place):
    lengths = [1, 2, 17, 511, 2048, 0, 900, 2500, 33]
    keeps = [1, 1, 16, 100, 2047, 0, 0, 1251, 33]
    cache = Cache(dtype, heads, heads, d, page, 2500, 18, layers=2, layer=1, seed=d)
    src = [4, 0, 8, 2, 6, 1, 3, 5, 7]
    check(cache, src, src if in_place else [17 - s for s in src], lengths, keeps, 12)
    cache.close()


def test_recent_keys_stay_whatever_they_weigh():
    cache = Cache(pkg.BF16, 2, 2, 64, 16, 200, 4, seed=1)
    for recent in (0, 1, 50, 120, 200, 5000):
        check(cache, [0, 1], [2, 3], [200, 151], [50, 120], recent)
    cache.close()


@pytest.mark.parametrize("in_place", [False, True])
def test_equal_odd_and_extreme_weights(in_place):
    import torch
    cache = Cache(pkg.BF16, 2, 2, 64, 16, 3000, 12, seed=2)
    w = torch.zeros((12, 2, cache.capacity), device="cuda")
    w[1] = 1.0
    w[2] = torch.randint(0, 3, w[2].shape, device="cuda", generator=cache.gen).float()
    w[3] = torch.randn(w[3].shape, device="cuda", generator=cache.gen)
    w[3, :, ::3] = float("nan")
    w[4] = float("nan")
    values = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-45, -1e-45, 3.4e38], device="cuda")
    w[5] = values[torch.randint(0, 8, w[5].shape, device="cuda", generator=cache.gen)]
    src = [0, 1, 2, 3, 4, 5]
    for keeps in ([1, 2, 700, 1500, 40, 1700], [2998, 2999, 2999, 2900, 2998, 2500]):
        check(cache, src, src if in_place else [s + 6 for s in src], [2999] * 6, keeps, 2, weights=w.clone())
    cache.close()


@pytest.mark.parametrize("in_place", [False, True])
def test_one_buffer_of_weights(in_place):
    cache = Cache(pkg.F16, 2, 2, 64, 16, 5000, 4, seed=3)
    check(cache, [0, 1], [0, 1] if in_place else [3, 2], [5000, 4100], [2500, 4099], 64, same_buffer=True)
    cache.close()


def test_more_requests_than_one_launch_takes():
    n = 150
    cache = Cache(pkg.BF16, 1, 1, 32, 8, 64, 2 * n, seed=4)
    rng = np.random.default_rng(4)
    lengths = rng.integers(1, 65, n)
    keeps = [int(rng.integers(0, x + 1)) for x in lengths]
    dst = [r if r % 3 else r + n for r in range(n)]   # some in place, some not
    check(cache, list(range(n)), dst, [int(x) for x in lengths], keeps, 3)
    cache.close()


def test_a_long_row():
    cache = Cache(pkg.BF16, 1, 1, 16, 16, 100000, 2, seed=5)
    check(cache, [0], [1], [99991], [33333], 77)
    check(cache, [0], [0], [99991], [99000], 77)
    cache.close()


def test_refusals_change_nothing():
    import torch
    cache = Cache(pkg.BF16, 2, 2, 64, 16, 64, 4, seed=6)
    rig = cache.rig
    w = torch.zeros((4, 2, 64), device="cuda")
    kept = torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
    before = rig.arena.clone()
    good = dict(src=[0, 1], dst=[2, 3], lengths=[60, 64], keeps=[30, 64], recent=4, w=w, out=w, stride=64, kept=kept, kept_stride=64, layer=0)

    def call(**kw):
        a = dict(good, **kw)
        rig.gqa.evict(rig.pages, rig.table, a["layer"], a["src"], a["dst"], a["lengths"], a["keeps"], a["recent"], a["w"], a["out"], a["stride"],
                      a["kept"], a["kept_stride"])

    for kw, words in [(dict(src=[0, 4]), "req_slot out of range"), (dict(dst=[2, 9]), "req_slot out of range"), (dict(lengths=[60, 65]), "does not fit"),
                      (dict(stride=63), "hold every key"), (dict(keeps=[61, 1]), "more keys than"), (dict(kept_stride=63), "hold every kept key"),
                      (dict(src=[0, 0]), "evicted from twice"), (dict(dst=[2, 2]), "move to one slot"), (dict(dst=[1, 3]), "another one is read from"),
                      (dict(dst=[1, 0]), "another one is read from"), (dict(w=None), "not be null"), (dict(kept=None), "not be null"),
                      (dict(out=w.data_ptr() + 2), "4-byte aligned"), (dict(layer=1), "exceeds layer count"), (dict(keeps=[1]), "lengths disagree")]:
        with pytest.raises(pkg.PsiError, match=words):
            call(**kw)
    call(src=[], dst=[], lengths=[], keeps=[])
    rig.ctx.sync()
    assert torch.equal(rig.arena, before)
    cache.close()
