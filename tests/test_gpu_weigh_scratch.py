"""Key weights of short runs whose scores have no place in scratch: the keys are read twice."""
import pytest

from gpuharness import pkg
from memory_rig import Cache, prepare

pytestmark = pytest.mark.gpu


def test_a_batch_beyond_the_scratch_limit():
    """65 requests of 65,600 keys, 8 KV heads, 16 rows: 2.03 GiB of scores.

    The bound is that of the other tests: a score is off by (D + 2) 2^-24 of its magnitude and the exponential, sum and quotient by 2^-21,
    twice, the sum over the keys by a half step for each."""
    import torch
    slots, first, run, heads, d = 65, 65597, 2, 8, 8
    cache = Cache(pkg.BF16, 64, heads, d, 16, first + run, slots, seed=1, max_tokens=256)
    batch = [(s, first - s % 3, run) for s in range(slots)]
    tokens = prepare(cache, batch)
    q = cache.randn(tokens, 64, d)
    weights = torch.zeros((slots, heads, cache.capacity), device="cuda")
    call = lambda: cache.rig.gqa.weigh_keys(cache.rig.pages, cache.rig.table, 0, q, weights, cache.capacity)
    tiles = sum(-(-(f + n) // 32) for _, f, n in batch) * heads
    assert tiles * 32 * 16 * 4 > 2 << 30
    prepare(cache, batch[:1])
    call()                                                              # scratch of a small batch exists, and does not serve the large one
    weights.zero_()
    prepare(cache, batch)
    call()
    cache.rig.ctx.sync()
    at, worst = 0, 0.0
    for slot, f, n in batch:
        k = cache.rows(slot, 0).double()[:, : f + n]                     # [heads][keys][d]
        x = q[at:at + n].double().view(n, heads, 8, d)
        at += n
        s = torch.einsum("hkd,thgd->htgk", k, x) * cache.scale
        magnitude = (torch.einsum("hkd,thgd->htgk", k.abs(), x.abs()) * cache.scale).amax(-1, keepdim=True)
        for t in range(n):
            s[:, t, :, f + t + 1:] = -float("inf")
        p = torch.softmax(s, -1)
        off = p * (2 * ((d + 2) * 2.0 ** -24 * magnitude + 2.0 ** -21) + (f + n + 64) * 2.0 ** -24)
        want, bound = p.sum((1, 2)), off.sum((1, 2)) + p.sum((1, 2)) * 64 * 2.0 ** -24 + 1e-30
        got = weights[slot].double()
        worst = max(worst, float(((got[:, : f + n] - want).abs() / bound).max()))
        assert (got[:, f + n:] == 0).all()
    assert worst <= 1.0, worst
    cache.close()
