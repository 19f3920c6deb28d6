"""Small caches and batches for the tests of key weights and eviction, and their definitions in 64 bits."""
import numpy as np

from gpuharness import Rig, bits_of, pkg, torch_dtype


def f64(tensor):
    return tensor.detach().double().cpu().numpy()


class Cache:
    """`slots` request slots of `capacity` tokens over a shuffled arena of random values."""

    def __init__(self, dtype, hq, hkv, d, page, capacity, slots, layers=1, layer=0, scale=None, max_tokens=4096, seed=0, kernel_mode=0):
        import torch
        self.torch, self.rng = torch, np.random.default_rng(seed)
        self.hq, self.hkv, self.d, self.page, self.slots, self.layer, self.dtype = hq, hkv, d, page, slots, layer, dtype
        per = -(-capacity // page)
        self.capacity = per * page
        self.scale = d ** -0.5 if scale is None else scale
        total = slots * layers * per
        self.rig = Rig(dtype, hq, hkv, d, page, self.scale, (slots, layers, 1, per), max_tokens, num_pages=total, kernel_mode=kernel_mode)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.gen = gen
        self.rig.arena.copy_(torch.randn(self.rig.arena.shape, generator=gen, device="cuda"))
        self.ids = self.rng.permutation(total).astype(np.uint32).reshape(slots, layers, per)
        for s in range(slots):
            for l in range(layers):
                self.rig.set_pages(s, l, self.ids[s, l])

    def randn(self, *shape, scale=1.0):
        return (self.torch.randn(shape, generator=self.gen, device="cuda") * scale).to(torch_dtype(self.dtype))

    def pages(self):
        return self.rig.arena.view(-1, 2, self.hkv, self.page, self.d)

    def rows(self, slot, which):
        """K (0) or V (1) rows of a slot as [Hkv][capacity][D], a copy."""
        ids = self.torch.from_numpy(self.ids[slot, self.layer].astype(np.int64)).cuda()
        return self.pages()[ids, which].transpose(0, 1).reshape(self.hkv, self.capacity, self.d)

    def set_row(self, slot, which, head, token, value):
        page = int(self.ids[slot, self.layer][token // self.page])
        self.pages()[page, which, head, token % self.page] = self.torch.as_tensor(value, device="cuda").to(self.rig.arena.dtype)

    def close(self):
        self.rig.close()


def weights_by_definition(cache, q, weights, batch):
    """weights after the batch, and a bound of the error that f32 arithmetic may leave, both [slots][Hkv][stride].

    A score is a sum of D products: off by at most (D + 2) half steps of 2^-24 of the sum of their magnitudes.  That much
    (as an exponent) and 2^-21 for the exponential, the row's sum and the quotient is what a weight may be off, twice (its own
    score and its row's normaliser); a column's sum over rows adds its own roundings."""
    want, bound = weights.astype(np.float64).copy(), np.zeros(weights.shape)
    group = cache.hq // cache.hkv
    at = 0
    for slot, first, run in batch:
        k = f64(cache.rows(slot, 0))
        x = f64(q)[at:at + run]
        at += run
        for h in range(cache.hkv):
            for i in range(run):
                see = first + i + 1
                for g in range(group):
                    products = k[h, :see] * x[i, h * group + g]
                    with np.errstate(all="ignore"):
                        s = products.sum(1) * cache.scale
                        top = s.max()
                        if not np.isfinite(top) or np.isnan(s).any():
                            continue
                        p = np.exp(s - top)
                    p /= p.sum()
                    magnitude = np.abs(np.where(np.isfinite(products), products, 0.0)).sum(1).max() * cache.scale
                    off = 2 * ((cache.d + 2) * 2.0 ** -24 * magnitude + 2.0 ** -21) + (see + 64) * 2.0 ** -24
                    want[slot, h, :see] += p
                    bound[slot, h, :see] += p * off
    bound += (np.abs(want) + np.abs(weights)) * 64 * 2.0 ** -24 + 1e-30
    return want, bound


def prepare(cache, batch):
    cu = np.concatenate([[0], np.cumsum([run for _, _, run in batch])]).astype(np.uint32)
    cache.rig.gqa.prepare([s for s, _, _ in batch], [f for _, f, _ in batch], cu)
    return int(cu[-1])


def evict_by_definition(weights, lengths, keeps, recent):
    """Kept indices of every request and head: `weights` [requests][Hkv][...] of the sources."""
    out = []
    for r, (n, keep) in enumerate(zip(lengths, keeps)):
        late = min(recent, keep)
        heads = []
        for h in range(weights.shape[1]):
            w = weights[r, h, : n - late].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w)
            light = np.isnan(weights[r, h, : n - late])
            order = np.lexsort((np.arange(n - late), light, -w))
            heads.append(np.concatenate([np.sort(order[: keep - late]), np.arange(n - late, n)]).astype(np.int64))
        out.append(heads)
    return out
