"""Key weights, eviction and linear attention together, as a server with a fixed budget of cached keys and a hybrid model runs them."""
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache, evict_by_definition, f64

pytestmark = pytest.mark.gpu


def softmax_rows(q, k, v, scale):
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p


@pytest.mark.parametrize("dtype,page", [(pkg.BF16, 16), (pkg.F16, 8), (pkg.F32, 12)])
def test_decoding_at_a_budget_of_keys_beside_a_layer_with_a_state(dtype, page):
    """Prompts of different lengths, then single tokens: attention over the cache, weights, a cut to the budget whenever a request
    is a page above it, and a linear-attention layer in the same steps.  The reference holds every head's rows itself."""
    import torch
    hq, hkv, d, budget, recent = 4, 2, 64, 96, 8
    cache = Cache(dtype, hq, hkv, d, page, 400, 3, seed=1, max_tokens=400)
    rig, ctx, scale = cache.rig, cache.rig.ctx, d ** -0.5
    tdtype = rig.arena.dtype
    weights = torch.zeros((3, hkv, cache.capacity), device="cuda")
    lin = pkg.LinearAttention(ctx, pkg.LinearConfig(1, 2, 64, 64, 0.125, dtype, 3, 1, 400))
    decay = np.array([-0.02, -0.4], np.float32)
    lin.set_decay(0, decay)
    states = torch.full((3, 1, 2, 64, 64), float("nan"), device="cuda")   # stale: a first token starts afresh
    slots, held = [2, 0], [[[], []], [[], []]]                             # per request and head: (k, v, weight)
    state = [np.zeros((2, 64, 64)), np.zeros((2, 64, 64))]
    lengths, seen = [0, 0], [0, 0]
    tol = {pkg.F32: 2e-5, pkg.BF16: 2e-2, pkg.F16: 4e-3}[dtype]
    kept = torch.zeros((2, hkv, cache.capacity), dtype=torch.int32, device="cuda")
    evictions = 0
    for step in range(40):
        runs = [150, 67] if step == 0 else [1, 1] if step % 5 else [3, 2]
        cu = np.concatenate([[0], np.cumsum(runs)]).astype(np.uint32)
        t = int(cu[-1])
        q, k, v = cache.randn(t, hq, d), cache.randn(t, hkv, d), cache.randn(t, hkv, d)
        out = torch.zeros_like(q)
        rig.gqa.prepare(slots, lengths, cu)
        rig.gqa.append_attend(rig.pages, rig.table, 0, k, v, q, out)
        rig.gqa.weigh_keys(rig.pages, rig.table, 0, q, weights, cache.capacity)
        lq, lk, lv = cache.randn(t, 1, 64), cache.randn(t, 1, 64), cache.randn(t, 2, 64)
        lout = torch.zeros_like(lv)
        lin.prepare(slots, seen, cu)
        lin.attend(0, states, lq, lk, lv, lout)
        qn, kn, vn, on = f64(q), f64(k), f64(v), f64(out)
        for r in range(2):
            for i in range(int(cu[r]), int(cu[r + 1])):
                for h in range(hkv):
                    held[r][h].append([kn[i, h], vn[i, h], 0.0])
                    ks, vs = np.stack([x[0] for x in held[r][h]]), np.stack([x[1] for x in held[r][h]])
                    for g in range(2):
                        o, p = softmax_rows(qn[i, h * 2 + g], ks, vs, scale)
                        assert np.abs(on[i, h * 2 + g] - o).max() <= tol, (step, r, i)
                        for x, w in zip(held[r][h], p):
                            x[2] += w
                state[r] = np.exp(decay.astype(np.float64))[:, None, None] * state[r] + f64(lk)[i, 0][None, :, None] * f64(lv)[i][:, None, :]
                lo = 0.125 * (f64(lq)[i, 0][None, :, None] * state[r]).sum(1)
                assert np.abs(f64(lout)[i] - lo).max() <= tol * max(1.0, np.abs(lo).max())
            lengths[r] += runs[r]
            seen[r] += runs[r]
        # f32 sums of many steps' weights: 2e-5 of the largest is far above their rounding
        got = weights.cpu().numpy()
        for r in range(2):
            for h in range(hkv):
                want = np.array([x[2] for x in held[r][h]])
                assert np.abs(got[slots[r], h, : lengths[r]] - want).max() <= 2e-5 * max(1.0, want.max()), (step, r, h)
                assert (got[slots[r], h, lengths[r]:] == 0.0).all()
        cut = [r for r in range(2) if lengths[r] >= budget + page]
        if cut:
            evictions += 1
            chosen = evict_by_definition(got[[slots[r] for r in cut]], [lengths[r] for r in cut], [budget] * len(cut), recent)
            rig.gqa.evict(rig.pages, rig.table, 0, [slots[r] for r in cut], [slots[r] for r in cut], [lengths[r] for r in cut], [budget] * len(cut),
                          recent, weights, weights, cache.capacity, kept, cache.capacity)
            ctx.sync()
            for x, r in enumerate(cut):
                for h in range(hkv):
                    assert (kept.cpu().numpy()[x, h, :budget] == chosen[x][h]).all()
                    held[r][h] = [held[r][h][i] for i in chosen[x][h]]
                lengths[r] = budget
    assert evictions >= 2
    assert np.abs(f64(states)[slots, 0] - np.stack(state)).max() <= 1e-4
    assert lin.device_status() == 0 and rig.gqa.device_status() == 0
    lin.close()
    cache.close()


def test_two_components_on_two_streams_have_scratch_of_their_own():
    import torch
    caches = []
    for s, shape in enumerate([(8, 2, 128, 16), (16, 4, 64, 8)]):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            c = Cache(pkg.BF16, *shape, 3000, 4, seed=s)
            batch = [(0, 2990, 2), (1, 1500, 40), (2, 700, 1)]
            cu = np.concatenate([[0], np.cumsum([n for _, _, n in batch])]).astype(np.uint32)
            c.rig.gqa.prepare([b[0] for b in batch], [b[1] for b in batch], cu)
            q = c.randn(int(cu[-1]), c.hq, c.d)
            weights = torch.zeros((4, c.hkv, c.capacity), device="cuda")
        caches.append((stream, c, q, weights))
    torch.cuda.synchronize()
    # alone first, then in turn: the sums of a call are added in a fixed order, so that the same 30 calls give the same bits
    alone = []
    for stream, c, q, weights in caches:
        for _ in range(30):
            c.rig.gqa.weigh_keys(c.rig.pages, c.rig.table, 0, q, weights, c.capacity)
        c.rig.ctx.sync()
        alone.append(weights.clone())
        weights.zero_()
    torch.cuda.synchronize()
    for _ in range(30):
        for _, c, q, weights in caches:
            c.rig.gqa.weigh_keys(c.rig.pages, c.rig.table, 0, q, weights, c.capacity)
    torch.cuda.synchronize()
    for (_, c, _, weights), want in zip(caches, alone):
        assert torch.equal(weights, want)
        c.close()


def test_eviction_stays_outside_captured_graphs():
    import torch
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = Cache(pkg.BF16, 2, 2, 64, 16, 64, 2, seed=3)
        w = torch.zeros((2, 2, c.capacity), device="cuda")
        kept = torch.zeros((1, 2, 64), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    c.rig.ctx.capture_begin()
    with pytest.raises(pkg.PsiError, match="outside captured graphs"):
        c.rig.gqa.evict(c.rig.pages, c.rig.table, 0, [0], [1], [60], [30], 4, w, w, c.capacity, kept, 64)
    c.rig.ctx.capture_end().close()
    c.close()


def test_objects_of_another_context_are_refused():
    import torch
    a, b = Cache(pkg.BF16, 2, 2, 64, 16, 64, 2, seed=4), Cache(pkg.BF16, 2, 2, 64, 16, 64, 2, seed=5)
    a.rig.gqa.prepare([0], [9], [0, 1])
    w = torch.zeros((2, 2, a.capacity), device="cuda")
    q = a.randn(1, 2, 64)
    kept = torch.zeros((1, 2, 64), dtype=torch.int32, device="cuda")
    for pages, table in [(b.rig.pages, a.rig.table), (a.rig.pages, b.rig.table)]:
        with pytest.raises(pkg.PsiError, match="share one context"):
            a.rig.gqa.weigh_keys(pages, table, 0, q, w, a.capacity)
        with pytest.raises(pkg.PsiError, match="share one context"):
            a.rig.gqa.evict(pages, table, 0, [0], [1], [60], [30], 4, w, w, a.capacity, kept, 64)
    a.close()
    b.close()


def test_the_checked_build_skips_and_reports_pages_beyond_the_arena():
    worker = Path(__file__).resolve().parent / "checked_memory_worker.py"
    done = subprocess.run([sys.executable, str(worker)], capture_output=True, text=True, timeout=900,
                          env={**os.environ, "PSI_CUDA_LIBRARY": "checked"})
    assert done.returncode == 0 and "checked memory ok" in done.stdout, done.stdout[-3000:] + done.stderr[-3000:]


def test_a_captured_step_of_both_layers_replays_for_later_batches():
    """Weights and states of replayed steps against the same steps launched one by one: decode rows, verify runs, a chunk."""
    import torch
    stream = torch.cuda.Stream()
    results = []
    for replayed in (False, True):
        with torch.cuda.stream(stream):
            c = Cache(pkg.BF16, 8, 2, 64, 16, 512, 3, seed=9, max_tokens=160)
            gqa, ctx = c.rig.gqa, c.rig.ctx
            lin = pkg.LinearAttention(ctx, pkg.LinearConfig(1, 2, 64, 64, 0.125, pkg.BF16, 3, 1, 160))
            lin.set_decay(0, [-0.1, -0.01])
            q, k, v, out = c.randn(160, 8, 64), c.randn(160, 2, 64), c.randn(160, 2, 64), c.randn(160, 8, 64)
            lq, lk, lv, lout = c.randn(160, 1, 64), c.randn(160, 1, 64), c.randn(160, 2, 64), c.randn(160, 2, 64)
            weights, states = torch.zeros((3, 2, c.capacity), device="cuda"), torch.zeros((3, 1, 2, 64, 64), device="cuda")
            if replayed:
                gqa.reserve_replay()

            def layers():
                gqa.append_attend(c.rig.pages, c.rig.table, 0, k, v, q, out)
                gqa.weigh_keys(c.rig.pages, c.rig.table, 0, q, weights, c.capacity)
                lin.attend(0, states, lq, lk, lv, lout)

            graph = None
            for batch in [[(0, 5, 1)], [(0, 6, 130), (1, 0, 30)], [(1, 30, 1), (0, 136, 3), (2, 100, 17)], [(2, 117, 1)], [(0, 139, 160)]]:
                cu = np.concatenate([[0], np.cumsum([n for _, _, n in batch])]).astype(np.uint32)
                # (a captured append covers the prepared capacity)
                gqa.prepare_bucketed_with_token_capacity([s for s, _, _ in batch], [f for _, f, _ in batch], cu, 160)
                lin.prepare([s for s, _, _ in batch], [f for _, f, _ in batch], cu)
                if graph is not None:
                    graph.launch()
                    continue
                layers()
                if replayed:
                    ctx.sync()
                    ctx.capture_begin()
                    layers()
                    graph = ctx.capture_end()
            ctx.sync()
            assert gqa.device_status() == 0 and lin.device_status() == 0
            results.append((weights.cpu().numpy(), states.cpu().numpy(), out.float().cpu().numpy(), lout.float().cpu().numpy()))
            if graph is not None:
                graph.close()
            lin.close()
            c.close()
    # the replayed steps split rows and keys otherwise: f32 sums of at most 1,280 rows and 64-key states in another order; bf16 outputs
    # of another order may land one step of 2^-8 apart
    (w0, s0, o0, l0), (w1, s1, o1, l1) = results
    assert np.abs(w0 - w1).max() <= 1e-5 * np.abs(w0).max()
    assert np.abs(s0 - s1).max() <= 1e-5 * np.abs(s0).max()
    assert np.abs(o0 - o1).max() <= 2.0 ** -7 * np.abs(o0).max() and np.abs(l0 - l1).max() <= 2.0 ** -7 * np.abs(l0).max()
