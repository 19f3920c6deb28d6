"""The operators of bounded sequence memory, as a serving program calls them: the attention weight that each cached key gathers
(``GQA.weigh_keys``), the eviction that it decides (``GQA.evict``), and linear attention with a decay for each head, whose state
does not grow (``LinearAttention``), for prompts and for single tokens.

A case is one call for one layer of one step.  What a program makes once per batch and uses in every layer (the prepared
batch, the page table, the buffers) is part of the state; so are the library's objects.  Lengths are evenly spaced quantiles
of the case's range; the seed orders the requests, places their pages and draws the values.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": (torch.float32, 4), "bf16": (torch.bfloat16, 2), "f16": (torch.float16, 2)}


def _weigh(name, dtype, heads, head_dim, page, requests, ctx, run=(1, 1), spread="even"):
    c = dict(op="weigh", dtype=dtype, q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim, page=page, requests=requests,
             ctx_lo=ctx[0], ctx_hi=ctx[1], run_lo=run[0], run_hi=run[1], spread=spread)
    return dict(c, name=name) if name else c


def _evict(name, dtype, kv_heads, head_dim, page, requests, ctx, keep, recent, in_place, spread="even"):
    c = dict(op="evict", dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, page=page, requests=requests, ctx_lo=ctx[0],
             ctx_hi=ctx[1], keep=keep, recent=recent, in_place=in_place, spread=spread)
    return dict(c, name=name) if name else c


def _linear(name, dtype, heads, dims, requests, run, fresh, fork):
    c = dict(op="linear", dtype=dtype, k_heads=heads[0], v_heads=heads[1], key_dim=dims[0], value_dim=dims[1],
             requests=requests, run_lo=run[0], run_hi=run[1], fresh=fresh, fork=fork)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One chat user, the next token: latency (40/8 heads, 8-token pages).
        _weigh("weigh-one", "bf16", (40, 8), 128, 8, 1, (777, 777)),
        # The everyday decode batch of the sparse 35B profile.
        _weigh("weigh-batch", "bf16", (16, 2), 256, 16, 32, (1024, 8192)),
        # Speculative decoding with one drafted token per request, dense 27B profile in f16.
        _weigh("weigh-verify", "f16", (24, 4), 256, 16, 64, (4096, 32768), run=(2, 2), spread="log"),
        # The end of long prompts looks back over the whole prompt before the cache is cut.
        _weigh("weigh-window", "bf16", (32, 8), 128, 16, 4, (4099, 16384), run=(64, 64)),
        # One user at the budget: a page's worth of keys leaves, in place.
        _evict("evict-one", "bf16", 8, 128, 8, 1, (1037, 1037), 0.985, 256, True),
        # A batch cut to half; the pages are shared with the prefix cache, so the kept rows go to pages of their own.
        _evict("evict-batch", "bf16", 2, 256, 16, 32, (1024, 8192), 0.5, 128, False),
        # Long documents of a float32 model cut to a quarter after the prompt.
        _evict("evict-long", "f32", 8, 128, 16, 2, (65001, 131072), 0.25, 512, False),
        # One chat user, the next token of a layer with a state.
        _linear("linear-one", "bf16", (16, 32), (128, 128), 1, (1, 1), 0.0, False),
        # The next token of a full batch.
        _linear("linear-batch", "bf16", (16, 32), (128, 128), 128, (1, 1), 0.0, False),
        # Drafts under verification: the state after them goes to a slot of its own, so that a rejection can go back.
        _linear("linear-verify", "f16", (16, 32), (128, 128), 32, (4, 8), 0.0, True),
        # New prompts of ragged length.
        _linear("linear-prompt", "bf16", (16, 32), (128, 128), 3, (611, 2500), 1.0, False),
        # A chunk of one long prompt behind an earlier chunk.
        _linear("linear-long", "f16", (32, 32), (128, 128), 1, (8192, 8192), 0.0, False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pair(rng, lo, hi):
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return min(a, b), max(a, b)


def draw(rng):
    op = rng.choice(("weigh", "evict", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "linear":
        k_heads = rng.choice((1, 4, 8, 16))
        heads = (k_heads, k_heads * rng.choice((1, 2)))
        dims = rng.choice(((128, 128), (128, 128), (64, 64), (64, 128), (128, 64), (96, 80)))
        if rng.random() < 0.5:  # single tokens and drafts
            return _linear(None, dtype, heads, dims, _log(rng, 1, 128), _pair(rng, 1, 8), rng.choice((0.0, 0.1)), rng.random() < 0.4)
        # prompts: a few, ragged; other types and sizes than the 16-bit ones of 64 and 128 stay short
        long = dtype != "f32" and 96 not in dims
        return _linear(None, dtype, heads, dims, _log(rng, 1, 4), _pair(rng, 9, 4096 if long else 700), rng.choice((0.0, 0.5, 1.0)),
                       rng.random() < 0.4)
    kv_heads = rng.choice((1, 2, 4, 8))
    head_dim = rng.choice((64, 128, 128, 256, 80, 96))
    page = rng.choice((8, 16, 16, 32, 12, 1))
    spread = rng.choice(("even", "log"))
    if op == "evict":
        return _evict(None, dtype, kv_heads, head_dim, page, _log(rng, 1, 12), _pair(rng, 40, 4096), rng.choice((0.1, 0.5, 0.9, 0.99)),
                      rng.choice((0, 1, 32, 100)), rng.random() < 0.5, spread)
    heads = (kv_heads * rng.choice((1, 3, 4, 5, 8)), kv_heads)
    kind = rng.random()
    if kind < 0.6:  # the next token, or drafts
        return _weigh(None, dtype, heads, head_dim, page, _log(rng, 1, 32), _pair(rng, 40, 6000), _pair(rng, 1, 8), spread)
    # the end of prompts, or whole short ones
    return _weigh(None, dtype, heads, head_dim, page, _log(rng, 1, 3), _pair(rng, 200, 4000), _pair(rng, 9, 200), spread)


def _lengths(lo, hi, n, spread):
    at = [(i + 0.5) / n for i in range(n)]
    if spread == "log":
        return [int(round(lo * (hi / lo) ** p)) for p in at]
    return [int(round(lo + (hi - lo) * p)) for p in at]


def _runs(case):
    """Query tokens of each request: quantiles in an order of their own, never more than the request's keys."""
    runs = _lengths(case["run_lo"], case["run_hi"], case["requests"], "even")[::-1]
    if case["op"] == "weigh":
        runs = [min(r, n) for r, n in zip(runs, _contexts(case))]
    return runs


def _contexts(case):
    return _lengths(case["ctx_lo"], case["ctx_hi"], case["requests"], case["spread"])


def _keeps(case):
    return [max(1, int(n * case["keep"])) for n in _contexts(case)]


def _randn(gen, dtype, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=dtype if dtype == torch.float32 else torch.bfloat16) * scale).to(dtype)


class _Objects:
    """The library's objects of one state, closed with it."""

    def __init__(self, *objects):
        self.objects = objects

    def __del__(self):
        for o in self.objects:
            o.close()


def _package():
    from __graft_entry__ import load_package
    return load_package()


def _cache(case, seed, rows_per_slot, num_slots):
    """A page arena with the pages of `num_slots` requests in random order, and the page IDs of each slot."""
    dtype, _ = _TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 31))
    per_slot = [-(-n // case["page"]) for n in rows_per_slot]
    total = sum(per_slot)
    ids = order.permutation(total).astype(np.uint32)
    most = max(per_slot)
    table = np.zeros((num_slots, most), np.uint32)
    at = 0
    for s, n in enumerate(per_slot):
        table[s, :n] = ids[at:at + n]
        at += n
    pages = _randn(gen, dtype, total, 2, case["kv_heads"], case["page"], case["head_dim"])
    return gen, order, pages, table


def _gqa_objects(case, state, table, q_heads, max_tokens):
    pkg = _package()
    ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    layout = pkg.GQAPageTableLayout(table.shape[0], 1, 1, table.shape[1])
    pages = state["pages"]
    page_bytes = pages[0].numel() * pages.element_size()
    arena = pkg.PageArena(ctx, pages.shape[0], page_bytes, device_ptr=pages)
    rows = pkg.GQARequestPageTable(ctx, layout)
    for s in range(table.shape[0]):
        rows.write_row(s, 0, table[s])
    dtype = {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[case["dtype"]]
    gqa = pkg.GQA(ctx, pkg.GQAConfig(q_heads, case["kv_heads"], case["head_dim"], state["scale"], page_bytes, dtype, layout,
                                     max_tokens, pkg.PLAN_BALANCED, pkg.KERNEL_AUTO, 0))
    state.update(gqa=gqa, arena=arena, rows=rows, objects=_Objects(gqa, rows, arena, ctx))


def _prepare_weigh(case, seed):
    dtype, _ = _TYPES[case["dtype"]]
    n, runs = _contexts(case), _runs(case)
    b = len(n)
    gen, order, pages, table = _cache(case, seed, n, b)
    tokens = sum(runs)
    stride = table.shape[1] * case["page"]
    state = dict(case=case, pages=pages, scale=case["head_dim"] ** -0.5, stride=stride,
                 q=_randn(gen, dtype, tokens, case["q_heads"], case["head_dim"], scale=2.0),
                 weights=torch.rand((b, case["kv_heads"], stride), generator=gen, device="cuda") * (4.0 * case["q_heads"] / case["kv_heads"] / case["ctx_hi"]))
    batch = order.permutation(b)  # the order of the step's requests; slot s holds request s
    cu = np.concatenate([[0], np.cumsum([runs[s] for s in batch])]).astype(np.uint32)
    most = max(runs)
    row = cu[:-1, None].astype(np.int64) + np.arange(most)
    state.update(
        slots=torch.tensor(batch, device="cuda"), page_ids=torch.tensor(table[batch].astype(np.int64), device="cuda"),
        # row (request, i) of the padded queries, and how many keys it sees (0: padding)
        row=torch.tensor(np.minimum(row, tokens - 1), device="cuda"),
        sees=torch.tensor(np.array([[n[s] - runs[s] + i + 1 if i < runs[s] else 0 for i in range(most)] for s in batch]), device="cuda"))
    if own:  # the objects and the prepared batch that a serving program keeps
        _gqa_objects(case, state, table, case["q_heads"], tokens)
        state["gqa"].prepare([int(s) for s in batch], [n[s] - runs[s] for s in batch], cu)
    state["host"] = (batch, n, runs, cu, table)
    return state


def _run_weigh(s):
    c, weights = s["case"], s["weights"]
    if own:
        s["gqa"].weigh_keys(s["arena"], s["rows"], 0, s["q"], weights, s["stride"])
        return weights
    b, heads, d = len(s["slots"]), c["kv_heads"], c["head_dim"]
    k = s["pages"][:, 0][s["page_ids"]].transpose(1, 2).reshape(b, heads, -1, d).float()
    q = s["q"][s["row"]].float().reshape(b, -1, heads, c["q_heads"] // heads, d).permute(0, 2, 1, 3, 4)
    score = torch.matmul(q.reshape(b, heads, -1, d), k.transpose(2, 3)) * s["scale"]
    sees = s["sees"].repeat_interleave(c["q_heads"] // heads, 1)[:, None, :, None]
    hidden = torch.arange(score.shape[3], device="cuda") >= sees
    score.masked_fill_(hidden, float("-inf"))
    top = score.amax(3, keepdim=True).clamp_min(-1e30)
    p = torch.exp(score.sub_(top))
    p = p / p.sum(3, keepdim=True).clamp_min(1e-30)
    weights[s["slots"]] = weights[s["slots"]] + p.sum(2)
    return weights


def _exact_weigh(case, seed):
    s = _prepare_weigh(case, seed)
    batch, n, runs, cu, table = s["host"]
    weights, group = s["weights"].double(), case["q_heads"] // case["kv_heads"]
    for r, slot in enumerate(batch):
        ids = torch.tensor(table[slot][: -(-n[slot] // case["page"])].astype(np.int64), device="cuda")
        for h in range(case["kv_heads"]):
            k = s["pages"][ids, 0, h].reshape(-1, case["head_dim"])[: n[slot]].double()
            q = s["q"][int(cu[r]):int(cu[r + 1]), h * group:(h + 1) * group].double()
            x = (q @ k.T) * s["scale"]
            first = n[slot] - runs[slot]
            see = torch.arange(n[slot], device="cuda")[None, :] <= first + torch.arange(runs[slot], device="cuda")[:, None]
            x = x.masked_fill(~see[:, None, :], float("-inf"))
            weights[slot, h, : n[slot]] += torch.softmax(x, 2).sum((0, 1))
    return weights


def _prepare_evict(case, seed):
    n, keeps = _contexts(case), _keeps(case)
    b = len(n)
    # without in_place, slot b + s takes what slot s keeps
    rows = n if case["in_place"] else n + keeps
    gen, order, pages, table = _cache(case, seed, rows, len(rows))
    stride = table.shape[1] * case["page"]
    # what attention leaves behind: most keys next to nothing, a few most of it, equal ones where nothing looked
    weights = torch.rand((len(rows), case["kv_heads"], stride), generator=gen, device="cuda") ** 6
    weights = torch.where(weights < 1e-6, torch.zeros_like(weights), weights)
    batch = order.permutation(b)
    state = dict(case=case, pages=pages, scale=1.0, stride=stride, weights=weights, weights_out=torch.zeros_like(weights),
                 kept=torch.zeros((b, case["kv_heads"], max(keeps)), dtype=torch.int32, device="cuda"))
    src = [int(s) for s in batch]
    dst = src if case["in_place"] else [s + b for s in src]
    state.update(src=src, dst=dst, lengths=[n[s] for s in src], keeps=[keeps[s] for s in src],
                 page_ids=torch.tensor(table.astype(np.int64), device="cuda"),
                 src_t=torch.tensor(src, device="cuda"), dst_t=torch.tensor(dst, device="cuda"),
                 len_t=torch.tensor([n[s] for s in src], device="cuda"), keep_t=torch.tensor([keeps[s] for s in src], device="cuda"))
    if own:  # the objects that a serving program keeps
        _gqa_objects(case, state, table, case["kv_heads"], b)
    return state


def _run_evict(s):
    c, kept, out = s["case"], s["kept"], s["weights_out"]
    if own:
        s["gqa"].evict(s["arena"], s["rows"], 0, s["src"], s["dst"], s["lengths"], s["keeps"], c["recent"], s["weights"], out,
                       s["stride"], kept, kept.shape[2])
        return s["pages"], out, kept
    page, heads = c["page"], c["kv_heads"]
    most, keep = max(s["lengths"]), s["keep_t"][:, None, None]
    w = s["weights"][s["src_t"], :, :most]
    at = torch.arange(most, device="cuda")
    length = s["len_t"][:, None, None]
    w = torch.where(at >= length, float("-inf"), torch.where(at >= length - keep.clamp_max(c["recent"]), float("inf"), w))
    order = torch.sort(w, dim=2, descending=True, stable=True).indices
    chosen = torch.where(at < keep, order, most).sort(dim=2).values[:, :, : kept.shape[2]]
    there = (torch.arange(kept.shape[2], device="cuda") < keep).expand_as(kept)
    kept.copy_(torch.where(there, chosen, kept))
    r, h, to = there.nonzero(as_tuple=True)
    come = chosen[r, h, to]
    a = s["page_ids"][s["src_t"][r], come // page]
    b = s["page_ids"][s["dst_t"][r], to // page]
    rows = s["pages"][a, :, h, come % page]
    s["pages"][b, :, h, to % page] = rows
    new = torch.zeros((len(s["src"]), heads, most), device="cuda")
    new[r, h, to] = s["weights"][s["src_t"][r], h, come]
    out[s["dst_t"], :, :most] = torch.where(at < length, new, out[s["dst_t"], :, :most])
    return s["pages"], out, kept


def _exact_evict(case, seed):
    s = _prepare_evict(case, seed)
    weights, out = s["weights"].cpu().numpy().astype(np.float64), s["weights_out"].cpu().numpy().astype(np.float64)
    kept = s["kept"].cpu().numpy()
    for r, (src, dst, n, keep) in enumerate(zip(s["src"], s["dst"], s["lengths"], s["keeps"])):
        recent = min(case["recent"], keep)
        for h in range(case["kv_heads"]):
            w = weights[src, h, : n - recent]
            heavy = np.lexsort((np.arange(n - recent), -w))[: keep - recent]
            rows = np.concatenate([np.sort(heavy), np.arange(n - recent, n)])
            kept[r, h, :keep] = rows
            out[dst, h, :keep], out[dst, h, keep:n] = weights[src, h, rows], 0.0
    return None, torch.from_numpy(out), torch.from_numpy(kept)


def _prepare_linear(case, seed):
    dtype, _ = _TYPES[case["dtype"]]
    runs = _runs(case)
    b, hv, dk, dv = len(runs), case["v_heads"], case["key_dim"], case["value_dim"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 31)).permutation(b)
    runs = [runs[s] for s in order]
    tokens = sum(runs)
    cu = np.concatenate([[0], np.cumsum(runs)]).astype(np.uint32)
    fresh = [i < round(case["fresh"] * b) for i in range(b)]
    slots = [int(s) for s in order]
    outs = [s + b for s in slots] if case["fork"] else slots
    # retention rates from 1 - 2^-5 to 1 - 2^-12 over the heads, drawn within
    rate = torch.rand(hv, generator=gen, device="cuda") * 7 + 5
    decay = torch.log1p(-torch.exp2(-rate))
    state = dict(case=case, scale=dk ** -0.5, decay=decay, tokens=tokens,
                 q=_randn(gen, dtype, tokens, case["k_heads"], dk), k=_randn(gen, dtype, tokens, case["k_heads"], dk),
                 v=_randn(gen, dtype, tokens, hv, dv), out=torch.zeros((tokens, hv, dv), dtype=dtype, device="cuda"),
                 states=torch.randn((2 * b if case["fork"] else b, 1, hv, dk, dv), generator=gen, device="cuda") * 3.0)
    most = max(runs)
    row = cu[:-1, None].astype(np.int64) + np.arange(most)
    live = np.arange(most) < np.array(runs)[:, None]
    state.update(slots=torch.tensor(slots, device="cuda"), outs=torch.tensor(outs, device="cuda"),
                 row=torch.tensor(np.minimum(row, tokens - 1), device="cuda"), live=torch.tensor(live, device="cuda"),
                 flat=torch.tensor(np.flatnonzero(live.reshape(-1)), device="cuda"),
                 run=torch.tensor(runs, device="cuda"), old=torch.tensor([0.0 if f else 1.0 for f in fresh], device="cuda"))
    if own:  # the object and the prepared batch that a serving program keeps
        pkg = _package()
        ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream)
        lin = pkg.LinearAttention(ctx, pkg.LinearConfig(case["k_heads"], hv, dk, dv, dk ** -0.5,
                                                        {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[case["dtype"]],
                                                        state["states"].shape[0], 1, tokens))
        lin.set_decay(0, decay.tolist())
        lin.prepare(slots, [0 if f else 1000 for f in fresh], cu, outs)
        state.update(linear=lin, objects=_Objects(lin, ctx))
    state["host"] = (slots, outs, cu, fresh)
    return state


def _run_linear(s):
    c, states = s["case"], s["states"]
    if own:
        s["linear"].attend(0, states, s["q"], s["k"], s["v"], s["out"])
        return s["out"], states
    share, most = c["v_heads"] // c["k_heads"], s["row"].shape[1]
    live = s["live"][:, None, :, None]
    q, k = (s[x][s["row"]].float().transpose(1, 2).repeat_interleave(share, 1) * live for x in ("q", "k"))
    v = s["v"][s["row"]].float().transpose(1, 2) * live
    i = torch.arange(most, device="cuda")
    back = i[:, None] - i[None, :]
    g = s["decay"][:, None, None]
    old = states[s["slots"], 0] * s["old"][:, None, None, None]
    score = torch.matmul(q, k.transpose(2, 3))
    score *= torch.where(back >= 0, torch.exp(g * back.clamp_min(0)), 0.0)
    out = torch.matmul(score, v) + torch.matmul(q, old) * torch.exp(g * (i[:, None] + 1))
    out = (out * s["scale"]).transpose(1, 2).reshape(-1, c["v_heads"], c["value_dim"])
    s["out"].copy_(out[s["flat"]])
    left = (s["run"][:, None, None] - 1 - i).clamp_min(0)[:, :, :, None]
    new = torch.matmul((k * torch.exp(g * left)).transpose(2, 3), v)
    states[s["outs"], 0] = new + old * torch.exp(g * s["run"][:, None, None, None])
    return s["out"], states


def _exact_linear(case, seed):
    s = _prepare_linear(case, seed)
    slots, outs, cu, fresh = s["host"]
    states = s["states"].double()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    decay = s["decay"].double()
    before, share, chunk = states.clone(), case["v_heads"] // case["k_heads"], 256
    for r in range(len(slots)):
        state = before[slots[r], 0] * (0.0 if fresh[r] else 1.0)
        for at in range(int(cu[r]), int(cu[r + 1]), chunk):
            end = min(at + chunk, int(cu[r + 1]))
            n = end - at
            q, k, v = (s[x][at:end].double().transpose(0, 1) for x in ("q", "k", "v"))
            q, k = q.repeat_interleave(share, 0), k.repeat_interleave(share, 0)
            t = torch.arange(n, device="cuda", dtype=torch.float64)
            rise = torch.exp(decay[:, None] * (t + 1))
            lag = torch.exp(torch.where(t[:, None] >= t[None, :], decay[:, None, None] * (t[:, None] - t[None, :]), float("-inf")))
            out[at:end] = (((q @ k.transpose(1, 2)) * lag) @ v + (q @ state) * rise[:, :, None]).transpose(0, 1) * s["scale"]
            fall = torch.exp(decay[:, None] * (n - 1 - t))
            state = state * torch.exp(decay * n)[:, None, None] + (k * fall[:, :, None]).transpose(1, 2) @ v
        states[outs[r], 0] = state
    return out, states


def prepare(case, seed):
    return {"weigh": _prepare_weigh, "evict": _prepare_evict, "linear": _prepare_linear}[case["op"]](case, seed)


def run(state):
    return {"weigh": _run_weigh, "evict": _run_evict, "linear": _run_linear}[state["case"]["op"]](state)


def exact(case, seed):
    return {"weigh": _exact_weigh, "evict": _exact_evict, "linear": _exact_linear}[case["op"]](case, seed)


def work(case):
    size = _TYPES[case["dtype"]][1]
    if case["op"] == "linear":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["key_dim"], case["value_dim"]
        runs = _runs(case)
        tokens, b = sum(runs), len(runs)
        states = (2 * b - round(case["fresh"] * b)) * hv * dk * dv * 4  # read unless fresh, and written
        return {"bytes": states + tokens * (2 * hk * dk + 2 * hv * dv) * size, "flops": 4.0 * tokens * hv * dk * dv}
    n = _contexts(case)
    heads, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "evict":
        keeps = _keeps(case)
        # every weight is read and its place written, the kept ones' indices come back, their K and V rows are read and written
        return {"bytes": heads * (sum(n) * 8 + sum(keeps) * (4 + 4 * d * size)), "flops": 0}
    runs = _runs(case)
    seen = sum(m * r - r * (r - 1) // 2 for m, r in zip(n, runs))
    return {"bytes": heads * sum(n) * (d * size + 8) + sum(runs) * case["q_heads"] * d * size, "flops": 2.0 * seen * case["q_heads"] * d}
