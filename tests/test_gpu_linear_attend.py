"""Linear attention with a decay for each head (LinearAttention) against its recurrence in 64 bits."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype

pytestmark = pytest.mark.gpu

EPS = {pkg.F32: 2.0 ** -24, pkg.BF16: 2.0 ** -8, pkg.F16: 2.0 ** -11}   # half a step, relative


class Rig:
    def __init__(self, dtype, hk, hv, dk, dv, slots=4, layers=1, max_tokens=2048, scale=None, seed=0, stream=None):
        import torch
        self.torch, self.dtype, self.hk, self.hv, self.dk, self.dv, self.slots, self.layers = torch, dtype, hk, hv, dk, dv, slots, layers
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.scale = dk ** -0.5 if scale is None else scale
        self.ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
        self.lin = pkg.LinearAttention(self.ctx, pkg.LinearConfig(hk, hv, dk, dv, self.scale, dtype, slots, layers, max_tokens))
        self.decay = np.zeros((layers, hv), np.float32)
        self.states = torch.randn((slots, layers, hv, dk, dv), generator=self.gen, device="cuda") * 2.0

    def set_decay(self, layer, values):
        self.decay[layer] = np.asarray(values, np.float32)
        self.lin.set_decay(layer, self.decay[layer])

    def randn(self, *shape):
        return self.torch.randn(shape, generator=self.gen, device="cuda").to(torch_dtype(self.dtype))

    def inputs(self, tokens):
        return self.randn(tokens, self.hk, self.dk), self.randn(tokens, self.hk, self.dk), self.randn(tokens, self.hv, self.dv)

    def close(self):
        self.ctx.sync()
        self.lin.close()
        self.ctx.close()


def by_definition(rig, layer, states, q, k, v, batch):
    """(out, its magnitude, states, their magnitude): the magnitudes are the same sums over absolute values."""
    f = lambda t: t.double().cpu().numpy()
    q, k, v, old = f(q), f(k), f(v), states.astype(np.float64)
    new, new_mag = old.copy(), np.abs(old)
    out, mag = np.zeros(v.shape), np.zeros(v.shape)
    share, at = rig.hv // rig.hk, 0
    lam = np.exp(rig.decay[layer].astype(np.float64))[:, None, None]
    for src, dst, index, run in batch:
        s = old[src, layer].copy() if index > 0 else np.zeros((rig.hv, rig.dk, rig.dv))
        m = np.abs(s)
        for t in range(at, at + run):
            kk, qq = np.repeat(k[t], share, 0), np.repeat(q[t], share, 0)
            s = lam * s + kk[:, :, None] * v[t][:, None, :]
            m = lam * m + np.abs(kk)[:, :, None] * np.abs(v[t])[:, None, :]
            out[t] = (qq[:, :, None] * s).sum(1) * rig.scale
            mag[t] = (np.abs(qq)[:, :, None] * m).sum(1) * rig.scale
        at += run
        if run > 0:
            new[dst, layer], new_mag[dst, layer] = s, m
    return out, mag, new, new_mag


def check(rig, batch, layer=0, inputs=None):
    """`batch`: (slot, slot of the new state, token index, tokens).

    f32 sums of n terms are off by at most n half steps of the sum of their magnitudes: the state has a term for each token, an
    output a term for each row of the state on top, each with a handful of roundings.  Prompts in 16 bits hold the
    state and the scores of a chunk in one rounding of at most half a bf16 or f16 step for the output alone; the output is rounded once more."""
    torch = rig.torch
    tokens = sum(n for _, _, _, n in batch)
    q, k, v = rig.inputs(tokens) if inputs is None else inputs
    out = torch.full((tokens + 2, rig.hv, rig.dv), 77.0, device="cuda").to(torch_dtype(rig.dtype))
    before = rig.states.cpu().numpy()
    cu = np.concatenate([[0], np.cumsum([n for _, _, _, n in batch])]).astype(np.uint32)
    rig.lin.prepare([s for s, _, _, _ in batch], [i for _, _, i, _ in batch], cu, [d for _, d, _, _ in batch])
    rig.lin.attend(layer, rig.states, q, k, v, out)
    rig.ctx.sync()
    want, mag, states, states_mag = by_definition(rig, layer, before, q, k, v, batch)
    got, got_states = out.double().cpu().numpy(), rig.states.double().cpu().numpy()
    most = max(n for _, _, _, n in batch)
    f32 = 2.0 ** -24
    bound = EPS[rig.dtype] * np.abs(want) + mag * f32 * (4 * most + rig.dk + 8) + 1e-30
    if rig.dtype != pkg.F32:
        bound += mag * EPS[rig.dtype]
    assert (np.abs(got[:tokens] - want) <= bound).all(), float((np.abs(got[:tokens] - want) / bound).max())
    assert (got[tokens:] == 77.0).all()
    written = np.zeros(got_states.shape, bool)
    for src, dst, index, n in batch:
        if n > 0:
            written[dst, layer] = True
    assert (got_states[~written] == before[~written]).all()
    off, bound = np.abs(got_states - states), states_mag * f32 * (4 * most + 8) + 1e-30
    assert (off <= bound)[written].all(), float((off / bound)[written].max())
    return got[:tokens]


DECAYS = lambda n, seed=0: -np.exp2(-np.random.default_rng(seed).uniform(0, 12, n)).astype(np.float32)


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16, pkg.F32])
@pytest.mark.parametrize("hk,hv,dk,dv", [(1, 1, 128, 128), (2, 4, 64, 64), (3, 3, 64, 128), (2, 2, 128, 64), (1, 2, 96, 80), (1, 1, 8, 8), (1, 1, 256, 256),
                                         (2, 6, 16, 40)])
def test_every_run_length(dtype, hk, hv, dk, dv):
    rig = Rig(dtype, hk, hv, dk, dv, slots=12, layers=2, seed=dk + dv)
    rig.set_decay(1, DECAYS(hv))
    check(rig, [(0, 0, 5, 1), (3, 3, 0, 2), (1, 1, 9, 8), (2, 2, 1, 9), (4, 4, 3, 0), (5, 5, 70, 64), (6, 7, 2, 65), (9, 9, 0, 200)], layer=1)
    check(rig, [(11, 10, 1, 1)], layer=1)
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_no_decay_strong_decay_and_a_decay_next_to_one(dtype):
    rig = Rig(dtype, 1, 6, 64, 64, seed=1)
    rig.set_decay(0, [0.0, -1e-7, -2.0 ** -12, -3.0, -40.0, -1e30])
    check(rig, [(0, 0, 1, 1), (1, 1, 1, 300), (2, 3, 0, 129)])
    rig.close()


def test_a_long_prompt_does_not_drift():
    rig = Rig(pkg.F32, 1, 2, 32, 32, seed=2, max_tokens=4096)
    rig.set_decay(0, [-2.0 ** -12, -2.0 ** -9])
    check(rig, [(0, 0, 1, 4096)])
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16, pkg.F32])
def test_a_prompt_in_pieces_is_the_prompt(dtype):
    """Chunks of a prompt and single tokens behind them go through the same states as the whole prompt."""
    import torch
    rig = Rig(dtype, 1, 2, 64, 64, slots=2, seed=3)
    rig.set_decay(0, [-0.01, -0.3])
    q, k, v = rig.inputs(150)
    outs = []
    for begin, end in [(0, 70), (70, 71), (71, 140), (140, 141), (141, 150)]:
        outs.append(check(rig, [(0, 0, begin, end - begin)], inputs=(q[begin:end], k[begin:end], v[begin:end])))
    whole = check(rig, [(1, 1, 0, 150)], inputs=(q, k, v))
    _, mag, _, _ = by_definition(rig, 0, rig.states.cpu().numpy(), q, k, v, [(1, 1, 0, 150)])
    assert (np.abs(np.concatenate(outs) - whole) <= 4 * EPS[dtype] * mag + 2.0 ** -24 * 2000 * mag).all()
    rig.close()


def test_a_fresh_request_reads_nothing_of_its_slot():
    rig = Rig(pkg.BF16, 1, 1, 64, 64, seed=4)
    rig.states.fill_(float("nan"))
    rig.lin.prepare([0, 1], [0, 0], [0, 1, 100], None)
    q, k, v = rig.inputs(100)
    out = rig.torch.zeros((100, 1, 64), device="cuda").bfloat16()
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    assert rig.torch.isfinite(out.float()).all() and rig.torch.isfinite(rig.states[:2]).all() and rig.torch.isnan(rig.states[2:]).all()
    rig.close()


def test_one_state_read_by_many_requests():
    rig = Rig(pkg.F16, 2, 2, 64, 64, slots=6, seed=5)
    rig.set_decay(0, [-0.1, -0.2])
    check(rig, [(0, 1, 7, 3), (0, 2, 7, 1), (0, 3, 7, 80)])
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_buffers_off_their_boundaries(dtype):
    rig = Rig(dtype, 1, 1, 64, 64, seed=6)
    rig.set_decay(0, [-0.05])
    make = lambda t: rig.torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)
    q, k, v = rig.inputs(90)
    check(rig, [(0, 0, 4, 1), (1, 1, 4, 89)], inputs=(make(q), make(k), make(v)))
    rig.close()


def test_the_same_call_gives_the_same_bits():
    rig = Rig(pkg.BF16, 2, 4, 128, 128, slots=8, seed=7)
    rig.set_decay(0, DECAYS(4))
    inputs = rig.inputs(700)
    batch = [(0, 4, 3, 1), (1, 5, 3, 6), (2, 6, 3, 693)]
    once = check(rig, batch, inputs=inputs)
    states = rig.states.clone()
    again = check(rig, batch, inputs=inputs)
    assert (once == again).all() and rig.torch.equal(states, rig.states)
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F32])
def test_captured_launches_follow_the_batch(dtype):
    import torch
    side = torch.cuda.Stream()
    rig = Rig(dtype, 1, 2, 64, 64, slots=4, seed=8, max_tokens=300, stream=side.cuda_stream)
    rig.set_decay(0, [-0.02, -0.5])
    q, k, v = rig.inputs(300)
    out = torch.zeros((300, 2, 64), device="cuda").to(torch_dtype(dtype))
    torch.cuda.synchronize()
    rig.lin.prepare([0], [1], [0, 1])
    rig.ctx.capture_begin()
    with pytest.raises(pkg.PsiError, match="stays outside captured graphs"):
        rig.lin.prepare([0], [1], [0, 1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    graph = rig.ctx.capture_end()
    for batch in ([(0, 0, 5, 1)], [(1, 1, 0, 150), (2, 3, 9, 2)], [(0, 0, 6, 300)], [(3, 3, 1, 1), (2, 2, 1, 1), (1, 1, 1, 1)]):
        before = rig.states.cpu().numpy()
        cu = np.concatenate([[0], np.cumsum([n for _, _, _, n in batch])]).astype(np.uint32)
        rig.lin.prepare([s for s, _, _, _ in batch], [i for _, _, i, _ in batch], cu, [d for _, d, _, _ in batch])
        graph.launch()
        rig.ctx.sync()
        n = int(cu[-1])
        want, mag, states, states_mag = by_definition(rig, 0, before, q[:n], k[:n], v[:n], batch)
        got = out.double().cpu().numpy()[:n]
        assert (np.abs(got - want) <= 2 * EPS[dtype] * mag + mag * 2.0 ** -24 * 1500).all()
        assert (np.abs(rig.states.double().cpu().numpy() - states) <= states_mag * 2.0 ** -24 * 1300 + 1e-30).all()
    graph.close()
    rig.close()


def test_refusals():
    import torch
    ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    good = dict(hk=2, hv=4, dk=64, dv=64, scale=0.1, dtype=pkg.BF16, slots=4, layers=2, tokens=16)

    def make(**kw):
        a = dict(good, **kw)
        return pkg.LinearAttention(ctx, pkg.LinearConfig(a["hk"], a["hv"], a["dk"], a["dv"], a["scale"], a["dtype"], a["slots"], a["layers"], a["tokens"]))

    for kw, words in [(dict(hk=0), "head counts"), (dict(hv=3), "multiple of k heads"), (dict(dk=12), "multiples of 8"), (dict(dv=264), "multiples of 8"),
                      (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(dtype=7), "dtype"), (dict(slots=0), "must be positive"),
                      (dict(tokens=1 << 31), "work counts")]:
        with pytest.raises(pkg.PsiError, match=words):
            make(**kw)
    lin = make()
    states = torch.zeros((4, 2, 4, 64, 64), device="cuda")
    q = torch.zeros((16, 2, 64), device="cuda").bfloat16()
    v = torch.zeros((16, 4, 64), device="cuda").bfloat16()
    with pytest.raises(pkg.PsiError, match="must be prepared"):
        lin.attend(0, states, q, q, v, v)
    for layer, values, words in [(2, [0.0] * 4, "layer out of range"), (0, [0.0, 0.0, 0.1, 0.0], "not positive"), (0, [float("-inf")] * 4, "finite"),
                                 (0, [0.0], "num_v_heads values")]:
        with pytest.raises(pkg.PsiError, match=words):
            lin.set_decay(layer, values)
    for args, words in [(([], [], [0]), "requires tokens"), (([0], [0], [0, 0]), "requires tokens"), (([0], [0], [1, 2]), "start at zero"),
                        (([0, 1], [0, 0], [0, 3, 2]), "nondecreasing"), (([0], [0], [0, 17]), "token capacity"), (([4], [0], [0, 1]), "out of range"),
                        (([0], [0], [0, 1], [4]), "out of range"), (([0, 0], [1, 1], [0, 1, 2]), "state of one slot"),
                        (([0, 1], [1, 1], [0, 1, 2], [2, 2]), "state of one slot"), (([0, 1], [1, 1], [0, 1, 2], [1, 2]), "another one reads"),
                        (([0, 1], [1], [0, 1, 2]), "lengths disagree")]:
        with pytest.raises(pkg.PsiError, match=words):
            lin.prepare(*args)
    lin.prepare([0, 1], [1, 0], [0, 1, 2], [1, 2])     # request 1 starts afresh: it reads no state
    for i in range(5):
        buffers = [states, q, q, v, v]
        buffers[i] = None
        with pytest.raises(pkg.PsiError, match="not be null"):
            lin.attend(0, *buffers)
    with pytest.raises(pkg.PsiError, match="layer out of range"):
        lin.attend(2, states, q, q, v, v)
    with pytest.raises(pkg.PsiError, match="16-byte aligned"):
        lin.attend(0, states.data_ptr() + 4, q, q, v, v)
    with pytest.raises(pkg.PsiError, match="aligned to their elements"):
        lin.attend(0, states, q.data_ptr() + 1, q, v, v)
    lin.close()
    ctx.close()
