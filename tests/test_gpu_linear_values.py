"""Linear attention where its arithmetic can go wrong: long prompts in pieces, values that are not finite, the ends of f16's range,
slots that two launches meet in."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype
from test_gpu_linear_attend import DECAYS, EPS, Rig, by_definition, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hk,hv,dk,dv", [(pkg.BF16, 1, 1, 64, 64), (pkg.F16, 1, 2, 128, 64), (pkg.BF16, 1, 1, 96, 128)])
def test_long_prompts_in_pieces(dtype, hk, hv, dk, dv):
    """One or two heads: the run is cut into pieces side by side, into its own slot and into another one."""
    rig = Rig(dtype, hk, hv, dk, dv, slots=6, seed=1, max_tokens=6000)
    rig.set_decay(0, [-2.0 ** -11, -2.0 ** -6][:hv])
    check(rig, [(0, 0, 7, 3001)])
    check(rig, [(1, 2, 7, 2048), (3, 3, 0, 1000), (4, 4, 5, 1), (5, 5, 2, 130)])
    assert rig.lin.device_status() == 0
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_nothing_before_them_nor_beside_them(dtype, bad):
    rig = Rig(dtype, 1, 1, 64, 64, slots=3, seed=2)
    rig.set_decay(0, [-0.05])
    tokens, at, column = 200, 90, 37
    q, k, v = rig.inputs(tokens)
    clean = check(rig, [(0, 1, 3, tokens)], inputs=(q, k, v))
    clean_state = rig.states[1].clone()
    v[at, 0, column] = bad
    out = rig.torch.zeros((tokens, 1, 64), device="cuda").to(torch_dtype(dtype))
    rig.lin.prepare([0], [3], [0, tokens], [1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    got, state = out.double().cpu().numpy(), rig.states[1].cpu().numpy()
    others = [c for c in range(64) if c != column]
    assert (got[:, :, others] == clean[:, :, others]).all() and (got[:at] == clean[:at]).all()
    assert not np.isfinite(got[at:, :, column]).any()
    assert (state[..., others] == clean_state.cpu().numpy()[..., others]).all() and not np.isfinite(state[..., column]).any()
    rig.close()


@pytest.mark.parametrize("which", [0, 1])
def test_a_query_or_key_that_is_not_finite_reaches_nothing_before_it(which):
    rig = Rig(pkg.BF16, 1, 1, 64, 64, slots=3, seed=3)
    tokens, at = 150, 70
    q, k, v = rig.inputs(tokens)
    clean = check(rig, [(0, 1, 3, tokens)], inputs=(q, k, v))
    (q, k)[which][at, 0, 5] = float("nan")
    out = rig.torch.zeros((tokens, 1, 64), device="cuda").bfloat16()
    rig.lin.prepare([0], [3], [0, tokens], [1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    got = out.double().cpu().numpy()
    assert (got[:at] == clean[:at]).all() and np.isnan(got[at]).all()
    if which == 0:
        assert (got[at + 1:] == clean[at + 1:]).all() and rig.torch.isfinite(rig.states[1]).all()
    else:
        assert np.isnan(got[at:]).all()
    rig.close()


def test_what_lies_behind_a_run_does_not_count():
    """The next request's rows hold NaN: nothing of them reaches this request's last chunk."""
    rig = Rig(pkg.F16, 1, 1, 64, 64, slots=4, seed=4)
    q, k, v = rig.inputs(200)
    for x in (q, k, v):
        x[70:] = float("nan")
    out = rig.torch.zeros((200, 1, 64), device="cuda").half()
    rig.lin.prepare([0, 1], [3, 3], [0, 70, 200], None)
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    assert rig.torch.isfinite(out[:70]).all() and rig.torch.isfinite(rig.states[0]).all() and rig.torch.isnan(rig.states[1]).all()
    rig.close()


@pytest.mark.parametrize("size", [60000.0, 200.0, 1e-3, 3e-6])
def test_f16_values_at_the_ends_of_their_range(size):
    """Scores and states far beyond f16's range, and values whose parts are far below its smallest normal number.

    Outputs and states are held to the bounds of every other test; a value below f16's normal range has steps of 2^-24 of
    its own in every part, 2^-36 and less once the low part's scale is taken off."""
    rig = Rig(pkg.F16, 1, 1, 64, 64, slots=2, seed=5, scale=1.0 / 64)
    rig.set_decay(0, [-0.03])
    rig.states.mul_(size)
    q, k, v = rig.inputs(150)
    k, v = (k.float().clamp(-1, 1) * 100).half(), (v.float().clamp(-1, 1) * size).half()
    torch = rig.torch
    out = torch.zeros((150, 1, 64), device="cuda").half()
    before = rig.states.cpu().numpy()
    rig.lin.prepare([0], [1], [0, 150], [1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    want, mag, states, states_mag = by_definition(rig, 0, before, q, k, v, [(0, 1, 1, 150)])
    got, got_states = out.double().cpu().numpy(), rig.states.double().cpu().numpy()
    f32 = 2.0 ** -24
    floor = 100 * 64 * 2.0 ** -36                      # 64 keys of 100 against the smallest steps of the weighted values
    assert (np.abs(got_states - states)[1] <= states_mag[1] * f32 * 700 + floor).all()
    fits = np.abs(want) < 65000.0
    bound = EPS[pkg.F16] * (np.abs(want) + mag) + mag * f32 * 700 + 2.0 ** -25
    assert (np.abs(got - want) <= bound)[fits].all()
    assert np.isinf(got[np.abs(want) > 66000.0]).all() and not np.isnan(got).any()
    rig.close()


def test_recurrent_and_chunked_forms_meet_at_every_length():
    """Runs from one token to just above a chunk, from the same state, in one batch: each is a prefix of the longest."""
    rig = Rig(pkg.BF16, 1, 2, 64, 64, slots=80, seed=6, max_tokens=4096)
    rig.set_decay(0, [-0.01, -0.7])
    q, k, v = rig.inputs(70)
    lengths = list(range(1, 71))
    rows = np.concatenate([np.arange(n) for n in lengths])
    at = rig.torch.from_numpy(rows).cuda()
    out = rig.torch.zeros((len(rows), 2, 64), device="cuda").bfloat16()
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.uint32)
    before = rig.states.cpu().numpy()
    rig.lin.prepare([79] * 70, [4] * 70, cu, list(range(70)))
    rig.lin.attend(0, rig.states, q[at].contiguous(), k[at].contiguous(), v[at].contiguous(), out)
    rig.ctx.sync()
    want, mag, _, _ = by_definition(rig, 0, before, q, k, v, [(79, 0, 4, 70)])
    got, states = out.double().cpu().numpy(), rig.states.double().cpu().numpy()
    for i, n in enumerate(lengths):
        o = got[cu[i]:cu[i + 1]]
        assert (np.abs(o - want[:n]) <= 2 * EPS[pkg.BF16] * mag[:n] + mag[:n] * 2.0 ** -24 * 400).all(), n
        s, m = by_definition(rig, 0, before, q[:n], k[:n], v[:n], [(79, 0, 4, n)])[2:]
        assert (np.abs(states[i] - s[0]) <= m[0] * 2.0 ** -24 * 300).all(), n
    rig.close()


def test_more_heads_than_a_grid_has_rows_are_refused():
    import torch
    ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    with pytest.raises(pkg.PsiError, match="up to 65535 v heads"):
        pkg.LinearAttention(ctx, pkg.LinearConfig(1, 65536, 8, 8, 1.0, pkg.BF16, 1, 1, 1))
    ctx.close()
