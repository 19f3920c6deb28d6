"""Chunked linear attention in the first chunk of a run: values that are not finite, and what lies behind a run of less than a chunk."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype
from test_gpu_linear_attend import Rig

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def attend(rig, slots, outs, indices, lengths, q, k, v):
    """(outputs, states) of one step from the rig's states, which stay as they were."""
    torch = rig.torch
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.uint32)
    states = rig.states.clone()
    out = torch.zeros((int(cu[-1]), rig.hv, rig.dv), device="cuda").to(torch_dtype(rig.dtype))
    torch.cuda.synchronize()
    rig.lin.prepare(slots, indices, cu, outs)
    rig.lin.attend(0, states, q, k, v, out)
    rig.ctx.sync()
    assert rig.lin.device_status() == 0
    return out, states


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("tokens,at", [(9, 0), (40, 5), (63, 62), (64, 1), (64, 63), (200, 5), (200, 31), (200, 63)])
def test_a_value_that_is_not_finite_in_a_runs_first_chunk(dtype, bad, tokens, at):
    """More (request, head) items than SMs: an item that is its CTA's first and one that is not."""
    import torch
    n, heads, column = 48, 4, 37
    rig = Rig(dtype, 2, heads, 64, 64, slots=2 * n, seed=tokens + at, max_tokens=n * tokens)
    rig.set_decay(0, [-0.05, -0.3, 0.0, -0.01])
    q, k, v = rig.inputs(n * tokens)
    slots, outs, indices, lengths = list(range(n)), list(range(n, 2 * n)), [3] * n, [tokens] * n
    clean, clean_states = attend(rig, slots, outs, indices, lengths, q, k, v)
    v.view(n, tokens, heads, 64)[:, at, :, column] = bad
    for _ in range(3):
        got, states = attend(rig, slots, outs, indices, lengths, q, k, v)
        a, b = got.view(n, tokens, heads, 64), clean.view(n, tokens, heads, 64)
        others = [c for c in range(64) if c != column]
        assert torch.equal(a[..., others], b[..., others]) and torch.equal(a[:, :at], b[:, :at])
        assert not torch.isfinite(a[:, at:, :, column]).any()
        assert torch.equal(states[..., others], clean_states[..., others])
        assert not torch.isfinite(states[n:, :, :, :, column]).any()
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
@pytest.mark.parametrize("tokens", [9, 20, 33, 63])
def test_a_neighbour_of_nan_rows_does_not_reach_a_short_run(dtype, tokens):
    import torch
    n, heads = 40, 4
    rig = Rig(dtype, 2, heads, 128, 128, slots=2 * n, seed=tokens, max_tokens=2 * n * tokens)
    rig.set_decay(0, [-0.05, -0.3, 0.0, -0.01])
    q, k, v = rig.inputs(2 * n * tokens)
    slots, indices, lengths = list(range(2 * n)), [3, 0] * n, [tokens] * (2 * n)
    clean, clean_states = attend(rig, slots, None, indices, lengths, q, k, v)
    for x in (q, k, v):
        x.view(n, 2, tokens, *x.shape[1:])[:, 1] = NAN
    for _ in range(3):
        got, states = attend(rig, slots, None, indices, lengths, q, k, v)
        a, b = got.view(n, 2, tokens, heads, 128), clean.view(n, 2, tokens, heads, 128)
        assert torch.equal(a[:, 0], b[:, 0]) and torch.isnan(a[:, 1]).all()
        assert torch.equal(states[0::2], clean_states[0::2]) and torch.isnan(states[1::2]).all()
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
def test_values_that_are_not_finite_in_the_pieces_of_a_long_run(dtype):
    """Chunk c of the run holds one in column c, at its sixth token: so does the first chunk of every piece."""
    import torch
    tokens = 60 * 64 + 20
    rig = Rig(dtype, 1, 1, 64, 64, slots=2, seed=1, max_tokens=tokens)
    rig.set_decay(0, [-0.01])
    q, k, v = rig.inputs(tokens)
    clean, _ = attend(rig, [0], [1], [5], [tokens], q, k, v)
    for c in range(60):
        v[64 * c + 5, 0, c] = (NAN, INF, -INF)[c % 3]
    got, states = attend(rig, [0], [1], [5], [tokens], q, k, v)
    for c in range(64):
        at = 64 * c + 5 if c < 60 else tokens
        assert torch.equal(got[:at, 0, c], clean[:at, 0, c]), c
        assert not torch.isfinite(got[at:, 0, c]).any(), c
        assert bool(torch.isfinite(states[1, 0, 0, :, c]).any()) == (c >= 60), c
    rig.close()


@pytest.mark.parametrize("tokens", [9, 20, 63, 100])
def test_what_the_buffers_hold_behind_a_replayed_batch_does_not_count(tokens):
    import torch
    side = torch.cuda.Stream()
    rig = Rig(pkg.BF16, 1, 2, 64, 64, slots=4, seed=2, max_tokens=300, stream=side.cuda_stream)
    rig.set_decay(0, [-0.02, -0.5])
    q, k, v = rig.inputs(300)
    torch.cuda.synchronize()
    clean, clean_states = attend(rig, [0], [1], [7], [tokens], q[:tokens].contiguous(), k[:tokens].contiguous(), v[:tokens].contiguous())
    for x in (q, k, v):
        x[tokens:] = NAN
    out, states = torch.full((300, 2, 64), 5.0, device="cuda").bfloat16(), rig.states.clone()
    torch.cuda.synchronize()
    rig.ctx.capture_begin()
    rig.lin.attend(0, states, q, k, v, out)
    graph = rig.ctx.capture_end()
    for _ in range(3):
        states.copy_(rig.states)
        torch.cuda.synchronize()
        graph.launch()
        rig.ctx.sync()
        assert torch.equal(out[:tokens], clean) and (out[tokens:] == 5.0).all() and torch.equal(states, clean_states)
    graph.close()
    rig.close()
