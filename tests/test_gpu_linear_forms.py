"""Runs on both sides of the length from which the chunked form is taken, against the recurrence in 64 bits."""
import pytest

from gpuharness import pkg
from test_gpu_linear_attend import DECAYS, Rig, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64), (72, 8)])
def test_runs_next_to_the_border(dtype, dk, dv):
    rig = Rig(dtype, 1, 2, dk, dv, slots=12, seed=dk + dv)
    rig.set_decay(0, DECAYS(2))
    check(rig, [(i, i, i % 2, n) for i, n in enumerate((8, 9, 10, 11, 15, 16, 17, 18))])
    check(rig, [(0, 1, 4, 9), (0, 2, 4, 10), (3, 3, 0, 16), (4, 4, 2, 17), (5, 5, 1, 1)])
    rig.close()


@pytest.mark.parametrize("tokens", [8, 9, 10, 16, 17])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_component_no_larger_than_the_border(dim, tokens):
    rig = Rig(pkg.BF16, 1, 1, dim, dim, slots=2, seed=tokens, max_tokens=tokens)
    check(rig, [(0, 1, 3, tokens)])
    rig.close()


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16, pkg.F32])
@pytest.mark.parametrize("tokens", [1, 12, 130])
def test_an_output_buffer_off_its_boundary(dtype, tokens):
    """The same bits as on a boundary, and nothing beside them."""
    import torch
    rig = Rig(dtype, 1, 2, 64, 72, slots=2, seed=tokens)
    q, k, v = rig.inputs(tokens)
    outs = []
    for offset in (0, 1):
        buffer = torch.full((tokens * 2 * 72 + 2,), 7.0, device="cuda").to(v.dtype)
        out = buffer[offset:offset + tokens * 2 * 72].view(tokens, 2, 72)
        rig.lin.prepare([0], [3], [0, tokens], [1])
        rig.lin.attend(0, rig.states, q, k, v, out)
        rig.ctx.sync()
        assert (buffer[:offset] == 7.0).all() and (buffer[offset + tokens * 2 * 72:] == 7.0).all()
        outs.append(out.clone())
    assert torch.equal(*outs)
    rig.close()
