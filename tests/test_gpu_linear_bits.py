"""Outputs of prompts in 16 bits: what is rounded on the way to them does not show beside their own rounding."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype
from test_gpu_linear_attend import EPS, Rig, by_definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [pkg.BF16, pkg.F16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("index", [0, 9])
def test_a_prompts_outputs_are_off_by_their_own_rounding(dtype, dk, dv, index):
    """With d the error before the last rounding and r that rounding's own, |error| <= |d| + |r|, in the root mean square as well.

    Scores and the state in two parts of 16 bits each, the first towards zero, are off by 2^-15 (bf16: 2^-7 left by the first part,
    half a step of 2^-8 of that by the second) or 2^-21 (f16: 2^-10 and 2^-11) of a term; a sum of terms of either sign by less of itself than its largest term
    is.  The rounding itself is 2^-8 or 2^-11 at most, 2^-10 or 2^-13 in the mean: d is a thirtieth of it, and 5 % is twice that.  One
    part alone would give 1.4 times the rounding."""
    import torch
    rig = Rig(dtype, 1, 3, dk, dv, slots=3, seed=dk + index, max_tokens=512)
    rig.set_decay(0, [-2.0 ** -9, -2.0 ** -5, -0.5])
    tokens = 300
    q, k, v = rig.inputs(tokens)
    before = rig.states.cpu().numpy()
    out = torch.zeros((tokens, 3, dv), device="cuda").to(torch_dtype(dtype))
    rig.lin.prepare([0], [index], [0, tokens], [1])
    rig.lin.attend(0, rig.states, q, k, v, out)
    rig.ctx.sync()
    want, mag, _, _ = by_definition(rig, 0, before, q, k, v, [(0, 1, index, tokens)])
    got = out.double().cpu().numpy()
    rounded = torch.from_numpy(want).to(torch_dtype(dtype)).double().numpy()
    rms = lambda x: np.sqrt((x * x).mean((0, 2)))
    assert (rms(got - want) <= 1.05 * rms(rounded - want)).all(), rms(got - want) / rms(rounded - want)
    parts = {pkg.BF16: 2.0 ** -14, pkg.F16: 2.0 ** -20}[dtype]         # of P and of the state
    bound = EPS[dtype] * np.abs(want) + mag * (parts + 2.0 ** -24 * (4 * tokens + dk + 8)) + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    rig.close()
