"""Linear attention behind a value that is not finite: every form keeps it to its column or request, as an infinity or as NaN."""
import numpy as np
import pytest

from gpuharness import pkg, torch_dtype
from test_gpu_linear_attend import Rig

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dk,dv,tokens", [(pkg.F32, 64, 64, 7), (pkg.F32, 72, 40, 100), (pkg.BF16, 72, 40, 3), (pkg.BF16, 256, 136, 20),
                                                (pkg.BF16, 72, 40, 100), (pkg.F16, 128, 128, 100)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_an_infinite_v_stays_in_its_column(dtype, dk, dv, tokens, bad):
    import torch
    rig = Rig(dtype, 1, 2, dk, dv, slots=4, seed=dk, max_tokens=2 * tokens)
    rig.set_decay(0, [-0.1, 0.0])
    q, k, v = rig.inputs(2 * tokens)
    results = []
    for value in (None, bad):
        if value is not None:
            v[1, 1, 9] = value                                           # request 0, its second token, head 1
        states, out = rig.states.clone(), torch.zeros((2 * tokens, 2, dv), device="cuda").to(torch_dtype(dtype))
        rig.lin.prepare([0, 1], [3, 3], [0, tokens, 2 * tokens], [2, 3])
        rig.lin.attend(0, states, q, k, v, out)
        rig.ctx.sync()
        results.append((states, out))
    (s0, o0), (s1, o1) = results
    hit_o, hit_s = torch.zeros(o0.shape, dtype=torch.bool, device="cuda"), torch.zeros(s0.shape, dtype=torch.bool, device="cuda")
    hit_o[1:tokens, 1, 9] = True
    hit_s[2, 0, 1, :, 9] = True
    assert torch.equal(torch.isfinite(o1), ~hit_o) and torch.equal(torch.isfinite(s1), ~hit_s)
    assert torch.equal(o1[~hit_o], o0[~hit_o]) and torch.equal(s1[~hit_s], s0[~hit_s])
    rig.close()
