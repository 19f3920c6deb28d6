"""Key weights with infinite scores, against the definition: a key at -inf gets nothing, a row that sees +inf adds nothing."""
import numpy as np
import pytest

from gpuharness import pkg
from memory_rig import Cache
from test_gpu_weigh_keys import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(pkg.BF16, 64), (pkg.F16, 128), (pkg.F32, 64), (pkg.BF16, 36)])
@pytest.mark.parametrize("tokens", [1, 6, 30, 150])
def test_infinite_scores(dtype, d, tokens):
    cache = Cache(dtype, 4, 2, d, 16, 400, 2, seed=tokens)
    first = 200
    q = cache.randn(tokens, 4, d).abs() + 0.25                            # an infinity in K is one of the same sign in every score
    row = np.full(d, 0.25, np.float32)
    row[1] = -np.inf
    for token in (3, 150, first):                                         # some rows' own key as well
        cache.set_row(0, 0, 0, token, row)
    plus = row.copy()
    plus[1] = np.inf
    if tokens > 4:
        cache.set_row(0, 0, 1, first + 4, plus)                           # the KV head's rows from token 4 on add nothing, those before do
    got = check(cache, [(0, first, tokens)], q=q, weights=cache.torch.zeros((2, 2, cache.capacity), device="cuda"))
    assert (got[0, 0, [3, 150, first]] == 0.0).all() and got[0, 0, 4] > 0.0
    assert got[0, 1, 0] > 0.0
    rows = 2 * min(tokens, 4)
    if tokens > 4:
        assert abs(got[0, 1].sum() - rows) <= 1e-3 * rows                  # a row's weights add up to one
        assert (got[0, 1, first + 4:] == 0.0).all()
    cache.close()
