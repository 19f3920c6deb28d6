"""Eviction of rows that no cluster's shared memory holds (above 393,216 keys)."""
import pytest

from gpuharness import pkg
from memory_rig import Cache
from test_gpu_evict import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dst", [0, 1])
@pytest.mark.parametrize("same_buffer", [False, True])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_rows_of_four_hundred_thousand_keys(dst, same_buffer, kind):
    import torch
    n = 400003
    cache = Cache(pkg.BF16, 1, 1, 8, 16, n, 3, seed=dst)
    w = torch.rand((3, 1, cache.capacity), generator=cache.gen, device="cuda")
    if kind == "ties":
        w = torch.floor(w * 3.0)
    elif kind == "odd":
        values = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-45, 3.4e38], device="cuda")
        w[:, :, ::2] = values[torch.randint(0, 7, w[:, :, ::2].shape, device="cuda", generator=cache.gen)]
    # beside a short row, which takes the same launch
    check(cache, [0, 2], [dst, 2], [n, 37], [200001, 20], 64, weights=w.clone(), same_buffer=same_buffer)
    check(cache, [0], [dst], [n - 2], [n - 3], 0, weights=w.clone(), same_buffer=same_buffer)
    cache.close()
