"""Worker of tests/test_gpu_bounded_memory.py: the kernels of key weights and eviction in the bounds-checked build
(PSI_CUDA_LIBRARY=checked, a process of its own), with a page table that holds an ID beyond the arena's declared pages.

As in checked_build_worker.py the arena declares half the pages that its buffer holds and the bad ID lies in the other half: the
access that a check must skip would have stayed inside the buffer."""
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))
sys.path.insert(0, str(ROOT / "tests"))

import torch

import __graft_entry__ as entry

pkg = entry.load_package()
PSI_ERR_PAGE_ID = 6
HQ, HKV, PAGE, DECLARED = 4, 2, 16, 24
GOOD, BAD = list(range(8)), [0, 1, DECLARED + 3, 3, 4, 5, 6, 7]


def component(dtype, d):
    tdtype = {pkg.F32: torch.float32, pkg.BF16: torch.bfloat16}[dtype]
    esz = 4 if dtype == pkg.F32 else 2
    buffer = torch.randn((2 * DECLARED, 2 * HKV * PAGE * d), device="cuda:0").to(tdtype)
    ctx = pkg.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    page_bytes = 2 * HKV * PAGE * d * esz
    pages = pkg.PageArena(ctx, DECLARED, page_bytes, device_ptr=buffer)
    layout = pkg.GQAPageTableLayout(2, 1, 8, 1)
    table = pkg.GQARequestPageTable(ctx, layout)
    gqa = pkg.GQA(ctx, pkg.GQAConfig(HQ, HKV, d, 0.1, page_bytes, dtype, layout, 128, pkg.PLAN_BALANCED, pkg.KERNEL_AUTO, 0))
    table.write_row(1, 0, list(range(8, 16)))
    return buffer, ctx, pages, table, gqa


def weigh(dtype, d, run):
    buffer, ctx, pages, table, gqa = component(dtype, d)
    q = torch.randn((run, HQ, d), device="cuda:0").to(buffer.dtype)
    results = []
    for row, status in ((BAD, PSI_ERR_PAGE_ID), (GOOD, 0)):
        table.write_row(0, 0, row)
        weights = torch.zeros((2, HKV, 128), device="cuda:0")
        gqa.prepare([0], [128 - run], [0, run])
        gqa.weigh_keys(pages, table, 0, q, weights, 128)
        assert gqa.device_status() == status, (dtype, d, run, row)
        assert bool((weights[1] == 0).all())
        results.append(weights)
    assert not torch.equal(*results)
    for x in (gqa, table, pages, ctx):
        x.close()


def evict(dtype, d, dst):
    buffer, ctx, pages, table, gqa = component(dtype, d)
    weights = torch.zeros((2, HKV, 128), device="cuda:0")
    weights[0, :, 40:] = 1.0                              # the first 40 keys go: rows move across the bad page
    kept = torch.zeros((1, HKV, 88), dtype=torch.int32, device="cuda:0")
    table.write_row(0, 0, BAD)
    before = buffer.clone()
    gqa.evict(pages, table, 0, [0], [dst], [128], [88], 4, weights, weights.clone(), 128, kept, 88)
    assert gqa.device_status() == PSI_ERR_PAGE_ID
    assert torch.equal(kept.cpu(), torch.arange(40, 128, dtype=torch.int32).expand(1, HKV, 88))
    assert torch.equal(buffer[DECLARED:], before[DECLARED:])           # nothing beyond the declared pages
    view, old = buffer.view(-1, 2, HKV, PAGE, d), before.view(-1, 2, HKV, PAGE, d)
    where = GOOD if dst == 0 else list(range(8, 16))
    for to in range(88):
        source, target = 40 + to, to
        if BAD[source // PAGE] >= DECLARED or (dst == 0 and BAD[target // PAGE] >= DECLARED):
            continue
        assert torch.equal(view[where[target // PAGE], :, :, target % PAGE], old[BAD[source // PAGE], :, :, source % PAGE]), to
    for to in range(88):                                              # a row whose source is bad keeps what it held
        if dst == 1 and BAD[(40 + to) // PAGE] >= DECLARED:
            assert torch.equal(view[where[to // PAGE], :, :, to % PAGE], old[where[to // PAGE], :, :, to % PAGE]), to
    table.write_row(0, 0, GOOD)
    gqa.evict(pages, table, 0, [0], [dst], [128], [88], 4, weights, weights.clone(), 128, kept, 88)
    assert gqa.device_status() == 0
    for x in (gqa, table, pages, ctx):
        x.close()


def main():
    assert pkg.library_path().name == "libpsi_cuda_checked.so", pkg.library_path()
    for dtype, d, run in ((pkg.BF16, 128, 1), (pkg.BF16, 128, 96), (pkg.F32, 128, 2), (pkg.F32, 20, 96), (pkg.BF16, 20, 5)):
        weigh(dtype, d, run)
    for dtype, d in ((pkg.BF16, 128), (pkg.F32, 128), (pkg.BF16, 10), (pkg.BF16, 11)):
        for dst in (0, 1):
            evict(dtype, d, dst)
    print("checked memory ok")


if __name__ == "__main__":
    main()
