"""Every form in which mf_adapter_apply's two launches run, against the exact results: the cases are picked by the rules of adapters.hip, which stand
here once more as plain arithmetic, so that a case that no longer reaches the form it is named for fails on the CPU.

Whole numbers as in test_gpu_adapters.py: every product and sum is exact in fp32, the results are compared bit for bit."""
from __future__ import annotations

import pytest
import torch

from test_gpu_adapters import Case, make_ids


def form(t, n, ms, adapters, rank, plan):
    """(rows of 16 a workgroup, blocks of ranks a workgroup of the first launch, parts of the sum over n), or None for the one launch"""
    if rank <= 32 and (rank + 16) * n * 2 <= 512 << 10 and sum(ms) * t <= 16 << 20:
        return None
    wide = t // 32 >= adapters if plan else t > 256
    per = (rank + 15) // 16
    blocks = per * len(ms)
    everything = t > 256 and blocks <= 2
    least = 2 if t > 256 and (t + 31) // 32 * ((blocks + 1) // 2) >= 256 else 1
    parts = max(1, min(512 * (2 if everything else 1) // ((t + 15) // 16), n // 64 // (8 * least), 16 if t <= 256 else 8 if everything else 4))
    return 2 if wide else 1, min(blocks, 2), parts


# t, n, ms, adapters, rank, order, plan, what runs
CASES = [
    # 16 rows, two blocks of ranks, several parts of n
    (1, 5120, (72, 72), 4, 64, "one", False, (1, 2, 10)),
    (1, 8192, (40,), 2, 256, "one", False, (1, 2, 16)),
    (7, 17408, (24, 40), 3, 16, "mixed", False, (1, 2, 16)),
    (100, 2048, (130, 66), 6, 48, "mixed", False, (1, 2, 4)),
    (100, 2048, (130, 66), 6, 48, "mixed", True, (1, 2, 4)),
    (200, 4096, (96, 96, 96), 48, 40, "mixed", True, (1, 2, 8)),
    (200, 4096, (96, 96, 96), 48, 40, "runs", False, (1, 2, 8)),
    (256, 1088, (33, 8, 64, 40), 3, 72, "runs", False, (1, 2, 2)),
    (400, 2112, (72,), 100, 40, "mixed", True, (1, 2, 4)),
    # 16 rows, one block
    (8, 17408, (96,), 3, 16, "mixed", False, (1, 1, 16)),
    (130, 16448, (72,), 40, 8, "mixed", True, (1, 1, 16)),
    # 32 rows, one block and several parts; two that a workgroup has all of
    (300, 8768, (64,), 3, 16, "runs", False, (2, 1, 8)),
    (300, 8768, (64,), 3, 16, "mixed", True, (2, 1, 8)),
    (600, 12032, (64, 64), 3, 16, "runs", False, (2, 2, 8)),
    (600, 12032, (64, 64), 3, 16, "mixed", True, (2, 2, 8)),
    (300, 8768, (200,), 3, 16, "runs", False, (2, 1, 8)),
    (517, 6656, (136, 65), 5, 24, "mixed", True, (2, 2, 4)),
    (517, 6656, (136, 65), 5, 24, "runs", False, (2, 2, 4)),
    # 32 rows, more blocks than a workgroup has; two units a wave at least
    (777, 2048, (96, 40), 5, 64, "runs", False, (2, 2, 4)),
    (2100, 2112, (40, 40), 3, 128, "runs", False, (2, 2, 2)),
    (2100, 2112, (40, 40), 3, 128, "mixed", True, (2, 2, 2)),
    # ranks and sizes of the one launch, but too many results for it
    (1000, 128, (16840,), 3, 16, "runs", False, (2, 1, 1)),
    (1000, 128, (16840,), 3, 16, "mixed", True, (2, 1, 1)),
]


@pytest.mark.parametrize("t, n, ms, adapters, rank, order, plan, runs", CASES)
def test_the_form_that_a_case_is_named_for(t, n, ms, adapters, rank, order, plan, runs):
    assert form(t, n, ms, adapters, rank, plan) == runs


@pytest.mark.gpu
@pytest.mark.parametrize("ranks", ["full", "mixed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, n, ms, adapters, rank, order, plan, runs", CASES)
def test_whole_numbers(gpu, t, n, ms, adapters, rank, order, plan, runs, dtype, ranks):
    c = Case(t, n, ms, adapters, rank, dtype=dtype, ranks=ranks, seed=t + rank)
    c.check(gpu, make_ids(order, t, adapters, 0.1 if ranks == "mixed" else 0.0, seed=t), plan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, n, ms, adapters, rank, order, plan, runs", CASES[::2])
def test_normal_numbers(gpu, t, n, ms, adapters, rank, order, plan, runs, dtype):
    c = Case(t, n, ms, adapters, rank, whole=False, dtype=dtype, ranks="mixed", seed=t)
    c.check(gpu, make_ids(order, t, adapters, 0.1, seed=t), plan, whole=False)


@pytest.mark.gpu
@pytest.mark.parametrize("t, adapters, rank, n", [(40, 3, 16, 128), (300, 5, 64, 192), (90, 20, 40, 640), (5000, 7, 16, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_plan_that_was_made_for_other_sizes_is_not_used(gpu, t, adapters, rank, n, dtype):
    """words with room for the call's plan that hold zeros, or the plan of fewer rows or of another number of adapters: the rows are taken as
    they lie"""
    from mference_amd import operators as ops
    c = Case(t, n, (72,), adapters, rank, dtype=dtype, seed=t)
    ids = make_ids("mixed", t, adapters, 0.2, seed=t)
    want, live = c.expected(ids)
    base = c.ys[0].clone()
    op = ops.LowRankAdapters(gpu, c.a, c.b, scales=c.scales)
    room = ops.AdapterGrouping(gpu, adapters).plan(t).words
    stale = [None, (t - 1, adapters), (t, adapters + 1), (t // 2, adapters)]
    for other in stale:
        words = torch.zeros(4 * room.numel() + 4096, dtype=torch.int32, device="cuda")
        if other:
            g = ops.AdapterGrouping(gpu, other[1])
            g.encode(make_ids("mixed", other[0], other[1], seed=3), ops.AdapterPlan(*other, words))
        c.ys[0].copy_(base)
        op.encode(c.x, ids, c.ys, plan=ops.AdapterPlan(t, adapters, words))
        assert torch.equal(c.ys[0][live], want[0][0][live].to(dtype)), other
        assert torch.equal(c.ys[0][~live], base[~live]), other
