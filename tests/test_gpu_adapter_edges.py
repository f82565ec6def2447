"""mf_adapter_apply on the GPU where its arguments end."""
from __future__ import annotations

import pytest
import torch

from mference_amd import operators as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t, n, rank", [(9, 128, 16), (40, 256, 24), (300, 192, 64), (70, 64, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [False, True])
def test_ranks_beyond_both_ends(gpu, t, n, rank, dtype, plan):
    """a rank below zero is none: the rows keep their bits, whatever the pool holds; one past the pool's counts as the pool's.  Whole numbers:
    |A x| <= 4 n and |B A x| <= 4 n rank < 2^24, so the results are exact, and correctly rounded."""
    g = torch.Generator(device="cuda")
    g.manual_seed(t)
    ints = lambda k, *s: torch.randint(-k, k + 1, s, generator=g, device="cuda").float()  # noqa: E731
    a, b, x = ints(2, 5, rank, n).bfloat16(), ints(1, 5, 72, rank).bfloat16(), ints(2, t, n).bfloat16()
    ranks = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31, rank + 1, -rank], dtype=torch.int32, device="cuda")
    for k in (0, 2, 4):
        a[k], b[k] = float("nan"), float("inf")
    ids = (torch.arange(t, device="cuda") * 3 % 5).int()
    y = ints(50, t, 72).to(dtype)
    want = y.double()
    for k in (1, 3):
        at = (ids == k).nonzero()[:, 0]
        want[at] += (x[at].double() @ a[k].double().t().contiguous()) @ b[k].double().t().contiguous()
    p = ops.AdapterGrouping(gpu, 5).encode(ids) if plan else None
    ops.LowRankAdapters(gpu, a, b, ranks=ranks).encode(x, ids, y, plan=p)
    assert torch.equal(y, want.to(dtype))
