"""mf_block_norm on both sides of the magnitude from which its sums of squares overflow: a root mean square of 2^64 / sqrt(d)."""
from __future__ import annotations

import math

import pytest
import torch

from mference_amd import operators as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1, 64, 1024, 4096, 16384, 65536])
@pytest.mark.parametrize("delta32", [False, True])
def test_both_sides_of_the_largest_magnitude(gpu, d, delta32):
    """Rows of +-v, v a power of two: the sum of squares d v^2 is a power of two (d is one of four), exact in any order, so its root and the division
    by it are too and the norm of a row is its signs.  From d v^2 = 2^128 on the sum is infinite and the norm 0."""
    limit = 64 - int(math.log2(d)) // 2
    sign = torch.where(torch.rand(3, d, device="cuda") < 0.5, -1.0, 1.0)
    one = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    for power, want in ((limit - 1, sign), (limit, torch.zeros_like(sign))):
        rows = sign * 2.0 ** power
        # the norm in front of the next block
        hidden, out = rows.bfloat16(), torch.full((3, d), 5.0, dtype=torch.bfloat16, device="cuda")
        ops.BlockNorm(gpu).encode(hidden, out=out, pre_weight=one)
        assert torch.equal(out.float(), want), power
        # the norm behind this one
        stream = torch.zeros(3, d, dtype=torch.bfloat16, device="cuda")
        ops.BlockNorm(gpu).encode(stream, rows if delta32 else rows.bfloat16(), post_weight=one)
        assert torch.equal(stream.float(), want), power
