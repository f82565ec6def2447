"""Views of heads that mf_head_norms takes and refuses by where their elements lie: host arithmetic, no device.  A zeroed block of memory stands
in for the context.  A call that passes every check reaches the HIP runtime, which has no device here (such calls are not made where there is
one: no kernel may see these addresses)."""
import ctypes as C
import random

import pytest
import torch

from mference_amd import _capi

INVALID, DIMENSION, LAUNCH = -1, -2, -7

needs_no_device = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the accepted calls would be launched")


@pytest.fixture
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def rows(x, heads, row, head, out=None, out_row=None, out_head=None):
    """heads of bf16 elements numbered from x on (numbers of elements, as addresses from 2^40 on)"""
    at = lambda e: (1 << 40) + 2 * e
    return _capi.HeadRows(x=at(x), out=at(x if out is None else out), weight=None, heads=heads, row_stride=row, head_stride=head,
                          out_row_stride=row if out_row is None else out_row, out_head_stride=head if out_head is None else out_head)


def call(ctx, q, k, t, dim):
    a = _capi.HeadNormsArgs(q=q, k=k or _capi.HeadRows(), t=t, head_dim=dim, eps=1e-6, rotation_scale=1.0)
    return _capi.lib().mf_head_norms(ctx, None, C.byref(a))


@needs_no_device
def test_one_row_of_a_long_cache(ctx):
    """one token's keys into a cache whose heads lie so far apart that all of them pass 2^32 elements: a row stride that one row does not have"""
    far = (1 << 32) // 64 + 8
    assert call(ctx, rows(0, 4, 0, 128), rows(1 << 20, 64, 0, 128, out=1 << 36, out_row=0, out_head=far), 1, 128) == LAUNCH
    assert call(ctx, rows(0, 64, 0, far), None, 1, 128) == LAUNCH
    assert call(ctx, rows(0, 64, 0, far), None, 2, 128) == DIMENSION  # (of two rows it is one that no argument holds)
    assert call(ctx, rows(0, 64, 128, far), None, 2, 128) == LAUNCH


@needs_no_device
@pytest.mark.parametrize("t", [1, 2, 300])
def test_queries_and_keys_head_by_head(ctx, t):
    """a head's query, key and value side by side, in place and to another buffer of that kind; rows in front of heads and behind"""
    h, dim = 5, 64
    row, head = 3 * h * dim, 3 * dim
    assert call(ctx, rows(0, h, row, head), rows(dim, h, row, head), t, dim) == LAUNCH
    assert call(ctx, rows(2 * dim, h, row, head), rows(0, h, row, head), t, dim) == LAUNCH
    assert call(ctx, rows(0, h, row, head, out=dim), None, t, dim) == LAUNCH
    row, head = 3 * dim, 3 * dim * t
    assert call(ctx, rows(0, h, row, head), rows(dim, h, row, head), t, dim) == LAUNCH


def test_queries_and_keys_that_meet(ctx):
    h, dim, t = 5, 64, 7
    row, head = 3 * h * dim, 3 * dim
    for shift in (1, dim - 1, head + dim - 1, head, row - dim + 1, row + 1, 2 * row + head - 1):
        assert call(ctx, rows(0, h, row, head), rows(shift, h, row, head), t, dim) == INVALID, shift
        assert call(ctx, rows(0, h, row, head, out=shift), None, t, dim) == INVALID, shift


@needs_no_device
def test_against_a_list_of_elements(ctx):
    """two sets of the same strides at random places: refused exactly where they share an element"""
    rng = random.Random(5)
    seen = {INVALID: 0, LAUNCH: 0}
    for _ in range(3000):
        dim, t, hq, hk = rng.randint(1, 6), rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 5)
        if rng.random() < 0.5:  # heads in rows
            head = dim + rng.randint(0, 9)
            row = (max(hq, hk) - 1) * head + dim + rng.randint(0, 9)
        else:
            row = dim + rng.randint(0, 9)
            head = (t - 1) * row + dim + rng.randint(0, 9)
        shift = rng.randint(0, 3 * (row + head))
        a, b = (0, shift) if rng.random() < 0.5 else (shift, 0)
        elements = lambda x, heads: {x + i * row + j * head + e for i in range(t) for j in range(heads) for e in range(dim)}
        want = INVALID if elements(a, hq) & elements(b, hk) else LAUNCH
        seen[want] += 1
        assert call(ctx, rows(a, hq, row, head), rows(b, hk, row, head), t, dim) == want, (dim, t, hq, hk, row, head, a, b)
    assert min(seen.values()) > 500
