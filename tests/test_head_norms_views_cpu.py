"""Views of heads that mf_head_norms takes and refuses by where their elements lie: host arithmetic, no device.  A zeroed block of memory stands
in for the context.  A call that passes every check reaches the HIP runtime, which has no device here (such calls are not made where there is
one: no kernel may see these addresses)."""
import ctypes as C

import pytest
import torch

from mference_amd import _capi

DIMENSION, LAUNCH = -2, -7

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
