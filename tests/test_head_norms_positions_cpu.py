"""Which positions HeadNorms takes beside a table of axes: without a device, the library's call caught in front of the C entry; and
mf_head_norms itself on a zeroed block of memory in the place of a context, as far as its checks."""
import ctypes as C
from struct import Struct

import pytest
import torch

from mference_amd import _capi
from mference_amd import operators as ops


class Nowhere:
    """a context of a device that CPU tensors say they lie on"""
    class device:
        index = -1
    handle = None


class Caught:
    def mf_head_norms(self, ctx, stream, args):
        self.args = Struct("@3P5I4x3P5I4x3P5Ii3f0P").unpack(args)
        return 0

    def mf_status_string(self, status):
        return b"refused"


@pytest.fixture
def caught(monkeypatch):
    lib = Caught()
    monkeypatch.setattr(_capi, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_on", lambda context, stream: 0)
    return lib


def encode(table, positions, t=5):
    op = ops.HeadNorms(Nowhere, 8, torch.ones(4), None if table is None else torch.tensor(table, dtype=torch.uint8))
    op.encode(torch.zeros(t, 2, 8, dtype=torch.bfloat16), positions=positions)


def asked(lib):
    """axes and position_stride of the call"""
    return lib.args[-6], lib.args[-5]


def positions(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("table", [[0, 1, 2, 0], [1, 1, 1, 1], [0, 255, 7, 0]])
def test_one_axis_for_a_table_of_several_is_refused(caught, table):
    with pytest.raises(ops.MfError):
        encode(table, positions(5))
    assert not hasattr(caught, "args")


@pytest.mark.parametrize("table", [None, [0, 0, 0, 0], [0, 255, 8, 0]])
def test_one_axis(caught, table):
    encode(table, positions(5))
    assert asked(caught) == (1, 5)


def test_one_axis_said_to_be_one(caught):
    encode([0, 1, 2, 0], positions(1, 5))  # (the others are none: their pairs are not turned)
    assert asked(caught) == (1, 5)


@pytest.mark.parametrize("t", [1, 5])
def test_one_row_for_all_axes(caught, t):
    encode([0, 1, 2, 0], positions(t).expand(3, t), t)
    assert asked(caught) == (3, _capi.SAME_POSITIONS)
    encode([0, 1, 2, 0], positions(3, 40)[:, 7:7 + t], t)
    assert asked(caught) == (3, 40)


def test_axes_that_overlap_are_refused(caught):
    with pytest.raises(ops.MfError):
        encode([0, 1, 2, 0], positions(40).as_strided((3, 5), (4, 1)))


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the accepted calls would be launched")
def test_the_c_call():
    ctx = C.cast(C.create_string_buffer(4096), C.c_void_p)
    row = _capi.HeadRows(x=1 << 40, out=1 << 40, heads=4)
    call = lambda **v: _capi.lib().mf_head_norms(ctx, None, C.byref(_capi.HeadNormsArgs(**{**dict(
        q=row, positions=1 << 41, inv_freq=1 << 42, axis_of_pair=1 << 43, t=10, head_dim=64, rotary_dim=32, axes=3, eps=1e-6, rotation_scale=1.0), **v})))
    assert call(position_stride=_capi.SAME_POSITIONS) == -7  # (as far as the HIP runtime)
    assert call(position_stride=9) == -2
    beside = (1 << 40) + 2 * 4 * 64 * 10
    assert call(position_stride=_capi.SAME_POSITIONS, positions=(1 << 40) - 40) == -7  # ten positions, not thirty
    assert call(position_stride=_capi.SAME_POSITIONS, positions=(1 << 40) - 36) == -1
    assert call(positions=(1 << 40) - 40) == -1
    assert call(position_stride=_capi.SAME_POSITIONS, positions=beside) == -7
