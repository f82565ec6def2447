"""Sizes and strides that the C ABI's 32-bit numbers do not hold are refused by the operators, and never cut down to smaller ones: no device,
tensors without memory."""
from types import SimpleNamespace

import pytest
import torch

from mference_amd import operators as ops

BIG = 1 << 32


class FakeContext:
    device = torch.device("cuda", 0)
    handle = None


@pytest.fixture(autouse=True)
def no_call(monkeypatch):
    lib = ops._capi.lib()

    class Library:
        def __getattr__(self, name):
            if name in ("mf_adapter_apply", "mf_adapter_group", "mf_block_norm"):
                raise AssertionError(f"{name} was called")
            return getattr(lib, name)

    library = Library()
    monkeypatch.setattr(ops._capi, "lib", lambda: library)
    monkeypatch.setattr(ops, "_address", lambda t, *_: 1 << 40)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)


def spread(rows, width, stride, dtype=torch.bfloat16):
    return torch.empty_strided((rows, width), (stride, 1), dtype=dtype, device="meta")


def adapters(num=2, rank=8, n=64, m=16):
    meta = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="meta")  # noqa: E731
    return ops.LowRankAdapters(FakeContext(), meta(num, rank, n), meta(num, m, rank))


@pytest.mark.parametrize("stride", [BIG, BIG + 64, BIG + 4096, 3 * BIG + 64])
def test_rows_far_apart(stride):
    with pytest.raises(ops.MfError):
        ops._row_stride(spread(2, 64, stride), "x", (2, 64))
    low, ids, ws = adapters(), torch.zeros(2, dtype=torch.int32), SimpleNamespace(is_contiguous=lambda: True, get_device=lambda: 0, data_ptr=lambda: 1 << 41, nbytes=1 << 20)
    for x, y in ((spread(2, 64, stride), spread(2, 16, 16)), (spread(2, 64, 64), spread(2, 16, stride))):
        with pytest.raises(ops.MfError):
            low.encode(x, ids, y, workspace=ws, stream=0)
    norm = ops.BlockNorm(FakeContext())
    for far in range(4):
        h, d, o, g = (spread(2, 64, stride if k == far else 64) for k in range(4))
        with pytest.raises(ops.MfError):
            norm.encode(h, d, out=o, pre_weight=torch.empty(64, dtype=torch.bfloat16, device="meta"), gate=g, gate_kind=ops.GATE_ELEMENT, stream=0)
    with pytest.raises(ops.MfError):
        norm.encode(spread(2, 64, 64), spread(2, 64, 64), gate=spread(2, 1, stride), gate_kind=ops.GATE_ROW, stream=0)


def test_strides_that_fit():
    assert ops._row_stride(spread(2, 64, BIG - 1), "x", (2, 64)) == BIG - 1


@pytest.mark.parametrize("t", [BIG, BIG + 5, (1 << 20) + 1, -1])
def test_numbers_of_rows(t):
    assert adapters().workspace_bytes(t) == 0
    with pytest.raises(ops.MfError):
        ops.AdapterGrouping(FakeContext(), 3).plan(t)
    with pytest.raises(ops.MfError):
        ops.AdapterPlan(t, 3, torch.zeros(1000, dtype=torch.int32))
    if t > 0:
        with pytest.raises(ops.MfError):
            ops.BlockNorm(FakeContext()).encode(spread(t, 1, 1), spread(t, 1, 1), stream=0)
        with pytest.raises(ops.MfError):
            adapters().encode(spread(t, 64, 64), torch.empty(t, dtype=torch.int32, device="meta"), spread(t, 16, 16), stream=0)
        with pytest.raises(ops.MfError):
            ops.AdapterGrouping(FakeContext(), 3).encode(torch.empty(t, dtype=torch.int32, device="meta"), stream=0)


def test_widths():
    for kw in (dict(n=BIG + 64), dict(rank=BIG + 8), dict(num=BIG + 2), dict(m=BIG + 16), dict(m=(1 << 28) + 1), dict(n=(1 << 22) + 64)):
        with pytest.raises(ops.MfError):
            adapters(**kw)
    with pytest.raises(ops.MfError):
        ops.BlockNorm(FakeContext()).encode(spread(1, BIG + 64, BIG + 64), spread(1, BIG + 64, BIG + 64), stream=0)
