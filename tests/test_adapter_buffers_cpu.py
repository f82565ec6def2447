"""Which stream's memory the buffers come from that AdapterGrouping.encode and LowRankAdapters.encode take by themselves.  A block that was
freed on the current stream may still be read or written by work of that stream: a call on another stream has to take its buffers as that
stream's own.  No device: streams, allocator and library are stand-ins."""
from contextlib import contextmanager

import pytest
import torch

from mference_amd import operators as ops

CURRENT, SIDE = 1000, 2000


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


class FakeContext:
    device = torch.device("cuda", 0)
    handle = None


@pytest.fixture
def world(monkeypatch):
    """taken: (bytes, stream whose memory it is); used: (tensor's bytes, other stream it is known to be used on)"""
    taken, used, now = [], [], [CURRENT]
    real_empty, lib = torch.empty, ops._capi.lib()

    @contextmanager
    def stream(s):
        before, now[0] = now[0], s.cuda_stream
        yield
        now[0] = before

    def empty(size, dtype=None, device=None):
        t = real_empty(size, dtype=dtype)
        taken.append((t.nbytes, now[0]))
        return t

    class Library:
        def __getattr__(self, name):
            return (lambda *a: 0) if name in ("mf_adapter_group", "mf_adapter_apply") else getattr(lib, name)

    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: Stream(handle))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Stream(0))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(now[0]))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: used.append((t.nbytes, s.cuda_stream)))
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now[0])
    monkeypatch.setattr(ops, "_address", lambda t, *_: t.data_ptr())
    library = Library()
    monkeypatch.setattr(ops._capi, "lib", lambda: library)
    return taken, used


STREAMS = [(None, CURRENT), (Stream(SIDE), SIDE), (SIDE, SIDE), (Stream(CURRENT), CURRENT), (CURRENT, CURRENT), (0, 0)]


@pytest.mark.parametrize("stream, owner", STREAMS)
def test_workspace(world, stream, owner):
    taken, _ = world
    low = ops.LowRankAdapters(FakeContext(), torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 8, dtype=torch.bfloat16))
    ids = torch.zeros(5, dtype=torch.int32)
    low.encode(torch.zeros(5, 64, dtype=torch.bfloat16), ids, torch.zeros(5, 16, dtype=torch.bfloat16), stream=stream)
    assert taken == [(low.workspace_bytes(5), owner)]


@pytest.mark.parametrize("stream, owner", STREAMS)
def test_plan(world, stream, owner):
    """a plan is the caller's afterwards, who may go on with it on the stream that was current: the allocator knows of both"""
    taken, used = world
    plan = ops.AdapterGrouping(FakeContext(), 3).encode(torch.zeros(5, dtype=torch.int32), stream=stream)
    assert taken == [(plan.words.nbytes, owner)]
    assert owner == CURRENT or (plan.words.nbytes, CURRENT) in used
