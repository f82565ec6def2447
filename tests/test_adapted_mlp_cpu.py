"""SharedExpertInt4.encode_adapted refuses what does not fit together in front of its first launch: no device, no library call.  Operands
are CPU tensors whose device is not looked at here."""
from contextlib import nullcontext
from types import SimpleNamespace

import pytest
import torch

from mference_amd import operators as ops


class FakeContext:
    device = torch.device("cuda", 0)
    handle = None


T, D, F, N = 12, 256, 384, 3


@pytest.fixture
def call(monkeypatch):
    def address(t, what, dtype, device):
        if t.dtype is not dtype:
            raise ValueError(f"{what} must be {dtype}")
        return t.data_ptr()

    def launched(*_, **__):
        raise AssertionError("reached its first launch")

    monkeypatch.setattr(ops, "_address", address)
    monkeypatch.setattr(ops.MPPPrefillInt4QMM, "workspace_bytes", launched)
    monkeypatch.setattr(ops.MPPPrefillInt4QMM, "encode", launched)
    monkeypatch.setattr(ops.torch.cuda, "current_stream", launched)
    ctx = FakeContext()
    w = lambda rows, n: SimpleNamespace(rows=rows, n=n)  # noqa: E731
    pool = lambda n, ms, adapters=N, device=0: SimpleNamespace(n=n, ms=ms, num_adapters=adapters, context=SimpleNamespace(device=torch.device("cuda", device)))  # noqa: E731
    args = dict(x=torch.zeros(T, D, dtype=torch.bfloat16), y=torch.zeros(T, D, dtype=torch.bfloat16), gate_up=pool(D, [F, F]), down=pool(F, [D]),
                ids=torch.zeros(T, dtype=torch.int32), plan=None, stream=None)

    def run(**over):
        a = {**args, **over}
        return ops.SharedExpertInt4(ctx).encode_adapted(a["x"], w(F, D), w(F, D), w(D, F), a["y"], a["gate_up"], a["down"], a["ids"], plan=a["plan"], stream=a["stream"])

    run.pool = pool
    return run


def plan(t, n):
    need = int(ops._capi.lib().mf_adapter_plan_bytes(t, n)) // 4
    return ops.AdapterPlan(t, n, torch.zeros(need, dtype=torch.int32))


def test_what_fits_goes_on(call):
    for p in (None, plan(T, N)):
        with pytest.raises(AssertionError, match="first launch"):
            call(plan=p)


def test_pools_of_different_numbers_of_adapters(call):
    for over in (dict(gate_up=call.pool(D, [F, F], N + 1)), dict(down=call.pool(F, [D], N - 1)), dict(down=call.pool(F, [D], N + 1), plan=plan(T, N))):
        with pytest.raises(ops.MfError):
            call(**over)


def test_plans_of_other_rows_or_adapters(call):
    for p in (plan(T + 1, N), plan(T, N + 1)):
        with pytest.raises(ops.MfError):
            call(plan=p)


def test_adapters_of_rows(call):
    for ids in (torch.zeros(T - 1, dtype=torch.int32), torch.zeros(T + 1, dtype=torch.int32), torch.zeros(T, 1, dtype=torch.int32), torch.zeros(2 * T, dtype=torch.int32)[::2],
                torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ops.MfError):
            call(ids=ids)
    with pytest.raises(ValueError):
        call(ids=torch.zeros(T, dtype=torch.int64))


def test_adapters_of_another_device(call):
    for over in (dict(gate_up=call.pool(D, [F, F], N, 1)), dict(down=call.pool(F, [D], N, 1))):
        with pytest.raises(ValueError, match="another device"):
            call(**over)


@pytest.mark.parametrize("bits", [(8, 4, 4), (4, 8, 4), (4, 4, 8), (4, 4, 3)])
def test_projections_that_refuse_their_operands(monkeypatch, bits):
    """the paths of all three are asked for before the first of them is launched (host arithmetic over the operands' addresses)"""
    lib, launches = ops._capi.lib(), []

    class Library:
        def __getattr__(self, name):
            return (lambda *a: launches.append(name) or 0) if name == "mf_qmm" else getattr(lib, name)

    class Stream(int):
        cuda_stream = 0

    stream = Stream()
    monkeypatch.setattr(ops, "_address", lambda t, *_: t.data_ptr())
    monkeypatch.setattr(ops.torch.cuda, "current_stream", lambda *_: stream)
    monkeypatch.setattr(ops.torch.cuda, "stream", lambda s: nullcontext())
    library = Library()
    monkeypatch.setattr(ops._capi, "lib", lambda: library)
    w = lambda rows, n, b: ops.QuantizedTensor(torch.zeros(rows, n, dtype=torch.uint8), torch.zeros(rows, n // 64, dtype=torch.bfloat16),  # noqa: E731
                                               torch.zeros(rows, n // 64, dtype=torch.bfloat16), b, rows, n)
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    pool = lambda n, ms: SimpleNamespace(n=n, ms=ms, num_adapters=N, context=FakeContext(), encode=lambda *a, **k: launches.append("adapters"))  # noqa: E731
    x, y = torch.zeros(T, D, dtype=torch.bfloat16), torch.zeros(T, D, dtype=torch.bfloat16)
    monkeypatch.setattr(ops.Elementwise, "encode_silu_mul", lambda *a, **k: launches.append("silu_mul"))
    run = lambda b: ops.SharedExpertInt4(FakeContext()).encode_adapted(x, w(F, D, b[0]), w(F, D, b[1]), w(D, F, b[2]), y, pool(D, [F, F]), pool(F, [D]),  # noqa: E731
                                                                       torch.zeros(T, dtype=torch.int32))
    with pytest.raises(ops.MfError):
        run(bits)
    assert not launches
    run((4, 4, 4))
    assert launches == ["mf_qmm", "mf_qmm", "adapters", "silu_mul", "mf_qmm", "adapters"]


def test_the_null_streams_handle(monkeypatch, call):
    """torch.cuda.ExternalStream(0) is no stream of handle 0 but one of torch's own: stream=0 has to be the device's default stream"""
    default, entered = SimpleNamespace(cuda_stream=0), []

    def no_handle(handle, device=None):
        raise AssertionError("a stream object of a handle of 0")

    class Entered(Exception):
        pass

    def stream(s):
        entered.append(s)
        raise Entered

    monkeypatch.setattr(ops.torch.cuda, "ExternalStream", no_handle)
    monkeypatch.setattr(ops.torch.cuda, "default_stream", lambda device=None: default)
    monkeypatch.setattr(ops.torch.cuda, "stream", stream)
    with pytest.raises(Entered):
        call(stream=0)
    assert entered == [default]
