"""What mf_adapter_group, mf_adapter_apply and mf_block_norm refuse, and the sizes they ask for: host arithmetic, no device.
A zeroed block of memory stands in for the context.  Nothing is launched by a refused call; one that passes every check reaches
the HIP runtime, which has no device here (or would be handed addresses that no kernel may see, so such calls are not made where
there is a device)."""
import ctypes as C

import numpy as np
import pytest
import torch

from mference_amd import _capi
from mference_amd import operators as ops

OK, INVALID, DIMENSION, SCRATCH, LAUNCH = 0, -1, -2, -4, -7

needs_no_device = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the accepted calls would be launched")


class Memory:
    """addresses that look like device buffers, apart from each other"""

    def __init__(self):
        self.at = 1 << 40

    def take(self, size, off=0):
        p = self.at + off
        self.at += (size + 4095) // 4096 * 4096 + 4096
        return p


@pytest.fixture
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def pool(num_adapters=4, rank=16, n=128, ranks=None, scales=None):
    return _capi.AdapterPool(num_adapters, rank, n, ranks, scales)


def apply_args(t=5, m=(96,), f32=0, p=None, x_stride=None, y_strides=None, **over):
    mem = Memory()
    p = p or pool()
    size = 4 if f32 else 2
    ys = y_strides or m
    targets = (_capi.AdapterTarget * len(m))()
    for g, k, st in zip(targets, m, ys):
        g.a, g.b = mem.take(p.num_adapters * p.rank * p.n * 2), mem.take(p.num_adapters * p.rank * k * 2)
        g.y, g.m, g.y_stride = mem.take(t * st * size + 64), k, st
    need = _capi.lib().mf_adapter_workspace_bytes(C.byref(p), len(m), t)
    args = dict(pool=C.byref(p), targets=targets, num_targets=len(m), x=mem.take(t * (x_stride or p.n) * 2 + 64), x_stride=x_stride or p.n, ids=mem.take(4 * t + 64),
                t=t, f32=f32, plan=None, ws=mem.take(need + 64), ws_bytes=need)
    args.update(over)
    return args


def apply(ctx, a):
    return _capi.lib().mf_adapter_apply(ctx, None, a["pool"], a["targets"], a["num_targets"], a["x"], a["x_stride"], a["ids"], a["t"], a["f32"], a["plan"], a["ws"], a["ws_bytes"])


def test_adapter_apply_refuses(ctx):
    base = apply_args()
    for name, value, status in [("pool", None, INVALID), ("targets", None, INVALID), ("num_targets", 0, INVALID), ("num_targets", 5, INVALID), ("x", None, INVALID),
                                ("ids", None, INVALID), ("ws", None, INVALID), ("t", (1 << 20) + 1, INVALID), ("x_stride", 127, DIMENSION),
                                ("x", base["x"] + 1, INVALID), ("ids", base["ids"] + 2, INVALID), ("ws", base["ws"] + 8, INVALID), ("plan", base["ws"] + 8, INVALID),
                                ("ws_bytes", base["ws_bytes"] - 1, SCRATCH)]:
        assert apply(ctx, {**base, name: value}) == status, name
    assert apply(None, base) == INVALID
    assert apply(ctx, {**base, "t": 0, "x": None, "ids": None, "ws": None}) == OK


@pytest.mark.parametrize("bad", [dict(num_adapters=0), dict(num_adapters=1025), dict(rank=0), dict(rank=4), dict(rank=12), dict(rank=264), dict(n=0), dict(n=96)])
def test_adapter_apply_refuses_pools(ctx, bad):
    base = apply_args()
    p = pool(**bad)
    assert _capi.lib().mf_adapter_workspace_bytes(C.byref(p), 1, 5) == 0
    assert apply(ctx, {**base, "pool": C.byref(p), "x_stride": 4096}) == DIMENSION


@pytest.mark.parametrize("field, value, status", [("a", 0, INVALID), ("b", 0, INVALID), ("y", 0, INVALID), ("m", 0, DIMENSION), ("y_stride", 95, DIMENSION),
                                                  ("a", 8, INVALID), ("b", 2, INVALID), ("y", 1, INVALID)])
def test_adapter_apply_refuses_targets(ctx, field, value, status):
    a = apply_args()
    g = a["targets"][0]
    setattr(g, field, getattr(g, field) + value if value and field in "aby" else value or None if field in "aby" else value)
    assert apply(ctx, a) == status


def test_adapter_apply_refuses_unaligned_fp32_results(ctx):
    a = apply_args(f32=1)
    a["targets"][0].y += 2
    assert apply(ctx, a) == INVALID


@pytest.mark.parametrize("ranks, scales", [(2, None), (None, 2)])
def test_adapter_apply_refuses_unaligned_tables(ctx, ranks, scales):
    assert apply(ctx, apply_args(p=pool(ranks=ranks and (1 << 50) + ranks, scales=scales and (1 << 50) + scales))) == INVALID


def test_adapter_apply_refuses_shared_memory(ctx):
    # y on x, in whole and by its last byte
    a = apply_args()
    for y in (a["x"], a["x"] + 2 * 128 * 5 - 2, a["x"] - 2 * 96 * 5 + 2):
        a["targets"][0].y = y
        assert apply(ctx, a) == INVALID
    # two results: the same rows; one buffer of rows of 192 whose columns meet, from either side, and around a row's end
    a = apply_args(m=(96, 96), y_strides=(192, 192))
    g = a["targets"]
    for off in (0, 2 * 95, -2 * 95, 2 * 192 * 2 + 2 * 10, 2 * 97):
        g[1].y = g[0].y + off
        assert apply(ctx, a) == INVALID, off
    # other strides
    a = apply_args(m=(96, 96), y_strides=(192, 200))
    a["targets"][1].y = a["targets"][0].y + 2 * 96
    assert apply(ctx, a) == INVALID


@needs_no_device
def test_adapter_apply_accepts(ctx):
    assert apply(ctx, apply_args()) == LAUNCH
    a = apply_args(m=(96, 96), y_strides=(192, 192))  # column ranges of one buffer
    a["targets"][1].y = a["targets"][0].y + 2 * 96
    assert apply(ctx, a) == LAUNCH
    a["targets"][1].y = a["targets"][0].y - 2 * 96
    assert apply(ctx, a) == LAUNCH
    # x and y column ranges of one buffer
    a = apply_args(x_stride=256, y_strides=(256,))
    a["targets"][0].y = a["x"] + 2 * 128
    assert apply(ctx, a) == LAUNCH


def test_adapter_group_refuses(ctx):
    lib = _capi.lib()
    need = lib.mf_adapter_plan_bytes(100, 7)
    assert need >= 4 * (100 + 8)
    ids, plan = 1 << 40, 1 << 41
    call = lambda c=ctx, i=ids, t=100, n=7, p=plan, b=need: lib.mf_adapter_group(c, None, i, t, n, p, b)  # noqa: E731
    assert call(c=None) == INVALID and call(i=None) == INVALID and call(p=None) == INVALID
    assert call(t=(1 << 20) + 1) == INVALID and call(n=0) == INVALID and call(n=1025) == INVALID
    assert call(p=plan + 4) == INVALID and call(i=ids + 1) == INVALID
    assert call(b=need - 1) == SCRATCH
    assert call(i=plan + 4 * 3) == INVALID  # the ids inside the plan
    assert lib.mf_adapter_plan_bytes((1 << 20) + 1, 7) == 0 and lib.mf_adapter_plan_bytes(5, 0) == 0 and lib.mf_adapter_plan_bytes(5, 1025) == 0
    assert lib.mf_adapter_plan_bytes(0, 1) > 0


def test_workspace_serves_smaller_batches():
    lib = _capi.lib()
    for p, targets in ((pool(), 1), (pool(rank=8, n=64), 1), (pool(rank=256, n=17408), 4), (pool(rank=16, n=5120), 2)):
        last = 0
        for t in [0] + sorted(set(int(1.13 ** k) for k in range(114)) | {15, 16, 17, 63, 64, 65, 1 << 20}):
            if t <= 1 << 20:
                now = lib.mf_adapter_workspace_bytes(C.byref(p), targets, t)
                assert now >= last, (t, targets)
                last = now
    assert lib.mf_adapter_workspace_bytes(C.byref(pool()), 0, 5) == 0 and lib.mf_adapter_workspace_bytes(C.byref(pool()), 5, 5) == 0
    assert lib.mf_adapter_workspace_bytes(None, 1, 5) == 0


def norm_args(t=3, d=40, **over):
    mem = Memory()
    a = _capi.BlockNormArgs()
    a.d, a.t, a.residual_scale, a.branch_scale, a.post_eps, a.pre_eps = d, t, 1.0, 1.0, 1e-6, 1e-6
    for name in ("hidden", "delta", "pre_weight", "out"):
        setattr(a, name, mem.take(t * d * 4 + 64))
    for k, v in over.items():
        setattr(a, k, v)
    return a, mem


def norm(ctx, a):
    return _capi.lib().mf_block_norm(ctx, None, C.byref(a))


@pytest.mark.parametrize("over, status", [
    (dict(d=0), DIMENSION), (dict(t=(1 << 20) + 1), INVALID), (dict(gate_kind=4), INVALID), (dict(gate_kind=-1), INVALID), (dict(gate_kind=1), INVALID),
    (dict(gate=1 << 50), INVALID), (dict(delta=None, post_weight=1 << 50), INVALID), (dict(delta=None, gate=1 << 50, gate_kind=1), INVALID),
    (dict(out=None), INVALID), (dict(pre_weight=None), INVALID), (dict(delta=None, out=None, pre_weight=None), INVALID), (dict(hidden=None), INVALID),
    (dict(hidden_stride=39), DIMENSION), (dict(delta_stride=39), DIMENSION), (dict(out_stride=39), DIMENSION),
    (dict(gate=1 << 50, gate_kind=2, gate_stride=39), DIMENSION), (dict(gate=(1 << 50) + 1, gate_kind=1), INVALID), (dict(post_weight=(1 << 50) + 1), INVALID)])
def test_block_norm_refuses(ctx, over, status):
    assert norm(ctx, norm_args(**over)[0]) == status


@pytest.mark.parametrize("d", [(1 << 28) + 1, (1 << 32) - 8, (1 << 32) - 1])
def test_block_norm_refuses_rows_that_are_too_long(ctx, d):
    a, _ = norm_args()
    a.d = d
    assert norm(ctx, a) == DIMENSION


def test_block_norm_refuses_unaligned_and_shared(ctx):
    for name in ("hidden", "delta", "pre_weight", "out"):
        a, _ = norm_args()
        setattr(a, name, getattr(a, name) + 1)
        assert norm(ctx, a) == INVALID, name
    a, _ = norm_args(delta_f32=1)
    a.delta += 2
    assert norm(ctx, a) == INVALID
    for one, other in (("out", "hidden"), ("out", "delta"), ("hidden", "delta"), ("out", "gate"), ("hidden", "gate"), ("out", "pre_weight"), ("hidden", "post_weight"),
                       ("hidden", "pre_weight"), ("out", "post_weight")):
        a, mem = norm_args()
        if other == "gate":
            a.gate, a.gate_kind = mem.take(1000), _capi.GATE_ELEMENT
        if other == "post_weight":
            a.post_weight = mem.take(1000)
        setattr(a, other, getattr(a, one))
        assert norm(ctx, a) == INVALID, (one, other)
        setattr(a, other, getattr(a, one) + 2 * 39)
        assert norm(ctx, a) == INVALID, (one, other)
    a, mem = norm_args(gate_kind=_capi.GATE_CHANNEL)
    a.gate = a.hidden + 2 * 3
    assert norm(ctx, a) == INVALID
    assert norm(None, norm_args()[0]) == INVALID and _capi.lib().mf_block_norm(ctx, None, None) == INVALID


@needs_no_device
def test_block_norm_accepts(ctx):
    assert norm(ctx, norm_args()[0]) == LAUNCH
    a, _ = norm_args(delta=None)
    assert norm(ctx, a) == LAUNCH
    a, _ = norm_args(out=None, pre_weight=None)
    assert norm(ctx, a) == LAUNCH
    a, _ = norm_args(t=0)
    assert norm(ctx, a) == OK
    # hidden and delta column ranges of one buffer
    a, _ = norm_args(hidden_stride=80, delta_stride=80)
    a.delta = a.hidden + 2 * 40
    assert norm(ctx, a) == LAUNCH


class FakeContext:
    device = torch.device("cuda", 0)
    handle = None


def test_operators_refuse_before_the_library():
    ctx = FakeContext()
    a, b = torch.zeros(4, 16, 128, dtype=torch.bfloat16), torch.zeros(4, 96, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.LowRankAdapters(ctx, a, b)
    for wa, wb in ((a[0], b), (a, b[:3]), (a, b[0]), (a, b[:, :, :8])):
        with pytest.raises(ops.MfError):
            ops.LowRankAdapters(ctx, wa, wb)
    with pytest.raises(ops.MfError):
        ops.LowRankAdapters(ctx, [a] * 5, [b] * 5)
    with pytest.raises(ops.MfError):
        ops.LowRankAdapters(ctx, [a, a], [b])
    for n in (0, 1025, -1):
        with pytest.raises(ops.MfError):
            ops.AdapterGrouping(ctx, n)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.AdapterGrouping(ctx, 3).encode(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ops.MfError):
        ops.AdapterGrouping(ctx, 3).plan((1 << 20) + 1)
    with pytest.raises(ops.MfError):
        ops.AdapterGrouping(ctx, 3).plan(-1)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.BlockNorm(ctx).encode(torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(2, 8, dtype=torch.bfloat16))


def test_rows_of_a_tensor():
    whole = torch.zeros(6, 40)
    for v, stride in ((whole, 40), (whole[:, 8:24], 40), (whole[::2], 80), (whole[:1], 40), (whole[:1, 3:5], 2), (whole[:, :1], 40), (whole[:0], 40)):
        assert ops._row_stride(v, "x", v.shape) == stride
    for bad in (whole.t(), whole[:, ::2], whole[0].expand(6, 40), whole[:1].expand(2, 40)):
        with pytest.raises(ops.MfError):
            ops._row_stride(bad, "x", bad.shape)
    with pytest.raises(ops.MfError):
        ops._row_stride(whole, "x", (6, 41))


def test_packed_arguments_are_the_structures():
    """the operators pack their arguments by hand: the same bytes as the ctypes structures'"""
    values = tuple(range(1 << 40, (1 << 40) + 6)) + (7, 8, 9, 10, 11, 12, 1, 2, 0.5, 0.25, 2.0, 4.0, 1.0)
    assert ops.BlockNorm._pack(*values) == bytes(_capi.BlockNormArgs(*values))
    one, two = (1 << 40, 1 << 41, 1 << 42, 96, 192), (1 << 43, 1 << 44, 1 << 45, 64, 192)
    assert ops.Struct("@" + "PPPII" * 2).pack(*one, *two) == bytes(_capi.AdapterTarget(*one)) + bytes(_capi.AdapterTarget(*two))


def test_a_plan_has_room():
    need = _capi.lib().mf_adapter_plan_bytes(40, 3) // 4
    assert ops.AdapterPlan(40, 3, torch.zeros(need, dtype=torch.int32)).rows.numel() == 40
    for t, n, words in ((40, 3, torch.zeros(need - 1, dtype=torch.int32)), (40, 3, torch.zeros(need, dtype=torch.int64)), (40, 3, torch.zeros(2 * need, dtype=torch.int32)[::2]),
                        (-1, 3, torch.zeros(need, dtype=torch.int32)), (40, 0, torch.zeros(need, dtype=torch.int32))):
        with pytest.raises(ops.MfError):
            ops.AdapterPlan(t, n, words)
