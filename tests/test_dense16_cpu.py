"""What mf_project, mf_head_norms and mf_bf16_experts refuse, and the sizes they ask for: host arithmetic, no device.  A zeroed block of
memory stands in for the context.  Nothing is launched by a refused call; one that passes every check reaches the HIP runtime, which has no
device here (such calls are not made where there is one: no kernel may see these addresses)."""
import ctypes as C

import pytest
import torch

from mference_amd import _capi
from mference_amd import operators as ops

OK, INVALID, DIMENSION, SCRATCH, LAUNCH, COUNT = 0, -1, -2, -4, -7, -10

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


# ------------------------------------------------------------------ projection

def project_args(**over):
    mem = Memory()
    v = dict(x=mem.take(1 << 20), w=mem.take(1 << 20), bias=mem.take(1 << 12), residual=mem.take(1 << 20), y=mem.take(1 << 20), t=20, m=96, n=128, x_stride=0, w_stride=0,
             residual_stride=0, y_stride=0, y_f32=0, gated=0, activation=0, ws=mem.take(1 << 24), ws_bytes=1 << 24)
    v.update(over)
    return v


def project(ctx, **over):
    v = project_args(**over)
    ws, size = v.pop("ws"), v.pop("ws_bytes")
    return _capi.lib().mf_project(ctx, None, C.byref(_capi.ProjectArgs(**v)), ws, size)


@pytest.mark.parametrize("over, status", [
    (dict(t=(1 << 20) + 1), INVALID), (dict(activation=4), INVALID), (dict(activation=-1), INVALID), (dict(m=0), DIMENSION), (dict(m=(1 << 24) + 1), DIMENSION), (dict(n=0), DIMENSION),
    (dict(n=(1 << 22) + 1), DIMENSION), (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID), (dict(x_stride=127), DIMENSION), (dict(w_stride=127), DIMENSION),
    (dict(y_stride=95), DIMENSION), (dict(residual_stride=95), DIMENSION), (dict(x=(1 << 50) + 1), INVALID), (dict(w=(1 << 50) + 1), INVALID), (dict(bias=(1 << 50) + 1), INVALID),
    (dict(y=(1 << 50) + 1), INVALID), (dict(residual=(1 << 50) + 1), INVALID), (dict(y=(1 << 50) + 2, y_f32=1), INVALID), (dict(residual=(1 << 50) + 2, y_f32=1), INVALID), (dict(t=0), OK),
    (dict(t=0, x=None, y=None), OK),
])
def test_project_refuses(ctx, over, status):
    assert project(ctx, **over) == status


def test_project_refuses_without_context_or_arguments(ctx):
    lib = _capi.lib()
    assert lib.mf_project(ctx, None, None, None, 0) == INVALID
    assert lib.mf_project(None, None, C.byref(_capi.ProjectArgs()), None, 0) == INVALID


def test_project_refuses_shared_memory(ctx):
    v = project_args()
    for name in ("x", "w", "bias"):
        assert project(ctx, y=v[name]) == INVALID, name
        assert project(ctx, y=v[name] + 100) == INVALID, name
    assert project(ctx, residual=v["y"] + 2) == INVALID
    assert project(ctx, residual=v["y"], residual_stride=128, y_stride=96) == INVALID  # another stride: other rows meet
    assert project(ctx, x=v["y"] + 2 * 96, x_stride=256, y_stride=128) == INVALID  # another stride: rows meet somewhere
    need = _capi.lib().mf_project_workspace_bytes(96, 1 << 20, 20, 0)
    for name in ("y", "x", "w", "residual") if need else ():
        assert project(ctx, n=1 << 20, ws=v[name] // 16 * 16) == INVALID, name


def test_project_asks_for_its_workspace(ctx):
    lib = _capi.lib()
    for t, m, n in ((1, 64, 1 << 20), (20, 64, 65536), (300, 128, 65536), (64, 5120, 17408)):
        need = lib.mf_project_workspace_bytes(m, n, t, 0)
        if need:
            far = dict(x=1 << 50, w=1 << 51, y=1 << 52, bias=None, residual=None, ws=1 << 53)
            assert project(ctx, t=t, m=m, n=n, **far, ws_bytes=need - 1) == SCRATCH
            assert project(ctx, t=t, m=m, n=n, **{**far, "ws": None}, ws_bytes=need) == INVALID
            assert project(ctx, t=t, m=m, n=n, **{**far, "ws": (1 << 53) + 8}, ws_bytes=need) == INVALID


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("m, n", [(1, 1), (64, 64), (64, 65536), (4096, 4096), (5120, 17408), (17408, 5120), (100, 1 << 20), (2113, 2816), (250000, 2048)])
def test_project_workspace_serves_fewer_rows(m, n, gated):
    lib = _capi.lib()
    sizes = [lib.mf_project_workspace_bytes(m, n, t, gated) for t in (*range(1, 300), 512, 777, 1024, 2048, 4096, 10000, 1 << 17, 1 << 20)]
    assert sizes == sorted(sizes)
    assert sizes[-1] <= 1 << 32
    for bad in ((0, n, 1), (m, 0, 1), (1 << 25, n, 1), (m, 1 << 23, 1), (m, n, (1 << 20) + 1)):
        assert lib.mf_project_workspace_bytes(*bad, gated) == 0


@needs_no_device
def test_project_accepts(ctx):
    v = project_args()
    for over in (dict(), dict(bias=None, residual=None), dict(residual=v["y"]), dict(residual=v["y"], residual_stride=128, y_stride=128), dict(t=1, residual=v["y"], residual_stride=128),
                 dict(y_f32=1), dict(gated=1, activation=3), dict(x=1 << 50, x_stride=1 << 31), dict(x=v["x"] + 2, w=v["w"] + 2), dict(x=v["y"] + 2 * 128, x_stride=512, y_stride=512)):
        assert project(ctx, **over) == LAUNCH, over


# ------------------------------------------------------------------ head norms

def head_args(q=None, k=None, **over):
    mem = Memory()
    qx, kx = mem.take(1 << 20), mem.take(1 << 20)
    qv = dict(x=qx, out=qx, weight=mem.take(512), heads=4, row_stride=0, head_stride=0, out_row_stride=0, out_head_stride=0)
    kv = dict(x=kx, out=kx, weight=mem.take(512), heads=2, row_stride=0, head_stride=0, out_row_stride=0, out_head_stride=0)
    qv.update(q or {}), kv.update(k or {})
    v = dict(positions=mem.take(4096), inv_freq=mem.take(512), axis_of_pair=mem.take(512), t=10, head_dim=64, rotary_dim=32, axes=3, position_stride=0, interleaved=0, eps=1e-6,
             weight_bias=0.0, rotation_scale=1.0)
    v.update(over)
    return _capi.HeadNormsArgs(q=_capi.HeadRows(**qv), k=_capi.HeadRows(**kv), **v)


def head_norms(ctx, **over):
    return _capi.lib().mf_head_norms(ctx, None, C.byref(head_args(**over)))


@pytest.mark.parametrize("over, status", [
    (dict(t=(1 << 20) + 1), INVALID), (dict(head_dim=0), DIMENSION), (dict(head_dim=1025), DIMENSION), (dict(rotary_dim=66), DIMENSION), (dict(rotary_dim=31), DIMENSION),
    (dict(rotary_dim=0), INVALID), (dict(positions=None), INVALID), (dict(inv_freq=None), INVALID), (dict(axes=0), DIMENSION), (dict(axes=9), DIMENSION), (dict(position_stride=9), DIMENSION),
    (dict(positions=(1 << 50) + 2), INVALID), (dict(inv_freq=(1 << 50) + 2), INVALID), (dict(q=dict(heads=65536)), DIMENSION), (dict(k=dict(heads=65536)), DIMENSION),
    (dict(q=dict(x=None)), INVALID), (dict(q=dict(out=None)), INVALID), (dict(k=dict(x=None)), INVALID), (dict(q=dict(x=(1 << 50) + 1)), INVALID), (dict(k=dict(out=(1 << 50) + 1)), INVALID),
    (dict(q=dict(weight=(1 << 50) + 1)), INVALID), (dict(q=dict(head_stride=63)), DIMENSION), (dict(q=dict(row_stride=255)), DIMENSION), (dict(k=dict(out_row_stride=127)), DIMENSION),
    (dict(q=dict(row_stride=64, head_stride=639)), DIMENSION), (dict(q=dict(head_stride=1 << 30)), DIMENSION), (dict(t=0), OK), (dict(q=dict(heads=0, x=None, out=None), k=dict(heads=0)), OK),
])
def test_head_norms_refuses(ctx, over, status):
    assert head_norms(ctx, **over) == status


def test_head_norms_refuses_without_context_or_arguments(ctx):
    lib = _capi.lib()
    assert lib.mf_head_norms(ctx, None, None) == INVALID
    assert lib.mf_head_norms(None, None, C.byref(head_args())) == INVALID
    assert head_norms(ctx, positions=None, inv_freq=None, rotary_dim=0, axes=0) == INVALID  # axis_of_pair without positions


def test_head_norms_refuses_shared_memory(ctx):
    a = head_args()
    q, k = a.q.x, a.k.x
    for over in (dict(q=dict(out=q + 2)), dict(q=dict(out=k)), dict(k=dict(x=q + 128)), dict(q=dict(out_row_stride=512)), dict(q=dict(head_stride=128, row_stride=512)),
                 dict(positions=q), dict(inv_freq=q + 64), dict(axis_of_pair=k), dict(q=dict(weight=k)), dict(k=dict(weight=k + 32)),
                 dict(q=dict(row_stride=64, head_stride=640), k=dict(x=q + 3 * 128, out=q + 3 * 128, row_stride=640, head_stride=64))):
        assert head_norms(ctx, **over) == INVALID, over


@needs_no_device
def test_head_norms_accepts(ctx):
    a = head_args()
    q = a.q.x
    wide = dict(row_stride=512, out_row_stride=512)
    for over in (dict(), dict(q=dict(weight=None)), dict(positions=None, inv_freq=None, axis_of_pair=None, rotary_dim=0, axes=0), dict(k=dict(heads=0, x=None, out=None)),
                 dict(q=wide, k=dict(x=q + 4 * 128, out=q + 4 * 128, **wide)),  # one buffer for both
                 dict(q=dict(row_stride=64, head_stride=640, out_row_stride=64, out_head_stride=640)), dict(q=dict(out=1 << 50, out_row_stride=64, out_head_stride=640)),
                 dict(q=dict(row_stride=64, head_stride=2560, out_row_stride=64, out_head_stride=2560), k=dict(x=q + 1280, out=q + 1280, row_stride=64, head_stride=2560, out_row_stride=64, out_head_stride=2560)),
                 dict(axes=1, position_stride=3), dict(q=dict(x=q + 2, out=q + 2)), dict(t=1, q=dict(row_stride=5, out_row_stride=7))):
        assert head_norms(ctx, **over) == LAUNCH, over


# ------------------------------------------------------------------ experts

def pool(**over):
    mem = Memory()
    v = dict(gate_up=mem.take(1 << 22), down=mem.take(1 << 22), gate_up_bias=mem.take(1 << 16), down_bias=mem.take(1 << 16), shared_gate_up=mem.take(1 << 20), shared_down=mem.take(1 << 20),
             shared_gate=mem.take(1 << 12), num_experts=8, top_k=2, d=64, f=32, shared_f=16, activation=1)
    v.update(over)
    return _capi.Bf16ExpertPool(**v)


def experts(ctx, p=None, **over):
    p = p or pool()
    mem = Memory()
    mem.at = 1 << 44
    v = dict(x=mem.take(1 << 20), x_stride=0, idx=mem.take(1 << 12), w=mem.take(1 << 12), residual=mem.take(1 << 20), residual_stride=0, t=5, y=mem.take(1 << 20), y_stride=0,
             ws=mem.take(1 << 22), ws_bytes=1 << 22)
    if callable(over.get("at")):
        v.update(over.pop("at")(v))
    v.update(over)
    return _capi.lib().mf_bf16_experts(ctx, None, C.byref(p), v["x"], v["x_stride"], v["idx"], v["w"], v["residual"], v["residual_stride"], v["t"], v["y"], v["y_stride"], v["ws"], v["ws_bytes"])


@pytest.mark.parametrize("over, status", [
    (dict(num_experts=0), DIMENSION), (dict(num_experts=513), DIMENSION), (dict(top_k=0), DIMENSION), (dict(top_k=9), DIMENSION), (dict(d=60), DIMENSION), (dict(d=0), DIMENSION), (dict(f=4), DIMENSION),
    (dict(f=(1 << 20) + 8), DIMENSION), (dict(shared_f=12), DIMENSION), (dict(activation=4), INVALID), (dict(gate_up=None), INVALID), (dict(down=None), INVALID), (dict(shared_gate_up=None), INVALID),
    (dict(shared_down=None), INVALID), (dict(gate_up=(1 << 50) + 8), INVALID), (dict(down=(1 << 50) + 2), INVALID), (dict(shared_gate_up=(1 << 50) + 8), INVALID),
    (dict(shared_down=(1 << 50) + 8), INVALID), (dict(gate_up_bias=(1 << 50) + 1), INVALID), (dict(down_bias=(1 << 50) + 1), INVALID), (dict(shared_gate=(1 << 50) + 1), INVALID),
])
def test_experts_refuse_pools(ctx, over, status):
    assert experts(ctx, pool(**over)) == status
    assert status != DIMENSION or _capi.lib().mf_bf16_experts_workspace_bytes(C.byref(pool(**over)), 5) == 0


@pytest.mark.parametrize("over, status", [
    (dict(t=65), COUNT), (dict(t=0), OK), (dict(x=None), INVALID), (dict(idx=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID), (dict(ws=None), INVALID), (dict(x=(1 << 50) + 1), INVALID),
    (dict(idx=(1 << 50) + 2), INVALID), (dict(w=(1 << 50) + 2), INVALID), (dict(residual=(1 << 50) + 1), INVALID), (dict(y=(1 << 50) + 1), INVALID), (dict(ws=(1 << 50) + 8), INVALID),
    (dict(x_stride=63), DIMENSION), (dict(y_stride=63), DIMENSION), (dict(residual_stride=63), DIMENSION),
])
def test_experts_refuse(ctx, over, status):
    assert experts(ctx, **over) == status


def test_experts_refuse_shared_memory_and_small_workspaces(ctx):
    p = pool()
    need = _capi.lib().mf_bf16_experts_workspace_bytes(C.byref(p), 5)
    assert experts(ctx, ws_bytes=need - 1) == SCRATCH
    for name in ("gate_up", "down", "gate_up_bias", "down_bias", "shared_gate_up", "shared_down", "shared_gate"):
        assert experts(ctx, y=getattr(p, name)) == INVALID, name
        assert experts(ctx, ws=getattr(p, name)) == INVALID, name
    for name in ("x", "idx", "w", "ws"):
        assert experts(ctx, at=lambda v, n=name: {"y": v[n]}) == INVALID, name
    for name in ("x", "idx", "w", "residual"):
        assert experts(ctx, at=lambda v, n=name: {"ws": v[n]}) == INVALID, name
    assert experts(ctx, at=lambda v: {"residual": v["y"] + 64}) == INVALID
    assert experts(ctx, at=lambda v: {"residual": v["y"], "residual_stride": 128}) == INVALID
    assert _capi.lib().mf_bf16_experts(None, None, C.byref(p), None, 0, None, None, None, 0, 0, None, 0, None, 0) == INVALID
    assert _capi.lib().mf_bf16_experts(ctx, None, None, None, 0, None, None, None, 0, 0, None, 0, None, 0) == INVALID


@pytest.mark.parametrize("over", [dict(), dict(shared_f=0), dict(num_experts=512, top_k=8), dict(f=2048, d=4096, shared_f=2048), dict(num_experts=1, top_k=8)])
def test_experts_workspace_serves_fewer_rows(over):
    lib = _capi.lib()
    sizes = [lib.mf_bf16_experts_workspace_bytes(C.byref(pool(**over)), t) for t in range(1, 65)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.mf_bf16_experts_workspace_bytes(C.byref(pool(**over)), 65) == 0


@needs_no_device
def test_experts_accept(ctx):
    for over in (dict(), dict(residual=None), dict(t=64), dict(at=lambda v: {"residual": v["y"]}), dict(x=(1 << 50) + 2), dict(x_stride=128, y_stride=100)):
        assert experts(ctx, **over) == LAUNCH, over
    none = dict(gate_up_bias=None, down_bias=None)
    assert experts(ctx, pool(**none)) == LAUNCH
    assert experts(ctx, pool(**none, shared_f=0, shared_gate_up=None, shared_down=None, shared_gate=None)) == LAUNCH


# ------------------------------------------------------------------ the operators in Python

def test_packed_arguments_are_the_structures():
    values = tuple(range(1 << 40, (1 << 40) + 5)) + tuple(range(7, 14)) + (1, 0, 2)
    assert ops.Projection._pack(*values) == bytes(_capi.ProjectArgs(*values))
    q, k = (1 << 40, 1 << 41, 1 << 42, 4, 5, 6, 7, 8), (1 << 43, 1 << 44, 1 << 45, 9, 10, 11, 12, 13)
    rest = (1 << 46, 1 << 47, 1 << 48, 1, 2, 3, 4, 5, 1, 0.5, 0.25, 2.0)
    assert ops.HeadNorms._pack(*q, *k, *rest) == bytes(_capi.HeadNormsArgs(_capi.HeadRows(*q), _capi.HeadRows(*k), *rest))


class Context:
    """a context of a device that tensors here do not lie on"""
    device = torch.device("cuda", 0)
    handle = None


def test_operators_refuse_before_the_library():
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    for call in (lambda: ops.Projection(Context, b(4)), lambda: ops.Projection(Context, b(5, 8), gated=True), lambda: ops.Projection(Context, b(0, 8)),
                 lambda: ops.Projection(Context, b(4, 8), activation=4),
                 lambda: ops.HeadNorms(Context, 0), lambda: ops.HeadNorms(Context, 1025), lambda: ops.HeadNorms(Context, 8, torch.zeros(5)), lambda: ops.HeadNorms(Context, 8, torch.zeros(0)),
                 lambda: ops.HeadNorms(Context, 8, axis_of_pair=torch.zeros(4, dtype=torch.uint8)), lambda: ops.HeadNorms.axes_of_sections(()), lambda: ops.HeadNorms.axes_of_sections((1, -1)),
                 lambda: ops.HeadNorms(Context, 8).encode(b(3, 8)), lambda: ops.HeadNorms(Context, 8).encode(b(3, 2, 8), k_out=b(3, 2, 8)),
                 lambda: ops.HeadNorms(Context, 8).encode(b(3, 2, 7)), lambda: ops.HeadNorms(Context, 8).encode(b(3, 2, 16)[..., ::2]), lambda: ops.HeadNorms(Context, 8).encode(b(1, 2, 8).expand(3, 2, 8)),
                 lambda: ops.Bf16Experts(Context, b(4, 16, 8), b(4, 8, 9), 2), lambda: ops.Bf16Experts(Context, b(4, 15, 8), b(4, 8, 7), 2), lambda: ops.Bf16Experts(Context, b(4, 16, 8), b(4, 8, 8), 9),
                 lambda: ops.Bf16Experts(Context, b(4, 16, 12), b(4, 12, 8), 2), lambda: ops.Bf16Experts(Context, b(4, 16, 8), b(4, 8, 8), 2, shared_down=b(8, 8)),
                 lambda: ops.Bf16Experts(Context, b(4, 16, 8), b(4, 8, 8), 2, shared_gate=b(8))):
        with pytest.raises(ops.MfError):
            call()
    for call in (lambda: ops.Projection(Context, b(4, 8)), lambda: ops.HeadNorms(Context, 8, torch.zeros(4)), lambda: ops.HeadNorms(Context, 8, q_weight=b(8)),
                 lambda: ops.HeadNorms(Context, 8).encode(b(3, 2, 8)), lambda: ops.Bf16Experts(Context, b(4, 16, 8), b(4, 8, 8), 2)):
        with pytest.raises(ValueError):  # not on the device
            call()
