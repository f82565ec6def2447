"""The workspace of mf_project and mf_bf16_experts against everything else of a call: refused exactly where they share a byte.  Host arithmetic, no device; the
buffers lie 2^40 bytes apart, so that a refusal is one of the two that were brought together.  A call that passes every check reaches the HIP
runtime, which has no device here (such calls are not made where there is one: no kernel may see these addresses)."""
import ctypes as C

import pytest
import torch

from mference_amd import _capi

INVALID, LAUNCH = -1, -7

pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the accepted calls would be launched")


@pytest.fixture
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def apart(*names):
    """an address for each, 2^40 bytes apart"""
    return {name: (k + 1) << 40 for k, name in enumerate(names)}


T, M, N = 20, 64, 65536


def project(ctx, **over):
    v = dict(apart("x", "w", "bias", "residual", "y", "ws"), t=T, m=M, n=N, x_stride=0, w_stride=0, residual_stride=0, y_stride=0, y_f32=0, gated=0, activation=0)
    v.update(over)
    need = _capi.lib().mf_project_workspace_bytes(v["m"], v["n"], v["t"], v["gated"])
    ws = v.pop("ws")
    return _capi.lib().mf_project(ctx, None, C.byref(_capi.ProjectArgs(**v)), ws, need)


def test_the_untouched_call_needs_a_workspace_and_is_taken(ctx):
    assert _capi.lib().mf_project_workspace_bytes(M, N, T, 0) > 0
    for over in (dict(), dict(gated=1), dict(y_f32=1)):
        assert project(ctx, **over) == LAUNCH


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("name, size", [("x", 2 * T * N), ("w", 2 * M * N), ("bias", 2 * M), ("residual", 2 * T * M), ("y", 2 * T * M)])
def test_the_workspace_of_a_projection(ctx, gated, name, size):
    size *= 2 if gated and name in ("w", "bias") else 1
    need = _capi.lib().mf_project_workspace_bytes(M, N, T, gated)
    at = apart("x", "w", "bias", "residual", "y", "ws")[name]
    assert size % 16 == 0 and need % 16 == 0
    for ws, want in ((at, INVALID), (at + size - 16, INVALID), (at - need + 16, INVALID), (at + size, LAUNCH), (at - need, LAUNCH)):
        assert project(ctx, ws=ws, gated=gated) == want, hex(ws)


@pytest.mark.parametrize("name", ["x", "w", "bias"])
def test_the_results_of_a_projection(ctx, name):
    size = {"x": 2 * T * N, "w": 2 * M * N, "bias": 2 * M}[name]
    at, own = apart("x", "w", "bias", "residual", "y", "ws")[name], 2 * T * M
    for y, want in ((at, INVALID), (at + size - 2, INVALID), (at - own + 2, INVALID), (at + size, LAUNCH), (at - own, LAUNCH)):
        assert project(ctx, y=y) == want, hex(y)


def test_the_residual_of_a_projection(ctx):
    y, own = apart("x", "w", "bias", "residual", "y", "ws")["y"], 2 * T * M
    for residual, want in ((y, LAUNCH), (y + 2, INVALID), (y - 2, INVALID), (y + own - 2, INVALID), (y + own, LAUNCH), (y - own, LAUNCH)):
        assert project(ctx, residual=residual) == want, hex(residual)


ROUTES, D, F, FS, EXPERTS = 40, 256, 64, 32, 8
POOL = ("gate_up", "down", "gate_up_bias", "down_bias", "shared_gate_up", "shared_down", "shared_gate")
SIZES = dict(gate_up=4 * EXPERTS * F * D, down=2 * EXPERTS * F * D, gate_up_bias=4 * EXPERTS * F, down_bias=2 * EXPERTS * D, shared_gate_up=4 * FS * D, shared_down=2 * FS * D, shared_gate=2 * D,
             x=2 * 20 * D, idx=4 * ROUTES, w=4 * ROUTES, residual=2 * 20 * D, y=2 * 20 * D)


def experts(ctx, **over):
    v = dict(apart(*POOL, "x", "idx", "w", "residual", "y", "ws"))
    v.update(over)
    p = _capi.Bf16ExpertPool(**{n: v[n] for n in POOL}, num_experts=EXPERTS, top_k=2, d=D, f=F, shared_f=FS, activation=1)
    need = _capi.lib().mf_bf16_experts_workspace_bytes(C.byref(p), 20)
    return _capi.lib().mf_bf16_experts(ctx, None, C.byref(p), v["x"], 0, v["idx"], v["w"], v["residual"], 0, 20, v["y"], 0, v["ws"], need), need


@pytest.mark.parametrize("name", SIZES)
def test_the_workspace_of_experts(ctx, name):
    got, need = experts(ctx)
    assert got == LAUNCH and need % 16 == 0
    at, size = apart(*POOL, "x", "idx", "w", "residual", "y", "ws")[name], SIZES[name]
    for ws, want in ((at, INVALID), (at + size - 16, INVALID), (at - need + 16, INVALID), (at + size, LAUNCH), (at - need, LAUNCH)):
        assert experts(ctx, ws=ws)[0] == want, hex(ws)


@pytest.mark.parametrize("name", [n for n in SIZES if n not in ("y", "residual")])
def test_the_results_of_experts(ctx, name):
    at, size, own = apart(*POOL, "x", "idx", "w", "residual", "y", "ws")[name], SIZES[name], SIZES["y"]
    for y, want in ((at, INVALID), (at + size - 2, INVALID), (at - own + 2, INVALID), (at + size, LAUNCH), (at - own, LAUNCH)):
        assert experts(ctx, y=y)[0] == want, hex(y)
