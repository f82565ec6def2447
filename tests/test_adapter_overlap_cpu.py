"""mf_adapter_apply refuses results or a workspace that share memory with what the call reads (the pool, its tables, the rows' adapters, the
plan, x) or with each other: such a call would read what other workgroups write.  Host arithmetic, no device."""
import ctypes as C

import pytest
import torch

from mference_amd import _capi
from test_adapters_cpu import INVALID, LAUNCH, OK, Memory, apply, apply_args, ctx, pool  # noqa: F401

needs_no_device = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the accepted calls would be launched")

T, M = 5, 96


def full_args(**over):
    """a call with everything it can be given; sizes: bytes of each block"""
    mem = Memory()
    mem.at = 1 << 46  # apart from what apply_args places
    p = pool(ranks=mem.take(16), scales=mem.take(16))
    a = apply_args(t=T, m=(M,), p=p, **over)
    a["keep"] = p
    plan_bytes = _capi.lib().mf_adapter_plan_bytes(T, p.num_adapters)
    a["plan"] = 1 << 45
    g = a["targets"][0]
    blocks = {"a": (g.a, p.num_adapters * p.rank * p.n * 2), "b": (g.b, p.num_adapters * M * p.rank * 2), "ids": (a["ids"], 4 * T), "ranks": (p.ranks, 4 * p.num_adapters),
              "scales": (p.scales, 4 * p.num_adapters), "plan": (a["plan"], plan_bytes), "x": (a["x"], 2 * p.n * T)}
    return a, blocks


BLOCKS = ["a", "b", "ids", "ranks", "scales", "plan", "x"]


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("f32", [0, 1])
def test_results_on_what_is_read(ctx, block, f32):  # noqa: F811
    a, blocks = full_args(f32=f32)
    size = 4 if f32 else 2
    p, n = blocks[block]
    for y in (p, p + (n - 1) // 4 * 4, p - size * T * M + 4):  # on it, by its last word, by its first
        a["targets"][0].y = y
        assert apply(ctx, a) == INVALID, (block, y - p)


@pytest.mark.parametrize("block", BLOCKS)
def test_workspace_on_what_is_read(ctx, block):  # noqa: F811
    a, blocks = full_args()
    p, n = blocks[block]
    for ws in ((p + 15) // 16 * 16, (p + n - 1) // 16 * 16, (p - a["ws_bytes"] + 16) // 16 * 16):
        if p - a["ws_bytes"] < ws < p + n:
            assert apply(ctx, {**a, "ws": ws}) == INVALID, (block, ws - p)


def test_workspace_on_the_results(ctx):  # noqa: F811
    a, _ = full_args()
    y, n = a["targets"][0].y, 2 * T * M
    for ws in (y, (y + n - 1) // 16 * 16, y - a["ws_bytes"] + 16):
        assert apply(ctx, {**a, "ws": ws // 16 * 16}) == INVALID, ws - y


@needs_no_device
def test_what_only_touches_is_taken(ctx):  # noqa: F811
    a, blocks = full_args()
    assert apply(ctx, a) == LAUNCH
    for block, (p, n) in blocks.items():
        y = a["targets"][0].y
        for at in (p + (n + 15) // 16 * 16, p - 2 * T * M):
            a["targets"][0].y = at
            assert apply(ctx, a) == LAUNCH, block
        a["targets"][0].y = y
        assert apply(ctx, {**a, "ws": p + (n + 15) // 16 * 16}) == LAUNCH, block
    # what the call reads, or its workspace, in the columns of the results' buffer that are not the results'
    a, _ = full_args(y_strides=(M + 1024,))
    y = a["targets"][0].y
    assert apply(ctx, {**a, "ids": y + 2 * M}) == LAUNCH and apply(ctx, {**a, "ids": y + 2 * M + 2 * (M + 1024)}) == LAUNCH
    assert apply(ctx, {**a, "ids": y + 2 * M - 4}) == INVALID and apply(ctx, {**a, "ids": y + 2 * (M + 1024) - 4 * T + 4}) == INVALID
    assert apply(ctx, {**a, "ids": y - 4 * T}) == LAUNCH and apply(ctx, {**a, "ids": y - 4 * T + 4}) == INVALID
    last = y + 2 * (T - 1) * (M + 1024)
    assert apply(ctx, {**a, "ids": last + 2 * M}) == LAUNCH and apply(ctx, {**a, "ids": last + 2 * M - 4}) == INVALID
    # more workspace than the call asks for: only what it uses counts
    a, _ = full_args()
    assert apply(ctx, {**a, "ws": a["x"] - (a["ws_bytes"] + 15) // 16 * 16, "ws_bytes": 1 << 20}) == LAUNCH


def test_a_batch_without_rows(ctx):  # noqa: F811
    a, _ = full_args()
    assert apply(ctx, {**a, "t": 0, "ws": a["targets"][0].y}) == OK
