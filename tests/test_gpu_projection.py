"""mf_project on the GPU against the definition in 64 bits."""
import pytest
import torch

from dense16_cases import ACTS, Placed, assert_near, generator, ints, project64, randn
from mference_amd import operators as ops

pytestmark = pytest.mark.gpu

SIZES = [  # t, n, m: one row to several tiles, one element to several steps, whole and broken pieces of eight
    (1, 1, 1), (1, 8, 16), (1, 64, 64), (1, 136, 33), (1, 2048, 512), (1, 1000, 129), (2, 33, 17), (3, 7, 5), (4, 5120, 256), (5, 320, 1000), (8, 4104, 96),
    (15, 64, 48), (16, 256, 128), (16, 8200, 64), (17, 256, 128), (20, 1000, 96), (31, 96, 130), (33, 520, 257), (48, 2048, 192), (63, 129, 65), (64, 512, 512), (65, 64, 72),
    (100, 1, 100), (100, 777, 321), (127, 200, 128), (128, 1024, 256), (129, 1032, 250), (200, 2816, 113), (255, 64, 256), (256, 256, 256), (257, 96, 264), (300, 2048, 512),
    (513, 136, 384), (777, 640, 260), (1024, 512, 1024), (1030, 1288, 1100), (2050, 256, 136),
]


def make(t, n, m, exact=False, gated=False, bias=True, residual=True, dtype=torch.bfloat16, pad=0, off=0, seed=0):
    g = generator(1000 * seed + 7 * t + 3 * n + m)
    rows = 2 * m if gated else m
    few = 3 if n < 8000 else 2  # sums of so many products of whole numbers stay below 2^24
    x = ints(g, few, t, n) if exact else randn(g, t, n)
    w = ints(g, few, rows, n) if exact else randn(g, rows, n) * n ** -0.5
    b = (ints(g, 50, rows) if exact else randn(g, rows)).bfloat16() if bias else None
    r = (ints(g, 100, t, m) if exact else randn(g, t, m)).to(dtype) if residual else None
    return (Placed(x.bfloat16(), pad, off), Placed(w.bfloat16(), pad, off), b, None if r is None else Placed(r, pad, off),
            Placed(torch.zeros((t, m), dtype=dtype, device="cuda"), pad, off, 7.0))


@pytest.mark.parametrize("t, n, m", SIZES)
@pytest.mark.parametrize("f32", [False, True])
def test_whole_numbers(gpu, t, n, m, f32):
    """sums of whole numbers are exact: the result is the one rounding of theirs"""
    x, w, b, r, y = make(t, n, m, exact=True, dtype=torch.float32 if f32 else torch.bfloat16)
    ops.Projection(gpu, w.rows, bias=b).encode(x.rows, y.rows, residual=r.rows)
    want, _ = project64(x.rows, w.rows, b, r.rows, "none", False)
    assert torch.equal(y.rows.float(), want.to(y.rows.dtype).float())
    assert y.only_rows_changed()


@pytest.mark.parametrize("place, t, n, m", [(i, *s) for i, s in enumerate(SIZES)])
def test_forms(gpu, place, t, n, m):
    """activations, gates, bias, residual, types and strides in turn over the sizes"""
    for turn in range(4):
        k = place + 5 * turn
        act, gated, bias, residual = ACTS[(k + turn) % 4], (k // 2 + turn) % 2 == 1, k % 3 != 0, k % 5 < 3
        dtype = torch.float32 if k % 4 == 1 else torch.bfloat16
        pad, off = ((0, 0), (16, 8), (3, 1), (8, 0), (1, 5))[(k + turn) % 5]
        x, w, b, r, y = make(t, n, m, gated=gated, bias=bias, residual=residual, dtype=dtype, pad=pad, off=off, seed=turn)
        op = ops.Projection(gpu, w.rows, bias=b, activation=ACTS.index(act), gated=gated)
        op.encode(x.rows, y.rows, residual=None if r is None else r.rows)
        want, far = project64(x.rows, w.rows, b, None if r is None else r.rows, act, gated)
        assert_near(y.rows, want, far, (act, gated, bias, residual, dtype, pad, off))
        assert y.only_rows_changed()
        again = Placed(torch.zeros((t, m), dtype=dtype, device="cuda"), pad, off, 7.0)
        op.encode(x.rows, again.rows, residual=None if r is None else r.rows)
        assert torch.equal(again.rows, y.rows)


@pytest.mark.parametrize("t, n, m, gated", [(1, 256, 100, False), (9, 512, 64, True), (40, 320, 48, False), (300, 256, 320, True), (520, 1024, 512, False)])
def test_in_place(gpu, t, n, m, gated):
    x, w, b, r, _ = make(t, n, m, gated=gated, pad=8)
    want, far = project64(x.rows, w.rows, b, r.rows, "silu", gated)
    ops.Projection(gpu, w.rows, bias=b, activation=ops.ACT_SILU, gated=gated).encode(x.rows, r.rows, residual=r.rows)
    assert_near(r.rows, want, far)
    assert r.only_rows_changed()


@pytest.mark.parametrize("t", [1, 16, 40, 130, 600])
def test_infinities_stay_with_their_row_and_column(gpu, t):
    n, m = 520, 150
    x, w, b, _, y = make(t, n, m, residual=False)
    row, col = t // 2, 77
    x.rows[row, 13] = float("inf")
    w.rows[col, 5] = float("nan")
    ops.Projection(gpu, w.rows, bias=b).encode(x.rows, y.rows)
    rows = torch.arange(t, device="cuda") != row
    cols = torch.arange(m, device="cuda") != col
    assert not torch.isfinite(y.rows[row]).any() and torch.isnan(y.rows[:, col]).all()
    assert torch.isfinite(y.rows[rows][:, cols]).all()
    want, far = project64(x.rows[rows], w.rows[cols], b[cols], None, "none", False)
    assert_near(y.rows[rows][:, cols], want, far)


@pytest.mark.parametrize("act", range(1, 4))
def test_activations_far_out(gpu, act):
    """large arguments of either sign: nothing, or the argument"""
    n = m = 64
    big = torch.zeros(1, n, device="cuda")
    big[0, 0] = 1.0
    w = torch.zeros(m, n, device="cuda")
    w[:, 0] = torch.tensor([s * 2.0 ** e for e in range(0, 128, 4) for s in (1, -1)], device="cuda")
    y = torch.empty(1, m, dtype=torch.bfloat16, device="cuda")
    ops.Projection(gpu, w.bfloat16(), activation=act).encode(big.bfloat16(), y)
    z = w[:, 0]
    far = z.abs() > 20  # (the smaller ones: test_forms)
    assert torch.equal(y[0].float()[far], torch.where(z > 0, z, torch.zeros_like(z))[far])


@pytest.mark.parametrize("t, n, m", [(1, 2048, 256), (12, 17408, 64), (33, 4096, 64), (200, 2816, 113), (300, 5120, 256), (600, 512, 512)])
def test_captured_graph(gpu, t, n, m):
    """replays between other work, with new inputs in the same memory: the eager call's bits"""
    x, w, b, r, y = make(t, n, m, gated=True, pad=8)
    op = ops.Projection(gpu, w.rows, bias=b, activation=ops.ACT_SILU, gated=True)
    ws = torch.empty(max(op.workspace_bytes(t), 16), dtype=torch.uint8, device="cuda")
    op.encode(x.rows, y.rows, residual=r.rows, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.encode(x.rows, y.rows, residual=r.rows, workspace=ws)
    other = torch.empty_like(ws)
    for k in range(4):
        x.rows.copy_(randn(generator(k), t, n).bfloat16())
        ws.fill_(255)
        graph.replay()
        got = y.rows.clone()
        y.rows.zero_()
        op.encode(x.rows, y.rows, residual=r.rows, workspace=other)
        torch.cuda.synchronize()
        assert torch.equal(got, y.rows)


def test_another_stream(gpu):
    t, n, m = 300, 2048, 512
    x, w, b, r, y = make(t, n, m)
    side = torch.cuda.Stream()
    op = ops.Projection(gpu, w.rows, bias=b)
    torch.cuda.synchronize()
    op.encode(x.rows, y.rows, residual=r.rows, stream=side)
    side.synchronize()
    want, far = project64(x.rows, w.rows, b, r.rows, "none", False)
    assert_near(y.rows, want, far)


def test_a_workspace_for_many_rows_serves_fewer(gpu):
    n, m = 4096, 256
    most = 0
    op = None
    for t in (600, 130, 60, 20, 7, 1):
        x, w, b, r, y = make(t, n, m)
        op = ops.Projection(gpu, w.rows, bias=b)
        most = most or op.workspace_bytes(600)
        assert op.workspace_bytes(t) <= most
        op.encode(x.rows, y.rows, residual=r.rows, workspace=torch.full((max(most, 16),), 255, dtype=torch.uint8, device="cuda"))
        want, far = project64(x.rows, w.rows, b, r.rows, "none", False)
        assert_near(y.rows, want, far)


def test_rows_past_4_gib(gpu):
    """offsets that pass 32 bits: the last rows of a long x and a long y"""
    t, n, m = 70000, 64, 64
    wide = 32768 + 64
    x = torch.zeros(t, wide, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(t, wide, dtype=torch.bfloat16, device="cuda")
    g = generator(5)
    w = ints(g, 3, m, n).bfloat16()
    x[:, :n] = ints(g, 3, t, n).bfloat16()
    ops.Projection(gpu, w).encode(x[:, :n], y[:, :m])
    want = x[:, :n].float() @ w.float().t()
    assert torch.equal(y[:, :m], want.bfloat16()) and not y[:, m:].any()
