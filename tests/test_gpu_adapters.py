"""mf_adapter_apply and mf_adapter_group on the GPU, against plain implementations in 64 bits.

Two kinds of inputs.  Whole numbers small enough that every product and every partial sum is exact in fp32 (and A x in the bf16
terms it is cut into): the fp32 result is then the exact one in any order of summation, and the bf16 result its correct rounding,
so both are compared bit for bit.  Normal numbers, compared within a bound:
  |y - y64| <= half a step of the result's type + slack,
  slack = (E + T) * S,  S = |c| |B| (|A| |x|), the sum of the magnitudes that meet in the result,
  E = 2 (n + rank + 64) 2^-24: an fp32 sum of n products is off by at most n half steps of its magnitudes whatever its order, and
      so are the sum over the rank, the joining of parts of the sum over n, and the scale; T: what the bf16 terms of A x leave out,
      2^-15 for bf16 results, nothing for fp32 ones.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from mference_amd import operators as ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_ids(order, t, adapters, bare=0.0, seed=0):
    r = np.random.RandomState(seed)
    if order == "one":
        ids = np.full(t, r.randint(adapters))
    elif order == "mixed":
        ids = r.randint(0, adapters, t)
    else:
        ids = np.repeat(r.randint(0, adapters, t), r.randint(1, max(2, t // 3), t))[:t]
    ids = np.where(r.random_sample(t) < bare, r.choice([-1, adapters, -2 ** 31, 2 ** 31 - 1], t), ids)
    return torch.from_numpy(ids.astype(np.int32)).cuda()


class Case:
    """x, pool and results; whole: whole numbers.  pad: columns around x and the ys in wider buffers; off: elements by which they
    start behind a 16-byte border."""

    def __init__(self, t, n, ms, adapters, rank, whole=True, dtype=torch.bfloat16, ranks="full", scales=True, pad=0, off=0, seed=1, wide=False):
        g = gen(seed)
        ints = lambda k, *s: torch.randint(-k, k + 1, s, generator=g, device="cuda").float()  # noqa: E731
        norm = lambda k, *s: torch.randn(s, generator=g, device="cuda") * k  # noqa: E731
        self.t, self.n, self.ms, self.adapters, self.rank, self.dtype = t, n, ms, adapters, rank, dtype
        if whole:
            # |A x| <= 4 n (wide: up to 3600 n < 2^24), in the mean 2 sqrt(n); c 1 or 2; |c B A x| <= 8 rank n (wide: one live column)
            kx, ka, kb = (60, 60, 1) if wide else (2, 2, 1)
            x, a, b = ints(kx, t, n), [ints(ka, adapters, rank, n) for _ in ms], [ints(kb, adapters, m, rank) for m in ms]
            if wide:
                for w in b:
                    w[:, :, 1:] = 0
            c = 2.0 ** torch.randint(0, 2, (adapters,), generator=g, device="cuda").float()
            ys = [ints(100, t, m) for m in ms]
        else:
            x, a, b = norm(1, t, n), [norm(n ** -0.5, adapters, rank, n) for _ in ms], [norm(0.1, adapters, m, rank) for m in ms]
            c = norm(1, adapters)
            ys = [norm(1, t, m) for m in ms]
        self.a, self.b = [w.bfloat16() for w in a], [w.bfloat16() for w in b]
        self.scales = c if scales else None
        self.ranks = None
        if ranks == "mixed":
            self.ranks = torch.randint(0, rank + 1, (adapters,), generator=g, device="cuda", dtype=torch.int32)
            self.ranks[0] = rank
            for k, r in enumerate(self.ranks.tolist()):  # what lies beyond an adapter's rank is never used
                for wa, wb in zip(self.a, self.b):
                    wa[k, r:] = float("nan")
                    wb[k, :, r:] = float("inf")
        self.x = self._placed(x.bfloat16(), pad, off)
        self.ys = [self._placed(y.to(dtype), pad, off) for y in ys]
        self.around = [y.clone() for y in self.buffers[1:]]

    def _placed(self, v, pad, off):
        if not hasattr(self, "buffers"):
            self.buffers, self.places = [], []
        t, w = v.shape
        stride = w + pad
        flat = torch.full((off + t * stride + 8,), 7.0, dtype=v.dtype, device="cuda")
        rows = flat[off:off + t * stride].view(t, stride)[:, pad // 2:pad // 2 + w]
        rows.copy_(v)
        self.buffers.append(flat)
        self.places.append(rows)
        return rows

    def expected(self, ids):
        """(results in 64 bits, sums of magnitudes, which rows have an adapter)"""
        ids = ids.cpu()
        out = []
        live = (ids >= 0) & (ids < self.adapters)
        for a, b, y in zip(self.a, self.b, self.ys):
            y, s = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
            for k in range(self.adapters):
                at = (ids == k).nonzero()[:, 0].cuda()
                if not at.numel():
                    continue
                r = self.rank if self.ranks is None else int(self.ranks[k])
                c = 1.0 if self.scales is None else self.scales[k].double()
                x, wa, wb = self.x[at].double(), a[k, :r].double(), b[k, :, :r].double()
                y[at] += c * ((x @ wa.t().contiguous()) @ wb.t().contiguous())
                s[at] += abs(c) * ((x.abs() @ wa.abs().t().contiguous()) @ wb.abs().t().contiguous())
            out.append((y, s))
        return out, live.cuda()

    def check(self, gpu, ids, plan, whole=True, **kw):
        want, live = self.expected(ids)
        before = [y.clone() for y in self.ys]
        op = ops.LowRankAdapters(gpu, self.a, self.b, scales=self.scales, ranks=self.ranks)
        p = ops.AdapterGrouping(gpu, self.adapters).encode(ids) if plan else None
        op.encode(self.x, ids, self.ys, plan=p, **kw)
        torch.cuda.synchronize()
        for y, was, (w, s) in zip(self.ys, before, want):
            assert torch.equal(y[~live].view(torch.int16 if y.dtype == torch.bfloat16 else torch.int32), was[~live].view(torch.int16 if y.dtype == torch.bfloat16 else torch.int32)), \
                "a row without an adapter changed"
            if whole:
                assert torch.equal(y[live], w[live].to(self.dtype)), (y[live].double() - w[live]).abs().max()
            else:
                e = 2 * (self.n + self.rank + 64) * 2.0 ** -24 + (2.0 ** -15 if self.dtype == torch.bfloat16 else 0.0)
                off = (y.double() - w).abs() - HALF[self.dtype] * w.abs() - e * s
                assert off.max() <= 0, (off.max(), (y.double() - w).norm() / w.norm())
        for flat, was, rows in zip(self.buffers[1:], self.around, self.places[1:]):  # what lies around the results
            keep = rows.clone()
            rows.copy_(was.as_strided(rows.shape, rows.stride(), rows.storage_offset()))
            assert torch.equal(flat, was), "written outside of the result's rows"
            rows.copy_(keep)


# ------------------------------------------------------------------ rows by adapter

@pytest.mark.parametrize("t", [0, 1, 2, 63, 64, 65, 200, 1023, 1025, 4096, 4097, 70001])
@pytest.mark.parametrize("adapters", [1, 2, 48, 1024])
def test_grouping(gpu, t, adapters):
    grouping = ops.AdapterGrouping(gpu, adapters)
    plan = None
    for k, (order, bare) in enumerate([("mixed", 0.0), ("runs", 0.2), ("one", 0.0), ("mixed", 1.0)]):
        ids = make_ids(order, max(t, 1), adapters, bare, seed=k)[:t].contiguous()
        plan = grouping.encode(ids, plan)
        torch.cuda.synchronize()
        v = ids.cpu().numpy()
        key = np.where((v >= 0) & (v < adapters), v, adapters)
        assert np.array_equal(plan.rows.cpu().numpy(), np.argsort(key, kind="stable")), (order, bare)
        assert np.array_equal(plan.offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(adapters + 1))), (order, bare)


def test_grouping_of_the_largest_batch(gpu):
    t, adapters = 1 << 20, 1000
    ids = make_ids("mixed", t, adapters, 0.1, seed=9)
    plan = ops.AdapterGrouping(gpu, adapters).encode(ids)
    v = ids.cpu().numpy()
    key = np.where((v >= 0) & (v < adapters), v, adapters)
    assert np.array_equal(plan.rows.cpu().numpy(), np.argsort(key, kind="stable"))
    assert np.array_equal(plan.offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(adapters + 1)))


def test_grouping_writes_its_words_only(gpu):
    from mference_amd import _capi
    for t, adapters in ((1, 1), (5, 3), (200, 48), (5000, 1024), (9000, 7)):
        need = _capi.lib().mf_adapter_plan_bytes(t, adapters) // 4
        words = torch.full((need + 64,), -77, dtype=torch.int32, device="cuda")
        ids = make_ids("mixed", t, adapters, 0.1)
        ops.AdapterGrouping(gpu, adapters).encode(ids, ops.AdapterPlan(t, adapters, words[:need]))
        assert bool((words[need:] == -77).all())


# ------------------------------------------------------------------ adapters

@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, n, ms, adapters, rank, order", [
    (1, 64, (1,), 1, 8, "one"), (1, 2048, (512, 512), 4, 16, "one"), (2, 128, (17,), 3, 8, "mixed"), (4, 512, (640, 640), 3, 32, "one"),
    (8, 1088, (200, 64, 136), 5, 16, "mixed"), (15, 192, (96,), 20, 24, "mixed"), (16, 320, (65,), 2, 40, "runs"), (17, 256, (129, 63), 17, 64, "mixed"),
    (33, 448, (256,), 4, 128, "runs"), (64, 704, (320, 320), 6, 16, "runs"), (65, 512, (1000,), 1, 16, "one"), (130, 128, (72, 72, 72, 72), 9, 8, "mixed"),
    (200, 640, (130, 130), 48, 24, "mixed"), (257, 1024, (512,), 3, 256, "runs"), (300, 512, (77,), 1024, 8, "mixed"), (513, 576, (192, 192), 5, 48, "runs"),
    (1500, 256, (64,), 7, 56, "mixed"), (2100, 128, (256, 256), 3, 16, "runs"),
])
def test_adapters_of_whole_numbers(gpu, t, n, ms, adapters, rank, order, dtype, plan):
    c = Case(t, n, ms, adapters, rank, dtype=dtype, seed=t + n)
    c.check(gpu, make_ids(order, t, adapters, seed=t), plan)


@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, n, ms, adapters, rank, order, bare", [
    (1, 512, (256,), 3, 16, "one", 1.0), (5, 320, (100, 40), 4, 24, "mixed", 0.4), (70, 256, (96,), 9, 40, "mixed", 0.3), (200, 384, (136, 136), 48, 24, "mixed", 0.1),
    (400, 192, (64,), 5, 64, "runs", 0.2), (1000, 128, (80,), 3, 16, "runs", 0.5)])
def test_adapters_of_several_ranks(gpu, t, n, ms, adapters, rank, order, bare, dtype, plan):
    """ranks from 0 to the whole rank, with NaN and infinities beyond them; rows without an adapter in between"""
    c = Case(t, n, ms, adapters, rank, dtype=dtype, ranks="mixed", seed=t)
    c.check(gpu, make_ids(order, t, adapters, bare, seed=t), plan)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad, off", [(0, 1), (3, 0), (8, 0), (64, 8), (5, 3), (0, 4)])
@pytest.mark.parametrize("t, n, ms", [(1, 128, (72,)), (9, 256, (131, 64)), (150, 192, (328,)), (700, 64, (96, 33))])
def test_adapters_between_other_columns(gpu, t, n, ms, pad, off, dtype):
    """rows of wider buffers, at any alignment; what lies around them stays"""
    c = Case(t, n, ms, 4, 16, dtype=dtype, pad=pad, off=off, seed=t + pad)
    c.check(gpu, make_ids("runs", t, 4, 0.1, seed=t), t > 100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_adapters_keep_the_whole_of_ax(gpu, t, dtype):
    """A x of more bits than two bf16 terms hold: fp32 results keep all of them, bf16 results are off by no more than the terms leave out"""
    c = Case(t, 4096, (40,), 2, 8, dtype=dtype, seed=t, wide=True)
    c.check(gpu, make_ids("mixed", t, 2, seed=t), t > 100, whole=dtype == torch.float32)


@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, n, ms, adapters, rank, order", [
    (1, 2048, (512, 512), 16, 16, "one"), (4, 5120, (1024, 1024), 8, 32, "one"), (8, 17408, (640,), 8, 16, "mixed"), (40, 2816, (352,), 11, 24, "mixed"), (200, 2816, (264, 264), 48, 24, "mixed"),
    (777, 1024, (520, 520), 5, 64, "runs"), (1030, 4096, (256,), 3, 16, "runs")])
def test_adapters_of_normal_numbers(gpu, t, n, ms, adapters, rank, order, dtype, plan):
    c = Case(t, n, ms, adapters, rank, whole=False, dtype=dtype, ranks="mixed", seed=t)
    c.check(gpu, make_ids(order, t, adapters, 0.1 if t > 4 else 0.0, seed=t), plan, whole=False)


@pytest.mark.parametrize("plan", [False, True])
def test_a_row_of_nan_or_infinity_stays_alone(gpu, plan):
    for t, order in ((7, "mixed"), (64, "runs"), (300, "mixed")):
        c = Case(t, 256, (96, 40), 3, 16, seed=t)
        ids = make_ids(order, t, 3, seed=t)
        want, _ = c.expected(ids)
        bad = sorted({0, t // 2, t - 1})
        for k, i in enumerate(bad):
            c.x[i, 5 * k + 1] = [float("nan"), float("inf"), -float("inf")][k % 3]
        p = ops.AdapterGrouping(gpu, 3).encode(ids) if plan else None
        ops.LowRankAdapters(gpu, c.a, c.b, scales=c.scales).encode(c.x, ids, c.ys, plan=p)
        rest = torch.ones(t, dtype=torch.bool, device="cuda")
        rest[bad] = False
        for y, (w, _) in zip(c.ys, want):
            assert torch.equal(y[rest], w[rest].bfloat16())
            assert not bool(torch.isfinite(y[bad]).all(1).any())


def test_infinity_of_x_keeps_its_sign(gpu):
    """A of ones, B of ones: an infinity of x is an infinity of the result, not a NaN, whatever A x is cut into"""
    for dtype in (torch.bfloat16, torch.float32):
        one = torch.ones(1, 16, 64, dtype=torch.bfloat16, device="cuda")
        b = torch.ones(1, 24, 16, dtype=torch.bfloat16, device="cuda")
        x = torch.ones(3, 64, dtype=torch.bfloat16, device="cuda")
        x[0, 3], x[1, 60] = float("inf"), -float("inf")
        y = torch.zeros(3, 24, dtype=dtype, device="cuda")
        ops.LowRankAdapters(gpu, one, b).encode(x, torch.zeros(3, dtype=torch.int32, device="cuda"), y)
        assert bool((y[0] == float("inf")).all()) and bool((y[1] == -float("inf")).all()) and bool((y[2] == 1024).all())


@pytest.mark.parametrize("power", [-120, -60, 60, 120])
def test_adapters_of_any_magnitude(gpu, power):
    """the whole-number case times powers of two, exact as before (subnormal bf16 numbers left aside)"""
    c = Case(20, 256, (96,), 3, 16, dtype=torch.float32, scales=False)
    ids = make_ids("mixed", 20, 3)
    want, _ = c.expected(ids)
    base = c.ys[0].double().clone()
    c.x.mul_(2.0 ** power)
    if abs(power) > 100:
        c.b[0].mul_(2.0 ** (-power // 2))
    scale = 2.0 ** (power + (-power // 2 if abs(power) > 100 else 0))
    c.ys[0].zero_()
    ops.LowRankAdapters(gpu, c.a, c.b).encode(c.x, ids, c.ys)
    assert torch.equal(c.ys[0].double(), (want[0][0] - base) * scale)


def test_rows_past_32_bits(gpu):
    """the last rows of a result of more than 2^32 elements"""
    t, m = (1 << 16) + 3, 65600
    rows = torch.zeros((t, m), dtype=torch.bfloat16, device="cuda")
    c = Case(1, 64, (m,), 2, 8, seed=4)
    x = torch.zeros((t, 64), dtype=torch.bfloat16, device="cuda")
    x[-3:] = c.x[0]
    ids = torch.full((t,), -1, dtype=torch.int32, device="cuda")
    ids[-3:] = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
    for plan in (False, True):
        rows[-4:] = 0
        p = ops.AdapterGrouping(gpu, 2).encode(ids) if plan else None
        ops.LowRankAdapters(gpu, c.a, c.b).encode(x, ids, rows, plan=p)
        for i, k in ((-3, 1), (-2, 0), (-1, 1)):
            want = c.b[0][k].double() @ (c.a[0][k].double() @ c.x[0].double())
            assert torch.equal(rows[i], want.bfloat16()), (plan, i)
        assert not bool(rows[-4].any()) and not bool(rows[:3].any())


def test_equal_calls_give_equal_bits(gpu):
    for t, order in ((1, "one"), (8, "mixed"), (200, "mixed"), (700, "runs")):
        c = Case(t, 2048, (300, 300), 12, 24, whole=False, seed=t)
        ids = make_ids(order, t, 12, seed=t)
        op, grouping = ops.LowRankAdapters(gpu, c.a, c.b, scales=c.scales), ops.AdapterGrouping(gpu, 12)
        first = None
        for k in range(4):
            ys = [y.clone() for y in c.ys]
            op.encode(c.x, ids, ys, plan=grouping.encode(ids) if t == 200 else None)
            first = first or ys
            assert all(torch.equal(a, b) for a, b in zip(first, ys))


def test_a_plan_of_other_sizes_is_refused_or_unused(gpu):
    c = Case(40, 128, (64,), 3, 16)
    ids = make_ids("mixed", 40, 3)
    op = ops.LowRankAdapters(gpu, c.a, c.b)
    with pytest.raises(ops.MfError):
        op.encode(c.x, ids, c.ys, plan=ops.AdapterGrouping(gpu, 3).plan(41))
    with pytest.raises(ops.MfError):
        op.encode(c.x, ids, c.ys, plan=ops.AdapterGrouping(gpu, 4).plan(40))
    with pytest.raises(ops.MfError):
        ops.AdapterGrouping(gpu, 3).encode(ids, ops.AdapterGrouping(gpu, 3).plan(39))
    with pytest.raises(ops.MfError):
        op.encode(c.x, ids, c.ys, workspace=torch.empty(op.workspace_bytes(40) - 4, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        op.encode(c.x.float(), ids, c.ys)
    with pytest.raises(ValueError):
        op.encode(c.x, ids.long(), c.ys)
    with pytest.raises(ValueError):
        op.encode(c.x, ids, [c.ys[0].half()])
    with pytest.raises(ops.MfError):
        op.encode(c.x, ids[:39], c.ys)
    with pytest.raises(ops.MfError):
        op.encode(c.x, ids, [c.x[:, :64]])
    op.encode(c.x[:0], ids[:0], [c.ys[0][:0]])


# ------------------------------------------------------------------ streams, threads, graphs

def test_workspace_of_a_larger_batch_and_other_streams(gpu):
    """one workspace for every smaller batch; two streams at once, each with its own buffers, and with buffers that the calls take"""
    big = Case(300, 512, (200, 200), 5, 16, seed=3)
    op, grouping = ops.LowRankAdapters(gpu, big.a, big.b, scales=big.scales), ops.AdapterGrouping(gpu, 5)
    ws = torch.empty(op.workspace_bytes(300), dtype=torch.uint8, device="cuda")
    for t in (300, 1, 17, 64, 120, 299):
        ids = make_ids("mixed", t, 5, seed=t)
        ws.fill_(255)
        ys, want = [y[:t].clone() for y in big.ys], [y[:t].clone() for y in big.ys]
        op.encode(big.x[:t], ids, ys, workspace=ws)
        op.encode(big.x[:t], ids, want)
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
    ids = make_ids("mixed", 300, 5)
    want = [y.clone() for y in big.ys]
    op.encode(big.x, ids, want, plan=grouping.encode(ids))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = [[y.clone() for y in big.ys] for _ in streams]
        torch.cuda.synchronize()
        for s, ys in zip(streams, got):
            with torch.cuda.stream(s):
                plan = grouping.encode(ids)
                op.encode(big.x, ids, ys, plan=plan)
        torch.cuda.synchronize()
        for ys in got:
            assert all(torch.equal(a, b) for a, b in zip(ys, want))
    # a stream by its handle, not the current one
    ys = [y.clone() for y in big.ys]
    torch.cuda.synchronize()
    plan = grouping.encode(ids, stream=streams[0])
    op.encode(big.x, ids, ys, plan=plan, stream=streams[0].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ys, want))


def test_captured_step(gpu):
    """grouping, adapters and block norm of a step as one graph, replayed with other rows, with eager work between the replays"""
    t, d, f = 90, 512, 384
    c = Case(t, d, (f, f), 6, 16, whole=False, seed=8)
    op, grouping, norm = ops.LowRankAdapters(gpu, c.a, c.b, scales=c.scales), ops.AdapterGrouping(gpu, 6), ops.BlockNorm(gpu)
    ids, plan = make_ids("mixed", t, 6), grouping.plan(t)
    hidden, delta, w = torch.empty(t, d, dtype=torch.bfloat16, device="cuda"), torch.empty(t, d, dtype=torch.bfloat16, device="cuda"), torch.ones(d, dtype=torch.bfloat16, device="cuda")
    x = torch.empty_like(hidden)
    ys = [torch.zeros(t, f, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def step(ids, plan, hidden, delta, x, ys):
        grouping.encode(ids, plan)
        norm.encode(hidden, delta, out=x, pre_weight=w, post_weight=w)
        op.encode(x, ids, ys, plan=plan)

    def fill(k):
        g = gen(k)
        hidden.copy_(torch.randn(t, d, generator=g, device="cuda"))
        delta.copy_(torch.randn(t, d, generator=g, device="cuda"))
        ids.copy_(make_ids("mixed", t, 6, 0.2, seed=k))
        for y in ys:
            y.zero_()

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, plan, hidden, delta, x, ys)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same calls
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(ids, plan, hidden, delta, x, ys)
        graphs.append(graph)
    for k in range(6):
        fill(k)
        eager = [v.clone() for v in (hidden, delta, x)] + [[y.clone() for y in ys]]
        step(ids.clone(), grouping.plan(t), *eager[:2], eager[2], eager[3])
        graphs[k % 2].replay()
        if k % 2:
            torch.cuda.synchronize()
        assert torch.equal(hidden, eager[0]) and torch.equal(x, eager[2]) and all(torch.equal(a, b) for a, b in zip(ys, eager[3])), k


# ------------------------------------------------------------------ a block

@pytest.mark.parametrize("t", [1, 6, 40, 150])
@pytest.mark.parametrize("d, f", [(512, 384), (256, 640)])
def test_block_with_adapters(gpu, t, d, f):
    """norm, the quantized MLP with adapters beside its projections, post norm, gate and residual: against the same block in 64 bits
    on the dequantized weights.  Narrowings on the way: x, gate and up (base, then sum), act, down (base, then sum), hidden -- nine
    roundings of 2^-9 each in the mean, whose errors the MLP passes on with about its own gain: 2 percent of the result's norm is
    ten times that."""
    g = gen(t + d)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q = ops.Quantization(gpu)
    gate, up, down = (q.quantize_affine(rn(r, k) * k ** -0.5, 4) for r, k in ((f, d), (f, d), (d, f)))
    wg, wu, wd = (q.dequantize(w).double() for w in (gate, up, down))
    n, r = 5, 16
    a = [(rn(n, r, d) * d ** -0.5).bfloat16() for _ in range(2)] + [(rn(n, r, f) * f ** -0.5).bfloat16()]
    b = [(rn(n, m, r) * 0.2).bfloat16() for m in (f, f, d)]
    scales = 0.5 + torch.rand(n, generator=g, device="cuda")
    hidden, delta, w1, w2, lw = rn(t, d).bfloat16(), rn(t, d).bfloat16(), (1 + 0.1 * rn(d)).bfloat16(), (1 + 0.1 * rn(d)).bfloat16(), rn(t, 1).bfloat16()
    ids = make_ids("mixed", t, n, 0.2, seed=t)
    # 64 bits
    lives = [int(k) if 0 <= int(k) < n else None for k in ids.tolist()]

    def adapted(w, wa, wb, x):
        y = x @ w.t().contiguous()
        for i, k in enumerate(lives):
            if k is not None:
                y[i] += scales[k].double() * (wb[k].double() @ (wa[k].double() @ x[i]))
        return y

    rms = lambda v, w: v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()  # noqa: E731
    h = hidden.double() + delta.double()
    x = rms(h, w1)
    gv, uv = adapted(wg, a[0], b[0], x), adapted(wu, a[1], b[1], x)
    y = adapted(wd, a[2], b[2], gv * torch.sigmoid(gv) * uv)
    want = h + torch.sigmoid(lw.double()) * rms(y, w2)
    # the library
    norm, mlp = ops.BlockNorm(gpu), ops.SharedExpertInt4(gpu)
    gu, dn = ops.LowRankAdapters(gpu, a[:2], b[:2], scales=scales), ops.LowRankAdapters(gpu, a[2:], b[2:], scales=scales)
    xs, ys = torch.empty_like(hidden), torch.empty_like(hidden)
    plan = ops.AdapterGrouping(gpu, n).encode(ids)
    norm.encode(hidden, delta, out=xs, pre_weight=w1)
    mlp.encode_adapted(xs, gate, up, down, ys, gu, dn, ids, plan=plan)
    norm.encode(hidden, ys, post_weight=w2, gate=lw, gate_kind=ops.GATE_ROW)
    off = float((hidden.double() - want).norm() / want.norm())
    assert off < 0.02, off
    # on another stream, and without a plan
    side = torch.cuda.Stream()
    again = torch.empty_like(ys)
    torch.cuda.synchronize()
    mlp.encode_adapted(xs, gate, up, down, again, gu, dn, ids, stream=side)
    side.synchronize()
    off = float((again.double() - ys.double()).norm() / ys.double().norm())
    assert off < 0.01, off


def test_mlp_refuses_other_adapters(gpu):
    """adapters of other sizes, too few of them, results of another type: refused in front of the first launch, y as it was"""
    g = gen(5)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q = ops.Quantization(gpu)
    t, d, f, n, r = 12, 256, 384, 3, 8
    gate, up, down = (q.quantize_affine(rn(m, k) * k ** -0.5, 4) for m, k in ((f, d), (f, d), (d, f)))
    pool = lambda n_in, *ms: ops.LowRankAdapters(gpu, [rn(n, r, n_in).bfloat16() for _ in ms], [rn(n, m, r).bfloat16() for m in ms])  # noqa: E731
    x, y, ids = rn(t, d).bfloat16(), rn(t, d).bfloat16(), make_ids("mixed", t, n, 0.0, seed=1)
    before, mlp = y.clone(), ops.SharedExpertInt4(gpu)
    right = (pool(d, f, f), pool(f, d))
    for gu, dn in ((pool(d, f), right[1]), (pool(f, f, f), right[1]), (right[0], pool(d, d)), (right[0], pool(f, f)), (right[0], pool(f, d, d))):
        with pytest.raises(ops.MfError):
            mlp.encode_adapted(x, gate, up, down, y, gu, dn, ids)
    for bad_x, bad_y in ((x.half(), y), (x, y.half()), (x[:, :-64], y), (x, y[:-1])):
        with pytest.raises((ops.MfError, ValueError)):
            mlp.encode_adapted(bad_x, gate, up, down, bad_y, *right, ids)
    torch.cuda.synchronize()
    assert torch.equal(y, before)


def test_operators_refuse_numbers_in_place_of_vectors(gpu):
    g = gen(6)
    a, b = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 16, 8, device="cuda", dtype=torch.bfloat16)
    low, number = ops.LowRankAdapters(gpu, a, b), torch.zeros((), device="cuda", dtype=torch.int32)
    x, y = (torch.randn(1, m, generator=g, device="cuda").bfloat16() for m in (64, 16))
    with pytest.raises(ops.MfError):
        low.encode(x, number, y)
    with pytest.raises(ops.MfError):
        low.encode(x[0], number.reshape(1), y)
    with pytest.raises(ops.MfError):
        ops.AdapterGrouping(gpu, 2).encode(number)
    with pytest.raises(ops.MfError):
        ops.BlockNorm(gpu).encode(x, x.clone(), gate=torch.zeros((), device="cuda", dtype=torch.bfloat16), gate_kind=ops.GATE_ROW)
    with pytest.raises(ops.MfError):
        ops.BlockNorm(gpu).encode(x[0], x[0].clone())


def test_buffers_of_a_call_on_another_stream(gpu):
    """a plan and a workspace that the calls take themselves, for a stream that is not the current one: their memory is not handed
    out again while that stream may still use it"""
    g = gen(7)
    t, n, m, k, r = 300, 4096, 512, 4, 64
    a, b = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((k, r, n), (k, m, r)))
    low, grouping = ops.LowRankAdapters(gpu, a, b), ops.AdapterGrouping(gpu, k)
    x, ids = torch.randn(t, n, generator=g, device="cuda").bfloat16(), make_ids("mixed", t, k, 0.1, seed=2)
    want = torch.zeros(t, m, device="cuda")
    low.encode(x, ids, want, plan=grouping.encode(ids))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(8):
        y = torch.zeros(t, m, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        plan = grouping.encode(ids, stream=side)
        words = plan.words.numel()
        low.encode(x, ids, y, plan=plan, stream=side)
        del plan
        torch.full((words,), -1, dtype=torch.int32, device="cuda")
        torch.full((low.workspace_bytes(t),), 255, dtype=torch.uint8, device="cuda")
        side.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("t", [700, 4096, 9000, 70001])
@pytest.mark.parametrize("adapters", [1, 5, 700])
@pytest.mark.parametrize("order", ["one", "runs"])
def test_an_adapter_of_many_tiles(gpu, t, adapters, order):
    """one adapter's rows fill more tiles of the plan than a lane writes by itself: every row once, by the plan and without it"""
    Case(t, 64, (9,), adapters, 8, seed=t).check(gpu, make_ids(order, t, adapters, 0.05, seed=adapters), True)
