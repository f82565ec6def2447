"""mf_block_norm on the GPU against the formula in 64 bits.

Tolerances: the stream is rounded once to bf16 (half a step, 2^-8 of the value); before that every fp32 operation is off by 2^-24 of
its result.  The mean of d squares: each thread adds at most d / 64 of them (wider workgroups fewer), then a tree: the sum of positive
terms is off by at most (d / 64 + 32) 2^-24 of itself, its root by half of that, and eight further operations follow (division, eps,
root, reciprocal, two or three products, the weight's bias): E = (d / 64 + 48) 2^-24 of the largest term.  A sigmoid of fp32 steps: 8 more.
out is compared with the norm of the stream that the call itself left, so that the first rounding does not count twice."""
from __future__ import annotations

import pytest
import torch

from mference_amd import operators as ops

pytestmark = pytest.mark.gpu

KINDS = {"none": ops.GATE_NONE, "row": ops.GATE_ROW, "element": ops.GATE_ELEMENT, "channel": ops.GATE_CHANNEL}


def rows(v, pad, off):
    """v as rows of a wider buffer that starts off elements behind a border; (rows, buffer)"""
    t, d = v.shape
    flat = torch.full((off + t * (d + pad) + 8,), 3.0, dtype=v.dtype, device="cuda")
    r = flat[off:off + t * (d + pad)].view(t, d + pad)[:, pad // 2:pad // 2 + d]
    r.copy_(v)
    return r, flat


def check(gpu, t, d, gate="none", post=True, pre=True, delta32=False, rs=1.0, bs=1.0, wb=0.0, pad=0, off=0, seed=1, eps=1e-6, post_eps=1e-5, size=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    hidden, hbuf = rows((rn(t, d) * 2 * size).bfloat16(), pad, off)
    delta = rn(t, d) * size
    delta, _ = rows(delta if delta32 else delta.bfloat16(), pad, off)
    w1 = (1 - wb + 0.3 * rn(d)).bfloat16() if post else None
    w2 = (1 - wb + 0.3 * rn(d)).bfloat16() if pre else None
    out, obuf = rows(torch.zeros(t, d, dtype=torch.bfloat16, device="cuda"), pad, off)
    gt = {"none": None, "row": rn(t, 1).bfloat16(), "element": rn(t, d).bfloat16() * 2, "channel": rn(d).bfloat16()}[gate]
    if gate == "element":
        gt, _ = rows(gt, pad, off)
    h, b = hidden.double(), delta.double()
    if post:
        b = b / (b.square().mean(1, keepdim=True) + post_eps).sqrt() * (w1.double() + wb)
    if gate in ("row", "element"):
        b = b * torch.sigmoid(gt.double())
    elif gate == "channel":
        b = b * gt.double()
    want = rs * h + bs * b
    outer = [v.clone() for v in (hbuf, obuf)]
    ops.BlockNorm(gpu).encode(hidden, delta, out=out if pre else None, pre_weight=w2, post_weight=w1, gate=gt, gate_kind=KINDS[gate], eps=eps, post_eps=post_eps,
                              residual_scale=rs, branch_scale=bs, weight_bias=wb)
    e = (d / 64 + 56) * 2.0 ** -24
    far = (hidden.double() - want).abs() - 2.0 ** -8 * want.abs() - e * (abs(rs) * h.abs() + abs(bs) * b.abs()) - 2.0 ** -134
    assert far.max() <= 0, far.max()
    if pre:
        z = hidden.double()
        want = z / (z.square().mean(1, keepdim=True) + eps).sqrt() * (w2.double() + wb)
        far = (out.double() - want).abs() - (2.0 ** -8 + e) * want.abs() - 2.0 ** -134
        # the weight plus its bias is rounded too: 2^-24 of the larger of the two
        far -= 2.0 ** -23 * (z / (z.square().mean(1, keepdim=True) + eps).sqrt()).abs() * abs(wb)
        assert far.max() <= 0, far.max()
    else:
        assert torch.equal(obuf, outer[1])
    for flat, was, r in ((hbuf, outer[0], hidden), (obuf, outer[1], out)):
        r.copy_(was.as_strided(r.shape, r.stride(), r.storage_offset()))
        assert torch.equal(flat, was), "written outside of the rows"


@pytest.mark.parametrize("gate", list(KINDS))
@pytest.mark.parametrize("post, pre, delta32", [(True, True, False), (False, True, True), (True, False, True), (False, False, False)])
@pytest.mark.parametrize("t, d", [(1, 2048), (3, 64), (8, 2816), (70, 520), (5, 1), (2, 7), (33, 1000), (300, 256)])
def test_block_norm(gpu, t, d, gate, post, pre, delta32):
    check(gpu, t, d, gate, post, pre, delta32, seed=t + d)


@pytest.mark.parametrize("t, d", [(1, 5120), (9, 4096), (777, 4096), (2, 8192), (3, 8200), (2, 16384), (2, 16392), (1, 40000), (3, 12345), (2100, 128)])
@pytest.mark.parametrize("gate, delta32", [("none", False), ("element", True)])
def test_block_norm_of_long_rows(gpu, t, d, gate, delta32):
    check(gpu, t, d, gate, True, True, delta32, rs=0.875, bs=0.22, wb=1.0, seed=d)


@pytest.mark.parametrize("pad, off", [(0, 1), (1, 0), (8, 0), (24, 8), (6, 3), (0, 4)])
@pytest.mark.parametrize("delta32", [False, True])
@pytest.mark.parametrize("t, d", [(1, 512), (6, 1000), (40, 2816), (3, 9000)])
def test_block_norm_between_other_columns(gpu, t, d, pad, off, delta32):
    check(gpu, t, d, "element", True, True, delta32, pad=pad, off=off, seed=d + pad)


@pytest.mark.parametrize("rs, bs, wb", [(1.0, 0.5, 0.0), (0.5, 0.5, 1.0), (0.0, 1.0, 0.0), (-1.0, 2.0, 0.0), (1.0, 0.0, 1.0)])
def test_block_norm_scales(gpu, rs, bs, wb):
    check(gpu, 11, 768, "row", True, True, False, rs, bs, wb, seed=5)
    check(gpu, 11, 768, "channel", False, True, True, rs, bs, wb, seed=6)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 2.0 ** 40])
def test_block_norm_of_any_magnitude(gpu, size):
    check(gpu, 5, 2816, "none", True, True, False, seed=7, size=size)
    check(gpu, 5, 1001, "row", True, True, True, seed=8, size=size)


def test_norm_of_the_stream_alone(gpu):
    """no block output: the stream is only read"""
    for t, d in ((1, 2048), (65, 1000)):
        hidden = torch.randn(t, d, device="cuda").bfloat16()
        was, w, out = hidden.clone(), (1 + 0.1 * torch.randn(d, device="cuda")).bfloat16(), torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
        ops.BlockNorm(gpu).encode(hidden, out=out, pre_weight=w)
        z = hidden.double()
        want = z / (z.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        assert torch.equal(hidden, was)
        assert ((out.double() - want).abs() <= (2.0 ** -8 + (d / 64 + 56) * 2.0 ** -24) * want.abs()).all()


def test_close_to_the_residual_norm(gpu):
    """without norm behind, gate and scales it is mf_residual_rmsnorm: the same stream bit for bit, the same norm within the order of a sum"""
    for t, d in ((1, 2048), (7, 2816), (40, 1000)):
        h1, dl, w = (torch.randn(t, d, device="cuda").bfloat16() for _ in range(3))
        w = w[0].contiguous()
        h2, o1, o2 = h1.clone(), torch.empty_like(h1), torch.empty_like(h1)
        ops.RMSNorm(gpu).encode_bf16w(h1, w, o1, d, 1e-6, t=t, delta=dl)
        ops.BlockNorm(gpu).encode(h2, dl, out=o2, pre_weight=w)
        assert torch.equal(h1, h2)
        assert ((o1.double() - o2.double()).abs() <= (2.0 ** -7 + 2.0 ** -15) * o1.double().abs()).all()


def test_rows_of_zeros_nan_and_infinity(gpu):
    """a row of zeros keeps eps under the root; NaN and infinities stay with their row"""
    t, d = 9, 512
    hidden, delta = torch.randn(t, d, device="cuda").bfloat16(), torch.randn(t, d, device="cuda").bfloat16()
    w = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    ref, ref_out = hidden.clone(), torch.empty_like(hidden)
    ops.BlockNorm(gpu).encode(ref, delta, out=ref_out, pre_weight=w, post_weight=w)
    h2, out = hidden.clone(), torch.empty_like(hidden)
    d2 = delta.clone()
    h2[1], d2[1] = 0, 0
    d2[3, 7], h2[5, 100], d2[7, 3] = float("nan"), float("inf"), -float("inf")
    ops.BlockNorm(gpu).encode(h2, d2, out=out, pre_weight=w, post_weight=w)
    for i in (0, 2, 4, 6, 8):
        assert torch.equal(h2[i], ref[i]) and torch.equal(out[i], ref_out[i])
    assert not bool(h2[1].any()) and not bool(out[1].any())
    assert bool(torch.isnan(h2[3]).all()) and bool(torch.isnan(out[3]).all())
    assert bool(h2[5, 100] == float("inf")) and bool(torch.isnan(out[5, 100]))
    assert bool(torch.isnan(out[7]).any())


def test_gates_at_their_ends(gpu):
    """logits of infinity open and close the gate exactly; a NaN logit stays with what it gates"""
    t, d = 4, 64
    delta = torch.ones(t, d, dtype=torch.bfloat16, device="cuda")
    logit = torch.tensor([[float("inf")], [-float("inf")], [0.0], [float("nan")]], device="cuda").bfloat16()
    for kind, g in ((ops.GATE_ROW, logit), (ops.GATE_ROW, logit[:, 0]), (ops.GATE_ELEMENT, logit.expand(t, d).contiguous())):
        hidden = torch.zeros(t, d, dtype=torch.bfloat16, device="cuda")
        ops.BlockNorm(gpu).encode(hidden, delta, gate=g, gate_kind=kind)
        assert bool((hidden[0] == 1).all()) and bool((hidden[1] == 0).all()) and bool((hidden[2] == 0.5).all()) and bool(torch.isnan(hidden[3]).all())


def test_rows_past_32_bits(gpu):
    t, d = (1 << 18) + 1, 16400
    hidden = torch.zeros((t, d), dtype=torch.bfloat16, device="cuda")
    hidden[-1] = 2
    out = torch.zeros_like(hidden)
    w = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    ops.BlockNorm(gpu).encode(hidden, out=out, pre_weight=w)
    assert bool((out[-1] == 1).all()) and not bool(out[-2].any()) and not bool(out[0].any())


def test_block_norm_refuses(gpu):
    n = ops.BlockNorm(gpu)
    h, dl, w = (torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    w = w[0]
    for kw in (dict(delta=dl[:3]), dict(delta=dl[:, :32]), dict(delta=dl, gate=w[:3], gate_kind=ops.GATE_ROW), dict(delta=dl, gate=w[:1].expand(4), gate_kind=ops.GATE_ROW),
               dict(delta=dl, gate=w, gate_kind=ops.GATE_ELEMENT), dict(delta=dl, gate=dl, gate_kind=ops.GATE_CHANNEL), dict(delta=dl, gate=w), dict(delta=dl, out=h, pre_weight=w),
               dict(delta=dl, out=dl, pre_weight=w), dict(delta=h), dict(delta=dl, pre_weight=w), dict(out=dl), dict(post_weight=w), dict(delta=dl, post_weight=w[:32]),
               dict(delta=dl[:1].expand(4, 64)), dict()):
        with pytest.raises(ops.MfError):
            n.encode(h, **kw)
    for kw in (dict(delta=dl.half()), dict(delta=dl, post_weight=w.float()), dict(delta=dl.cpu())):
        with pytest.raises(ValueError):
            n.encode(h, **kw)
    n.encode(h[:0], dl[:0])
