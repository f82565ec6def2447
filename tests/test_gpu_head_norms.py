"""mf_head_norms on the GPU against the definition in 64 bits."""
import pytest
import torch

from dense16_cases import assert_near, generator, heads64, randn
from mference_amd import operators as ops

pytestmark = pytest.mark.gpu

CASES = [  # t, q heads, k heads, head_dim, pairs, axes, interleaved, norm
    (1, 16, 2, 256, 32, 1, False, True), (1, 1, 1, 128, 64, 1, False, True), (1, 1, 0, 64, 32, 1, False, True), (2, 4, 2, 72, 36, 2, False, True), (3, 5, 1, 80, 20, 3, True, True),
    (7, 32, 8, 128, 64, 3, False, True), (9, 3, 3, 1, 0, 1, False, True), (5, 2, 1, 3, 1, 1, False, True), (5, 2, 2, 6, 3, 2, True, False), (17, 6, 2, 96, 48, 1, True, True),
    (64, 8, 8, 64, 32, 2, False, False), (33, 12, 4, 192, 96, 8, False, True), (130, 40, 8, 128, 64, 1, False, True), (100, 7, 1, 1024, 512, 1, False, True),
    (31, 2, 2, 1000, 77, 3, True, True), (12, 3, 1, 130, 65, 1, False, True), (257, 16, 16, 128, 64, 1, True, True), (40, 64, 4, 64, 8, 1, False, True), (21, 9, 9, 48, 16, 2, False, True),
    (11, 4, 2, 256, 128, 3, False, True), (1025, 4, 1, 128, 64, 1, False, True), (6, 128, 1, 576, 32, 1, True, True), (19, 3, 2, 512, 256, 1, False, False), (300, 2, 1, 32, 16, 1, False, True),
]


def frequencies(pairs, base=1e6):
    return torch.tensor([base ** (-p / pairs) for p in range(pairs)], dtype=torch.float32, device="cuda") if pairs else None


def inputs(t, q, k, dim, pairs, axes, norm, far=0, seed=0):
    g = generator(seed + 31 * t + q + dim)
    whole = (randn(g, t, q + 2 * k + 1, dim) * 2).bfloat16()
    weights = [randn(g, dim).bfloat16() if norm else None for _ in range(2)]
    positions = torch.randint(0, 4000, (axes, t), generator=g, device="cuda", dtype=torch.int32) + far if pairs else None
    table = torch.randint(0, axes, (pairs,), generator=g, device="cuda", dtype=torch.uint8) if axes > 1 and pairs else None
    return whole, weights, positions, table


@pytest.mark.parametrize("t, q, k, dim, pairs, axes, interleaved, norm", CASES)
@pytest.mark.parametrize("far", [0, 1000000])
def test_in_place_in_a_wider_buffer(gpu, t, q, k, dim, pairs, axes, interleaved, norm, far):
    whole, (wq, wk), positions, table = inputs(t, q, k, dim, pairs, axes, norm, far)
    freq, before = frequencies(pairs), whole.clone()
    op = ops.HeadNorms(gpu, dim, freq, table, interleaved, wq, wk, eps=1e-5, weight_bias=1.0 if far else 0.0, rotation_scale=1.0 if far else 0.75)
    op.encode(whole[:, :q], whole[:, q:q + k] if k else None, positions)
    for at, w in ((slice(0, q), wq), (slice(q, q + k), wk)):
        want, off = heads64(before[:, at], w, positions, freq, table, interleaved, 1e-5, 1.0 if far else 0.0, 1.0 if far else 0.75)
        assert_near(whole[:, at], want, off)
    assert torch.equal(whole[:, q + k:], before[:, q + k:])  # the values' heads


@pytest.mark.parametrize("t, q, k, dim, pairs, axes, interleaved, norm", CASES)
def test_heads_first_and_elsewhere(gpu, t, q, k, dim, pairs, axes, interleaved, norm):
    """results in buffers of their own, heads in front of rows, rows of odd places"""
    whole, (wq, wk), positions, table = inputs(t, q, k, dim, pairs, axes, norm, seed=9)
    freq, before = frequencies(pairs), whole.clone()
    q_out = torch.full((q, t + 2, dim + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    k_flat = torch.full((5 + t * (k * dim + 1) + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
    qo = q_out.transpose(0, 1)[1:t + 1, :, 1:dim + 1]
    ko = k_flat[5:5 + t * (k * dim + 1)].view(t, k * dim + 1)[:, :k * dim].unflatten(1, (k, dim)) if k else None
    kept_q, kept_k = q_out.clone(), k_flat.clone()
    op = ops.HeadNorms(gpu, dim, freq, table, interleaved, wq, wk)
    op.encode(whole[:, :q], whole[:, q:q + k] if k else None, positions, q_out=qo, k_out=ko)
    for got, at, w in ((qo, slice(0, q), wq), (ko, slice(q, q + k), wk)):
        if got is None:
            continue
        want, off = heads64(before[:, at], w, positions, freq, table, interleaved, 1e-6, 0.0, 1.0)
        assert_near(got, want, off)
    kept_q.transpose(0, 1)[1:t + 1, :, 1:dim + 1] = qo
    assert torch.equal(q_out, kept_q) and torch.equal(whole, before)
    if k:
        kept_k[5:5 + t * (k * dim + 1)].view(t, k * dim + 1)[:, :k * dim] = ko.flatten(1)
        assert torch.equal(k_flat, kept_k)


def test_only_the_norm_and_only_the_rotation(gpu):
    whole, (wq, wk), positions, _ = inputs(13, 6, 2, 128, 64, 1, True)
    before = whole.clone()
    ops.HeadNorms(gpu, 128, q_weight=wq).encode(whole[:, :6], whole[:, 6:8])  # keys without a weight stay as they are
    want, off = heads64(before[:, :6], wq, None, None, None, False, 1e-6, 0.0, 1.0)
    assert_near(whole[:, :6], want, off)
    assert torch.equal(whole[:, 6:], before[:, 6:])
    now = whole.clone()
    freq = frequencies(64)
    ops.HeadNorms(gpu, 128, freq).encode(whole[:, 6:8], positions=positions[0])
    want, off = heads64(now[:, 6:8], None, positions, freq, None, False, 0, 0, 1)
    assert_near(whole[:, 6:8], want, off)
    assert torch.equal(whole[:, :6], now[:, :6])


@pytest.mark.parametrize("dim, interleaved", [(128, False), (128, True), (72, False), (50, True)])
def test_axes_past_the_last_and_positions_of_any_sign(gpu, dim, interleaved):
    pairs = dim // 2
    whole, (wq, _), _, _ = inputs(9, 4, 1, dim, pairs, 2, True)
    positions = torch.tensor([[0, 1, -1, 2147483647, -2147483648, 5, 123456789, -77, 1 << 20], [9, 8, 7, 6, 5, 4, 3, 2, 1]], dtype=torch.int32, device="cuda")
    table = (torch.arange(pairs, device="cuda") % 4).to(torch.uint8)  # 2 and 3 are no axes: those pairs are not turned
    freq, before = frequencies(pairs, 1e4), whole.clone()
    ops.HeadNorms(gpu, dim, freq, table, interleaved, wq).encode(whole[:, :4], positions=positions)
    want, off = heads64(before[:, :4], wq, positions, freq, table, interleaved, 1e-6, 0.0, 1.0)
    assert_near(whole[:, :4], want, off)


def test_zero_rows_and_infinities_stay_with_their_head(gpu):
    whole, (wq, wk), positions, _ = inputs(6, 4, 2, 128, 64, 1, True)
    whole[2, 1] = 0.0
    whole[3, 2, 7] = float("inf")
    whole[4, 5, 100] = float("nan")
    freq, before = frequencies(64), whole.clone()
    ops.HeadNorms(gpu, 128, freq, q_weight=wq, k_weight=wk).encode(whole[:, :4], whole[:, 4:6], positions)
    assert not whole[2, 1].any() and not torch.isfinite(whole[4, 5]).any()
    fine = torch.ones(6, 4, dtype=torch.bool, device="cuda")
    fine[3, 2] = False
    want, off = heads64(before[:, :4], wq, positions, freq, None, False, 1e-6, 0.0, 1.0)
    assert_near(whole[:, :4][fine], want[fine], off[fine])
    # beside an infinity the others of its head are 0, its pair is not a number
    rest = [e for e in range(128) if e not in (7, 71)]
    assert not whole[3, 2, rest].any() and not torch.isfinite(whole[3, 2, [7, 71]]).any()


@pytest.mark.parametrize("device", ["cpu"])
def test_sections(device):
    assert ops.HeadNorms.axes_of_sections((2, 3), device=device).tolist() == [0, 0, 1, 1, 1]
    assert ops.HeadNorms.axes_of_sections((3, 2, 1), turns=True, device=device).tolist() == [0, 1, 2, 0, 1, 0]


@pytest.mark.parametrize("t", [1, 300])
def test_captured_graph_and_another_stream(gpu, t):
    whole, (wq, wk), positions, table = inputs(t, 16, 4, 128, 64, 3, True)
    op = ops.HeadNorms(gpu, 128, frequencies(64), table, False, wq, wk)
    out = torch.empty(t, 20, 128, dtype=torch.bfloat16, device="cuda")
    call = lambda **kw: op.encode(whole[:, :16], whole[:, 16:20], positions, q_out=out[:, :16], k_out=out[:, 16:], **kw)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    side = torch.cuda.Stream()
    for k in range(3):
        positions.add_(17 * k)
        whole.copy_((randn(generator(k), *whole.shape)).bfloat16())
        graph.replay()
        got = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        call(stream=side)
        side.synchronize()
        assert torch.equal(got, out)


def test_rows_past_4_gib(gpu):
    """a cache of heads in front of rows, its last heads past 2^32 bytes"""
    t, k, dim = 5, 3, 64
    cache = torch.zeros(k, (1 << 31) // 2 // dim // 1, dim, dtype=torch.bfloat16, device="cuda")  # a head's rows: 2 GiB
    whole, (wq, wk), positions, _ = inputs(t, 2, k, dim, 32, 1, True)
    out = cache.transpose(0, 1)[-t:]
    freq, before = frequencies(32), whole.clone()
    ops.HeadNorms(gpu, dim, freq, q_weight=wq, k_weight=wk).encode(whole[:, :2], whole[:, 2:2 + k], positions, k_out=out)
    want, off = heads64(before[:, 2:2 + k], wk, positions, freq, None, False, 1e-6, 0.0, 1.0)
    assert_near(out, want, off)
    assert not cache[:, :-t].any()
