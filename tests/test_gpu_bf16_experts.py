"""mf_bf16_experts on the GPU against the definition in 64 bits, and a layer of 16-bit operators from end to end."""
import pytest
import torch

from dense16_cases import ACTS, Placed, assert_near, experts64, generator, heads64, ints, project64, randn
from mference_amd import operators as ops

pytestmark = pytest.mark.gpu

CASES = [  # t, d, f, experts, top_k, shared_f
    (1, 64, 64, 8, 2, 0), (1, 8, 8, 1, 1, 8), (1, 2048, 512, 32, 8, 512), (2, 264, 72, 5, 3, 40), (3, 136, 200, 512, 8, 0), (4, 512, 256, 16, 4, 256), (7, 104, 1032, 9, 6, 24),
    (8, 1024, 128, 64, 8, 128), (15, 256, 64, 4, 4, 64), (16, 320, 96, 20, 8, 96), (17, 320, 96, 20, 8, 96), (24, 72, 40, 3, 2, 16), (33, 256, 320, 12, 2, 0), (40, 40, 24, 2, 1, 8),
    (61, 512, 128, 64, 8, 0), (64, 256, 64, 256, 8, 64), (64, 128, 136, 1, 1, 0), (64, 64, 64, 8, 8, 2048), (5, 5120, 64, 3, 2, 0), (9, 64, 2048, 6, 3, 0),
]


class Layer:
    def __init__(self, t, d, f, experts, top_k, shared_f, bias=True, gate=True, residual=True, exact=False, seed=0, pad=0, off=0):
        g = generator(seed + 13 * t + d + f)
        v = (lambda *s, scale=1.0: ints(g, 2, *s).bfloat16()) if exact else (lambda *s, scale=1.0: (randn(g, *s) * scale).bfloat16())
        self.x = Placed(v(t, d), pad, off)
        self.kw = dict(gate_up=v(experts, 2 * f, d, scale=d ** -0.5), down=v(experts, d, f, scale=f ** -0.5))
        if bias:
            self.kw.update(gate_up_bias=v(experts, 2 * f), down_bias=v(experts, d))
        if shared_f:
            self.kw.update(shared_gate_up=v(2 * shared_f, d, scale=d ** -0.5), shared_down=v(d, shared_f, scale=shared_f ** -0.5))
            if gate:
                self.kw.update(shared_gate=v(d, scale=d ** -0.5))
        self.idx = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:top_k] for _ in range(t)]).int()
        self.w = ints(g, 2, t, top_k) if exact else torch.rand((t, top_k), generator=g, device="cuda")
        self.residual = Placed(v(t, d), pad, off) if residual else None
        self.y = Placed(torch.zeros((t, d), dtype=torch.bfloat16, device="cuda"), pad, off, 7.0)
        self.top_k = top_k

    def op(self, ctx, act="silu"):
        kw = dict(self.kw)
        return ops.Bf16Experts(ctx, kw.pop("gate_up"), kw.pop("down"), self.top_k, activation=ACTS.index(act), **kw)

    def run(self, ctx, act="silu", y=None, residual="own", **more):
        r = self.residual and self.residual.rows if residual == "own" else residual
        self.op(ctx, act).encode(self.x.rows, self.idx, self.w, self.y.rows if y is None else y, residual=r, **more)

    def want(self, act="silu"):
        return experts64(self.x.rows, self.idx, self.w, residual=self.residual and self.residual.rows, act=act, **self.kw)


@pytest.mark.parametrize("place, t, d, f, experts, top_k, shared_f", [(i, *c) for i, c in enumerate(CASES)])
def test_layer(gpu, place, t, d, f, experts, top_k, shared_f):
    for turn in range(2):
        k = place + 3 * turn
        pad, off = ((0, 0), (3, 1), (8, 8))[k % 3]
        layer = Layer(t, d, f, experts, min(top_k, experts), shared_f, bias=k % 2 == 0, gate=k % 4 != 1, residual=k % 3 != 1, seed=turn, pad=pad, off=off)
        act = ACTS[(k + turn) % 4]
        layer.run(gpu, act)
        want, far = layer.want(act)
        assert_near(layer.y.rows, want, far, (act, pad, off))
        assert layer.y.only_rows_changed()
        first = layer.y.rows.clone()
        layer.run(gpu, act)
        assert torch.equal(first, layer.y.rows)


@pytest.mark.parametrize("t, d, f, experts, top_k, shared_f", [(1, 64, 40, 4, 2, 0), (5, 136, 64, 7, 3, 16), (20, 64, 32, 8, 4, 0), (64, 48, 24, 16, 8, 8)])
def test_whole_numbers(gpu, t, d, f, experts, top_k, shared_f):
    """sums of whole numbers are exact, activations of them in two bf16 terms too: one rounding at the end"""
    layer = Layer(t, d, f, experts, top_k, shared_f, exact=True, gate=False)
    for name in ("gate_up", "shared_gate_up"):  # a few ones a row: activations below 2^16
        if name in layer.kw:
            v = layer.kw[name]
            v.mul_((torch.rand(v.shape, generator=generator(3), device="cuda") < 0.1).bfloat16())
    layer.run(gpu, "none")
    want, _ = layer.want("none")
    assert want.abs().max() < 2 ** 24
    assert torch.equal(layer.y.rows, want.bfloat16())


@pytest.mark.parametrize("t", [1, 6, 40])
def test_routes_that_name_no_expert_and_one_twice(gpu, t):
    layer = Layer(t, 128, 64, 9, 4, 32)
    layer.idx[:, 1] = layer.idx[:, 0]
    layer.idx[::2, 2] = 9
    layer.idx[1::3, 3] = -1
    layer.w[::2, 2] = float("nan")  # the weight of a route without an expert is not used
    layer.run(gpu)
    want, far = layer.want()
    assert_near(layer.y.rows, want, far)
    layer.idx.fill_(-1)  # no live expert at all
    layer.run(gpu)
    want, far = layer.want()
    assert_near(layer.y.rows, want, far)


@pytest.mark.parametrize("t", [1, 20, 64])
def test_all_tokens_on_one_expert(gpu, t):
    layer = Layer(t, 256, 72, 300, 8, 0)
    layer.idx.fill_(299)
    layer.run(gpu)
    want, far = layer.want()
    assert_near(layer.y.rows, want, far)


def test_infinities_stay_with_their_token_and_idle_experts_are_not_read(gpu):
    layer = Layer(12, 256, 64, 16, 2, 0)
    layer.idx.copy_(torch.randint(0, 8, layer.idx.shape, generator=generator(1), device="cuda"))
    for v in layer.kw.values():
        v[8:] = float("nan")
    layer.x.rows[5, 3] = float("inf")
    layer.run(gpu)
    rest = [i for i in range(12) if i != 5]
    want, far = layer.want()
    assert_near(layer.y.rows[rest], want[rest], far[rest])
    assert not torch.isfinite(layer.y.rows[5]).all()


def test_in_place_and_captured(gpu):
    layer = Layer(9, 512, 128, 16, 4, 64, pad=8)
    want, far = layer.want()
    op, rows = layer.op(gpu), layer.residual.rows
    kept = rows.clone()
    ws = torch.full((op.workspace_bytes(64),), 255, dtype=torch.uint8, device="cuda")
    op.encode(layer.x.rows, layer.idx, layer.w, rows, residual=rows, workspace=ws)
    assert_near(rows, want, far)
    assert layer.residual.only_rows_changed()
    rows.copy_(kept)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.encode(layer.x.rows, layer.idx, layer.w, layer.y.rows, residual=rows, workspace=ws)
    for k in range(4):
        layer.idx.copy_(torch.randint(-1, 16, layer.idx.shape, generator=generator(k), device="cuda"))
        ws.fill_(255)
        graph.replay()
        got = layer.y.rows.clone()
        layer.y.rows.zero_()
        op.encode(layer.x.rows, layer.idx, layer.w, layer.y.rows, residual=rows)
        torch.cuda.synchronize()
        assert torch.equal(got, layer.y.rows)
        want, far = layer.want()
        assert_near(got, want, far)


def test_another_stream(gpu):
    layer = Layer(6, 512, 128, 16, 4, 64)
    want, far = layer.want()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    layer.run(gpu, stream=side)
    side.synchronize()
    assert_near(layer.y.rows, want, far)


@pytest.mark.parametrize("t", [1, 6, 40])
def test_a_layer_from_end_to_end(gpu, t):
    """projection of queries, keys and values with its bias, head norms with positions of three axes in place, projection back into the stream,
    the norm between the blocks, the router, the experts into the stream: every step against its definition, from what the step before left"""
    d, q, k, dim, f, experts, top_k = 256, 6, 2, 64, 96, 16, 4
    g = generator(t)
    v = lambda *s, scale=1.0: (randn(g, *s) * scale).bfloat16()
    x, stream = v(t, d), v(t, d)
    qkv = torch.empty(t, (q + 2 * k) * dim, dtype=torch.bfloat16, device="cuda")
    w, b = v((q + 2 * k) * dim, d, scale=d ** -0.5), v((q + 2 * k) * dim, scale=0.2)
    ops.Projection(gpu, w, bias=b).encode(x, qkv)
    assert_near(qkv, *project64(x, w, b, None, "none", False))
    heads, before = qkv.view(t, q + 2 * k, dim), qkv.view(t, q + 2 * k, dim).clone()
    freq = torch.tensor([1e4 ** (-p / 32) for p in range(32)], dtype=torch.float32, device="cuda")
    table = ops.HeadNorms.axes_of_sections((12, 10, 10), turns=True)
    positions = torch.randint(0, 5000, (3, t), generator=g, device="cuda", dtype=torch.int32)
    wq, wk = v(dim), v(dim)
    ops.HeadNorms(gpu, dim, freq, table, q_weight=wq, k_weight=wk).encode(heads[:, :q], heads[:, q:q + k], positions)
    assert_near(heads[:, :q], *heads64(before[:, :q], wq, positions, freq, table, False, 1e-6, 0.0, 1.0))
    assert_near(heads[:, q:q + k], *heads64(before[:, q:q + k], wk, positions, freq, table, False, 1e-6, 0.0, 1.0))
    wo = v(d, q * dim, scale=(q * dim) ** -0.5)
    kept = stream.clone()
    ops.Projection(gpu, wo).encode(qkv[:, :q * dim], stream, residual=stream)  # (attention would stand in front)
    assert_near(stream, *project64(qkv[:, :q * dim], wo, None, kept, "none", False))
    normed, wn = torch.empty_like(stream), v(d)
    ops.BlockNorm(gpu).encode(stream, out=normed, pre_weight=wn)
    idx = torch.empty(t, top_k, dtype=torch.int32, device="cuda")
    weights, logits = torch.empty(t, top_k, device="cuda"), torch.empty(t, experts, device="cuda")
    wr = v(experts, d, scale=d ** -0.5)
    ops.FamilyRouters(gpu).encode_router_top_k(wr, normed, torch.zeros(experts, device="cuda"), idx, weights, experts, d, 1.0, logits, top_k=top_k, t=t)
    kw = dict(gate_up=v(experts, 2 * f, d, scale=d ** -0.5), down=v(experts, d, f, scale=f ** -0.5), shared_gate_up=v(2 * f, d, scale=d ** -0.5),
              shared_down=v(d, f, scale=f ** -0.5), shared_gate=v(d, scale=d ** -0.5))
    kept = stream.clone()
    ops.Bf16Experts(gpu, kw["gate_up"], kw["down"], top_k, **{n: kw[n] for n in kw if n.startswith("shared")}).encode(normed, idx, weights, stream, residual=stream)
    assert_near(stream, *experts64(normed, idx, weights, residual=kept, **kw))
