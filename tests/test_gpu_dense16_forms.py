"""The operators of layers kept in 16 bits in each form that their sizes choose on a card of 256 units: shapes of tiles, sums in parts, rows and groups of
workgroups; and calls that run at once."""
import pytest
import torch

from dense16_cases import ACTS, Placed, assert_near, generator, heads64, project64, randn
from mference_amd import operators as ops
from test_gpu_bf16_experts import Layer
from test_gpu_head_norms import frequencies
from test_gpu_projection import make

pytestmark = pytest.mark.gpu

PROJECT = [  # t, n, m, gated: what they come to
    (3, 264, 4100, 0), (2, 520, 4100, 1), (4, 263, 4100, 0), (6, 199, 4100, 1),  # few rows, nine of W a workgroup, two waves or (gated) four
    (12, 264, 4100, 0), (13, 263, 4100, 1), (16, 263, 4100, 0), (9, 200, 9001, 0), (7, 136, 8195, 1), (8, 264, 4097, 0),  # up to 16 rows, of W 9 to 12 a workgroup
    (20, 4104, 33, 0), (20, 8199, 33, 1), (20, 5128, 33, 1), (300, 4104, 33, 0), (40, 4103, 260, 1), (513, 8200, 100, 1), (700, 8200, 130, 0),  # 32 x 32, 2 to 15 parts
    (40, 520, 4100, 0), (20, 520, 4100, 1), (20, 5128, 1100, 1), (20, 8200, 1100, 0),  # 32 x 64, 1 to 8 parts
    (100, 328, 4100, 0), (40, 327, 4100, 1), (40, 4103, 4100, 0), (700, 5128, 33, 1), (40, 8200, 1100, 1), (513, 8199, 33, 0),  # 64 x 64, 1 to 15 parts
    (130, 520, 7000, 0), (100, 520, 4100, 1), (40, 8200, 4100, 0), (3000, 8200, 33, 1),  # 64 x 128, 1 and 4 parts
    (777, 1032, 7000, 0), (513, 1032, 5000, 1), (1500, 327, 5000, 0), (4090, 327, 1000, 1),  # 128 x 128, two workgroups a unit
    (1500, 328, 4100, 0), (513, 328, 6100, 1), (100, 8200, 4100, 0), (6000, 8200, 33, 1),  # 128 x 128, one
    (777, 1032, 5000, 0), (400, 1032, 5000, 1), (400, 8200, 5000, 0), (130, 8200, 3000, 1),  # 128 x 192, 1 to 4 parts
    (2050, 200, 7000, 0), (1500, 200, 5000, 1),  # 256 x 128
    (3000, 1032, 7000, 0), (2050, 1032, 5000, 1),  # 256 x 192
    (6000, 328, 5000, 0), (2050, 328, 7000, 1),  # 256 x 256
]


@pytest.mark.parametrize("t, n, m, gated", PROJECT)
def test_projection_shapes(gpu, t, n, m, gated):
    gated = bool(gated)
    x, w, b, r, y = make(t, n, m, gated=gated, pad=8 if n % 8 == 0 else 3, off=8 if n % 8 == 0 else 1, dtype=torch.float32 if m == 5000 else torch.bfloat16)
    op = ops.Projection(gpu, w.rows, bias=b, activation=ops.ACT_GELU_TANH, gated=gated)
    ws = torch.full((max(op.workspace_bytes(t), 16),), 255, dtype=torch.uint8, device="cuda")
    op.encode(x.rows, y.rows, residual=r.rows, workspace=ws)
    want, far = project64(x.rows, w.rows, b, r.rows, "gelu_tanh", gated)
    assert_near(y.rows, want, far)
    assert y.only_rows_changed()
    first = y.rows.clone()
    y.rows.zero_()
    op.encode(x.rows, y.rows, residual=r.rows, workspace=ws)
    assert torch.equal(first, y.rows)


EXPERTS = [  # t, d, f, experts, top_k, shared_f
    (3, 5120, 64, 4, 3, 0), (8, 4104, 40, 12, 8, 264), (1, 16, 2056, 4, 2, 0), (8, 2816, 136, 40, 8, 136),  # up to eight tokens: rows of one and of two rounds
    (9, 5128, 72, 6, 2, 24), (30, 5120, 64, 8, 3, 0),  # one group
    (9, 2816, 328, 9, 2, 1032), (64, 4104, 64, 5, 4, 0), (20, 2568, 8, 30, 8, 64),  # two, the second with nothing of f of 8
    (12, 520, 264, 16, 4, 64), (61, 1024, 520, 40, 8, 0), (64, 256, 72, 512, 8, 2056), (10, 64, 136, 3, 1, 8),  # four, of them one or two without a part of the sum
]


@pytest.mark.parametrize("t, d, f, experts, top_k, shared_f", EXPERTS)
def test_experts_rows_and_groups(gpu, t, d, f, experts, top_k, shared_f):
    layer = Layer(t, d, f, experts, top_k, shared_f, pad=8, off=8)
    layer.run(gpu)
    want, far = layer.want()
    assert_near(layer.y.rows, want, far)
    assert layer.y.only_rows_changed()
    first = layer.y.rows.clone()
    for _ in range(3):
        layer.run(gpu)
        assert torch.equal(first, layer.y.rows)


@pytest.mark.parametrize("t, most", [(33, 1), (64, 2), (64, 3), (17, 2)])
def test_experts_with_many_routes(gpu, t, most):
    """experts of whole and broken runs of 16 routes, beside ones that nobody names"""
    layer = Layer(t, 200, 72, 24, 8, 40)
    layer.idx.copy_(torch.arange(t * 8, device="cuda").view(t, 8).int() % most * 11)  # (an expert several times a token)
    layer.run(gpu)
    want, far = layer.want()
    assert_near(layer.y.rows, want, far)


def test_calls_at_once(gpu):
    """two streams, each with a workspace of its own, over the same weights: the results of each alone"""
    p = [make(t, 4104, 260, seed=t) for t in (40, 300)]
    op = ops.Projection(gpu, p[0][1].rows, bias=p[0][2], activation=ops.ACT_SILU)
    layers = [Layer(t, 512, 264, 16, 4, 64) for t in (6, 40)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    expert = layers[0].op(gpu)

    def both(at, stream):
        x, _, _, r, y = p[at]
        layer = layers[at]
        ws = torch.empty(max(op.workspace_bytes(x.rows.shape[0]), 16), dtype=torch.uint8, device="cuda")
        ews = torch.empty(expert.workspace_bytes(layer.x.rows.shape[0]), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

        def run():
            op.encode(x.rows, y.rows, residual=r.rows, workspace=ws, stream=stream)
            expert.encode(layer.x.rows, layer.idx, layer.w, layer.y.rows, residual=layer.residual.rows, workspace=ews, stream=stream)
        return run

    runs = [both(at, streams[at]) for at in range(2)]
    want = []
    for at in range(2):
        runs[at]()
        torch.cuda.synchronize()
        want.append((p[at][4].rows.clone(), layers[at].y.rows.clone()))
    for _ in range(10):
        for at in range(2):
            p[at][4].rows.zero_(), layers[at].y.rows.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for at in range(2):
                runs[at]()
        torch.cuda.synchronize()
        for at in range(2):
            assert torch.equal(p[at][4].rows, want[at][0]) and torch.equal(layers[at].y.rows, want[at][1])


def test_two_graphs_share_a_workspace(gpu):
    """replayed one after the other: what one left in the workspace is nothing to the other"""
    p = [make(t, 4104, 260, seed=t) for t in (40, 300)]
    op = ops.Projection(gpu, p[0][1].rows, bias=p[0][2])
    layers = [Layer(t, 512, 264, 16, 4, 64) for t in (6, 40)]
    expert = layers[0].op(gpu)
    ws = torch.empty(max(max(op.workspace_bytes(t) for t in (40, 300)), expert.workspace_bytes(40)), dtype=torch.uint8, device="cuda")
    graphs = []
    want = []
    for at in range(2):
        x, _, _, r, y = p[at]
        layer = layers[at]

        def run():
            op.encode(x.rows, y.rows, residual=r.rows, workspace=ws)
            expert.encode(layer.x.rows, layer.idx, layer.w, layer.y.rows, residual=layer.residual.rows, workspace=ws)

        run()
        torch.cuda.synchronize()
        want.append((y.rows.clone(), layer.y.rows.clone()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
    for k in range(6):
        at = k * 5 % 2
        p[at][4].rows.zero_(), layers[at].y.rows.zero_()
        graphs[at].replay()
        torch.cuda.synchronize()
        assert torch.equal(p[at][4].rows, want[at][0]) and torch.equal(layers[at].y.rows, want[at][1])


@pytest.mark.parametrize("t, dim", [(1, 256), (70, 128), (33, 72), (40, 34)])
def test_heads_of_a_strided_output(gpu, t, dim):
    """q and k in a wider buffer to another one, tokens first: what lies between stays"""
    g = generator(t + dim)
    whole = randn(g, t, 7, dim).bfloat16()
    out = torch.full((t, 9, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    weights = [randn(g, dim).bfloat16() for _ in range(2)]
    freq = frequencies(dim // 2)
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    op = ops.HeadNorms(gpu, dim, q_weight=weights[0], k_weight=weights[1], inv_freq=freq, eps=1e-6)
    op.encode(whole[:, :4], whole[:, 5:7], positions=pos, q_out=out[:, 1:5], k_out=out[:, 6:8])
    for rows, to, weight in ((whole[:, :4], out[:, 1:5], weights[0]), (whole[:, 5:7], out[:, 6:8], weights[1])):
        want, far = heads64(rows, weight, pos.view(1, -1), freq, None, False, 1e-6, 0.0, 1.0)
        assert_near(to, want, far)
    assert (out[:, [0, 5, 8]] == 7).all()
