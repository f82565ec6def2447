"""Views of heads and of positions in mf_head_norms on the GPU, against the definition in 64 bits."""
import pytest
import torch

from dense16_cases import assert_near, generator, heads64, randn
from mference_amd import operators as ops
from test_gpu_head_norms import frequencies

pytestmark = pytest.mark.gpu


def test_one_row_of_a_long_cache(gpu):
    """one token's keys into a cache whose heads lie 2^31 elements and more apart"""
    dim, far = 64, (1 << 31) + 64
    whole = randn(generator(1), 1, 6, dim).bfloat16()
    cache = torch.empty(2 * far, dtype=torch.bfloat16, device="cuda")
    at = cache[1024:].as_strided((1, 2, dim), (dim, far, 1), 1024)
    at.fill_(7.0)
    around = [cache[1024 + h * far + s * dim:1024 + h * far + (s + 1) * dim] for h in range(2) for s in (-1, 1)]
    for v in around:
        v.fill_(7.0)
    freq, weight, positions = frequencies(dim // 2), randn(generator(2), dim).bfloat16(), torch.tensor([1234567], dtype=torch.int32, device="cuda")
    kept = whole.clone()
    ops.HeadNorms(gpu, dim, freq, q_weight=weight, k_weight=weight).encode(whole[:, :4], whole[:, 4:], positions, k_out=at)
    for got, part in ((whole[:, :4], kept[:, :4]), (at, kept[:, 4:])):
        want, off = heads64(part, weight, positions.view(1, 1), freq, None, False, 1e-6, 0.0, 1.0)
        assert_near(got, want, off)
    assert torch.equal(whole[:, 4:], kept[:, 4:]) and all((v == 7).all() for v in around)


@pytest.mark.parametrize("t", [1, 3, 130])
@pytest.mark.parametrize("rows_first", [True, False])
@pytest.mark.parametrize("dim, interleaved", [(128, False), (72, True), (50, False), (130, True)])
def test_query_key_and_value_head_by_head(gpu, t, rows_first, dim, interleaved):
    """queries and keys in place in a buffer that holds a head's query, key and value side by side, and queries to the place of the values"""
    h = 4
    whole = randn(generator(t + dim), *((t, h, 3, dim) if rows_first else (h, t, 3, dim))).bfloat16()
    view = whole if rows_first else whole.transpose(0, 1)
    kept = view.clone()
    weights, freq = [randn(generator(k), dim).bfloat16() for k in range(2)], frequencies(dim // 2)
    positions = torch.arange(t, dtype=torch.int32, device="cuda")
    op = ops.HeadNorms(gpu, dim, freq, interleaved=interleaved, q_weight=weights[0], k_weight=weights[1])
    want = [heads64(kept[:, :, i], weights[i], positions.view(1, -1), freq, None, interleaved, 1e-6, 0.0, 1.0) for i in range(2)]
    op.encode(view[:, :, 0], view[:, :, 1], positions)
    for i in range(2):
        assert_near(view[:, :, i], *want[i])
    assert torch.equal(view[:, :, 2], kept[:, :, 2])
    view.copy_(kept)
    op.encode(view[:, :, 0], positions=positions, q_out=view[:, :, 2])
    assert_near(view[:, :, 2], *want[0])
    assert torch.equal(view[:, :, :2], kept[:, :, :2])


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("dim, interleaved", [(128, False), (72, True), (130, False)])
def test_one_row_of_positions_for_all_axes(gpu, t, dim, interleaved):
    """text in a model of three axes: a row of positions expanded over them turns as three equal rows do"""
    pairs = dim // 2
    whole, weight = randn(generator(t), t, 3, dim).bfloat16(), randn(generator(9), dim).bfloat16()
    positions = torch.randint(0, 100000, (t,), generator=generator(3), device="cuda", dtype=torch.int32)
    table = ops.HeadNorms.axes_of_sections((pairs - 2 * (pairs // 3), pairs // 3, pairs // 3), turns=True)
    op = ops.HeadNorms(gpu, dim, frequencies(pairs), table, interleaved, q_weight=weight)
    got, same = torch.empty_like(whole), torch.empty_like(whole)
    op.encode(whole, positions=positions.expand(3, t), q_out=got)
    op.encode(whole, positions=positions.expand(3, t).contiguous(), q_out=same)
    assert torch.equal(got, same)
    want, off = heads64(whole, weight, positions.expand(3, t), frequencies(pairs), table, interleaved, 1e-6, 0.0, 1.0)
    assert_near(got, want, off)
    with pytest.raises(ops.MfError):
        op.encode(whole, positions=positions, q_out=got)
