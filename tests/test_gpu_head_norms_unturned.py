"""Pairs whose axis is none, in mf_head_norms: they are not turned, whatever their elements hold."""
import pytest
import torch

from dense16_cases import assert_near, generator, heads64, randn
from mference_amd import operators as ops
from test_gpu_head_norms import frequencies

pytestmark = pytest.mark.gpu

CASES = [(128, 64, False), (128, 64, True), (128, 16, False), (72, 36, False), (72, 36, True), (50, 25, False), (50, 25, True), (50, 10, True), (130, 65, False), (130, 65, True), (6, 3, True), (3, 1, False)]


def elements(dim, pairs, interleaved):
    """element numbers of the pairs, and the table that leaves every second pair without an axis"""
    p = torch.arange(pairs, device="cuda")
    first, second = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
    table = torch.where(p % 2 == 0, 255, p % 4 // 2 * 2).to(torch.uint8)  # none, axis 0, none, axis 2 of two axes: none as well
    return first, second, table, table >= 2


@pytest.mark.parametrize("dim, pairs, interleaved", CASES)
@pytest.mark.parametrize("scale", [1.0, 0.75, 0.0])
def test_they_are_copied(gpu, dim, pairs, interleaved, scale):
    first, second, table, none = elements(dim, pairs, interleaved)
    whole = randn(generator(dim + pairs), 5, 4, dim).bfloat16()
    whole[1, 0, first[none]] = float("inf")
    whole[2, 1, second[none]] = float("nan")
    whole[3, 2, first[none]] = -float("inf")
    positions = torch.tensor([[0, 1, 7, 1000, 123456], [3, 1, 4, 1, 5]], dtype=torch.int32, device="cuda")
    out = torch.full_like(whole, 7.0)
    ops.HeadNorms(gpu, dim, frequencies(pairs, 1e4), table, interleaved, rotation_scale=scale).encode(whole, positions=positions, q_out=out)
    still = torch.ones(dim, dtype=torch.bool, device="cuda")
    still[first[~none]] = False
    still[second[~none]] = False
    assert torch.equal(out[:, :, still].view(torch.int16), whole[:, :, still].view(torch.int16))
    if (~none).any():  # the others as the definition has them
        clean = whole.clone()
        clean[:, :, still] = 0
        want, off = heads64(clean, None, positions, frequencies(pairs, 1e4), table, interleaved, 0, 0, scale)
        assert_near(out[:, :, ~still], want[:, :, ~still], off[:, :, ~still])


@pytest.mark.parametrize("dim, pairs, interleaved", CASES)
def test_beside_an_infinity_of_a_normed_head(gpu, dim, pairs, interleaved):
    """the norm leaves 0 for the others of the head, the other one of the pair among them"""
    first, second, table, none = elements(dim, pairs, interleaved)
    whole = randn(generator(dim), 3, 2, dim).bfloat16()
    at = int(first[none][-1])
    whole[1, 1, at] = float("inf")
    weight = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
    positions = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    ops.HeadNorms(gpu, dim, frequencies(pairs, 1e4), table, interleaved, q_weight=weight).encode(whole, positions=positions)
    rest = torch.arange(dim, device="cuda") != at
    assert torch.isnan(whole[1, 1, at]) and not whole[1, 1, rest].any()
