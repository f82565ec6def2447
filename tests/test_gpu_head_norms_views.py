"""Views of heads in mf_head_norms on the GPU, against the definition in 64 bits."""
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
