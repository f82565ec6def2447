"""The activations of the 16-bit operators where they are small: negative arguments, whose results are compared by their own size."""
import math

import pytest
import torch

from dense16_cases import ACTS, HALF_STEP, act64
from mference_amd import operators as ops

pytestmark = pytest.mark.gpu


def arguments():
    """bf16 values of -12 .. 12, closely where a sum of one and erf loses its digits"""
    v = torch.cat([torch.linspace(-12, 12, 385), torch.linspace(-6, -3.5, 320), torch.tensor([-1e-20, -1e-3, 0.0, 1e-3])])
    return torch.unique(v.bfloat16()).cuda()


def relative(z, kind):
    """the most that an activation in fp32 is off for an exact argument, relative to it: the exponent's roundings times its size (a constant and a
    product each, four more of the tanh form's cubic; erfc moves by 2 u^2 + 1 of its argument's), 1 ulp each of exp2 and reciprocal, 16 of erfc, and
    two more roundings"""
    z = z.abs()
    if kind == "silu":
        return (2 * z + 6) * 2.0 ** -23
    if kind == "gelu_tanh":
        return (6 * 2 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3) + 6) * 2.0 ** -23
    return (z * z + 1 + 16 + 2) * 2.0 ** -23


def check(got, z, kind, factor=1.0):
    """got: kind(z) * factor, narrowed once; a product by the factor is one more rounding"""
    want = act64(z.double(), kind)
    keep = want.abs() > 1e-36  # (gelu_tanh falls off faster: what is below 2^-119 is 0)
    off = relative(z.double(), kind) + 2.0 ** -23
    far = (got.double() - want * factor).abs() - (off + HALF_STEP[got.dtype] * (1 + off)) * (want * factor).abs()
    assert (far <= 0)[..., keep].all(), (kind, far[..., keep].max().item())


@pytest.mark.parametrize("kind", ACTS[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 12, 40, 600])
def test_projection(gpu, t, dtype, kind):
    z = arguments()
    x = torch.zeros(t, 64, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = 1.0
    w = torch.zeros(z.numel(), 64, dtype=torch.bfloat16, device="cuda")
    w[:, 3] = z
    y = torch.empty(t, z.numel(), dtype=dtype, device="cuda")
    ops.Projection(gpu, w, activation=ACTS.index(kind)).encode(x, y)
    check(y, z, kind)
    up = torch.zeros_like(w)
    up[:, 3] = 2.0 ** 30
    ops.Projection(gpu, torch.cat([w, up]), activation=ACTS.index(kind), gated=True).encode(x, y)
    check(y, z, kind, 2.0 ** 30)


@pytest.mark.parametrize("kind", ACTS[1:])
@pytest.mark.parametrize("t", [1, 20])
def test_experts(gpu, t, kind):
    z = arguments()
    f = (z.numel() + 7) // 8 * 8
    gate_up = torch.zeros(1, 2 * f, 8, dtype=torch.bfloat16, device="cuda")
    gate_up[0, :z.numel(), 3] = z
    gate_up[0, f:, 3] = 2.0 ** 30
    d = f
    x = torch.zeros(t, d, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = 1.0
    wide = torch.zeros(1, 2 * f, d, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :8] = gate_up
    down = torch.eye(d, f, device="cuda").bfloat16().unsqueeze(0)
    y = torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
    idx, weight = torch.zeros(t, 1, dtype=torch.int32, device="cuda"), torch.ones(t, 1, device="cuda")
    ops.Bf16Experts(gpu, wide.contiguous(), down.contiguous(), 1, activation=ACTS.index(kind)).encode(x, idx, weight, y)
    want = act64(z.double(), kind) * 2.0 ** 30
    off = relative(z.double(), kind) + 2.0 ** -23 + 2.0 ** -16  # (two bf16 terms of an activation)
    far = (y[:, :z.numel()].double() - want).abs() - (off + HALF_STEP[y.dtype] * (1 + off)) * want.abs()
    keep = want.abs() > 1e-27
    assert (far <= 0)[:, keep].all(), (kind, far[:, keep].max().item())
