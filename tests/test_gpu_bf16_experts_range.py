"""Activations of 16-bit experts that fp32 holds and bf16 rounds up to an infinity: between 2^127 (2 - 2^-8) and 2^128."""
import pytest
import torch

from mference_amd import operators as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 8, 20, 64])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("shared", [False, True])
def test_activations_near_the_end_of_fp32(gpu, t, sign, shared):
    d = f = 64
    half = 181.0 / 128.0  # its square, times 2^127, is 2^127 * 1.99957: exact in fp32, and nearer to 2^128 than to the last bf16
    up = torch.zeros(2 * f, d, dtype=torch.bfloat16, device="cuda")
    up[:f, 0] = half * 2.0 ** 63
    up[f:, 0] = sign * half * 2.0 ** 64
    down = (torch.eye(d, f, device="cuda") * 2.0 ** -64).bfloat16()
    x = torch.zeros(t, d, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1.0
    y = torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
    idx, w = torch.full((t, 1), -1 if shared else 0, dtype=torch.int32, device="cuda"), torch.ones(t, 1, device="cuda")
    more = dict(shared_gate_up=up, shared_down=down) if shared else {}
    ops.Bf16Experts(gpu, up.unsqueeze(0).contiguous(), down.unsqueeze(0).contiguous(), 1, activation=ops.ACT_NONE, **more).encode(x, idx, w, y)
    want = torch.full((t, d), sign * half * half * 2.0 ** 63, dtype=torch.float64, device="cuda").bfloat16()  # (one product a result: exact but for its rounding)
    assert torch.equal(y, want)


@pytest.mark.parametrize("t", [1, 20])
def test_an_infinite_activation_stays_one(gpu, t):
    d = f = 64
    up = torch.zeros(2 * f, d, dtype=torch.bfloat16, device="cuda")
    up[:, 0] = 2.0 ** 64
    up[f, 0] = -2.0 ** 64
    down = torch.eye(d, f, device="cuda").bfloat16()
    x = torch.zeros(t, d, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1.0
    y = torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
    idx, w = torch.zeros(t, 1, dtype=torch.int32, device="cuda"), torch.ones(t, 1, device="cuda")
    ops.Bf16Experts(gpu, up.unsqueeze(0).contiguous(), down.unsqueeze(0).contiguous(), 1, activation=ops.ACT_NONE).encode(x, idx, w, y)
    assert not torch.isfinite(y).any()  # (an infinity times the zeros of the other rows: not a number there)
