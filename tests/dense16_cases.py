"""Inputs and definitions in 64 bits of the operators of layers kept in 16 bits, shared by their GPU tests."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # the most that one rounding is off, relative
ACTS = ("none", "silu", "gelu_tanh", "gelu")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def ints(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").float()


class Placed:
    """rows [t, w] inside a wider buffer, `off` elements from its start, what lies around them filled: with NaN where a call only reads (a value
    from outside a row would show in the result), with 7 where it writes"""

    def __init__(self, v, pad=0, off=0, fill=float("nan")):
        t, w = v.shape
        self.flat = torch.full((off + t * (w + pad) + 64,), fill, dtype=v.dtype, device=v.device)
        self.rows = self.flat[off:off + t * (w + pad)].view(t, w + pad)[:, pad // 2:pad // 2 + w]
        self.rows.copy_(v)
        self.before = self.flat.clone()

    def only_rows_changed(self):
        now = self.flat.clone()
        at = now.as_strided(self.rows.shape, self.rows.stride(), self.rows.storage_offset())
        at.copy_(self.before.as_strided(self.rows.shape, self.rows.stride(), self.rows.storage_offset()))
        return torch.equal(now.view(torch.int16), self.before.view(torch.int16))


def act64(z, kind):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    if kind == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    return z


def act_error(z, off, kind):
    """the most an activation in fp32 is off, where its argument is off by `off`: no activation's slope passes 1.13; the sigmoid's exponent takes
    a rounding of its argument (2^-23 |z| of at most 88, beyond which the result is nothing or z) and one ulp each of exp2, sum and reciprocal, and
    erf is good to 2^-22; all of it times |z|"""
    if kind == "none":
        return off
    return 1.13 * off + z.abs() * (2.0 ** -22 * z.abs().clamp(max=88) + 2.0 ** -21)


def sum_error(terms, magnitudes):
    """the most a sum of so many exact products is off in fp32, whatever the order: a rounding a step"""
    return terms * 2.0 ** -24 * magnitudes


def project64(x, w, bias, residual, act, gated):
    """the projection in 64 bits, and the most that fp32 sums may move it"""
    x, w = x.double(), w.double()
    rows, n = w.shape
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    off = sum_error(n + 1, size)
    if gated:
        m = rows // 2
        a, a_off = act64(z[:, :m], act), act_error(z[:, :m], off[:, :m], act)
        y, y_off = a * z[:, m:], a_off * z[:, m:].abs() + a.abs() * off[:, m:] + a_off * off[:, m:] + 2.0 ** -24 * (a * z[:, m:]).abs()
    else:
        y, y_off = act64(z, act), act_error(z, off, act)
    if residual is not None:
        y_off = y_off + 2.0 ** -24 * (y.abs() + residual.double().abs())
        y = y + residual.double()
    return y, y_off


def assert_near(got, want, off, what=""):
    """a result within its fp32 error and one rounding (of what it may have been off to)"""
    half = HALF_STEP[got.dtype]
    far = (got.double() - want).abs() - (off + half * (want.abs() + off)) - 1e-38
    worst = far.max().item() if far.numel() else 0.0
    assert not torch.isnan(far).any(), what
    assert worst <= 0.0, (what, worst, int((far > 0).sum()))


def heads64(h, weight, positions, inv_freq, axis_of_pair, interleaved, eps, weight_bias, scale):
    """norm and rotation of [t, heads, dim] in 64 bits, and the most that fp32 may move it"""
    z = h.double()
    dim = z.shape[2]
    off = torch.zeros_like(z)
    if weight is not None:
        z = z / torch.sqrt((z * z).sum(2, keepdim=True) / dim + eps) * (weight.double() + weight_bias)
        off = z.abs() * (dim / 2 + 8) * 2.0 ** -24  # a rounding a square (half of it behind the root), and of root, quotient, weight and products
    if positions is None:
        return z, off
    positions = positions.view(-1, positions.shape[-1])
    pairs = inv_freq.numel()
    axis = torch.zeros(pairs, dtype=torch.long, device=h.device) if axis_of_pair is None else axis_of_pair.long()
    turned = axis < positions.shape[0]
    angle = positions.double()[axis.clamp(max=positions.shape[0] - 1)].t() * inv_freq.double()
    c, s = [torch.where(turned, f(angle) * scale, torch.full_like(angle, one)).unsqueeze(1) for f, one in ((torch.cos, 1.0), (torch.sin, 0.0))]
    at, bt = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b, ao, bo = z[..., at].clone(), z[..., bt].clone(), off[..., at].clone(), off[..., bt].clone()
    # the angle is reduced in 64 bits and then one of fp32 up to pi (2^-23), sine and cosine are good to 2^-22
    turn = 2.0 ** -21 * abs(scale)
    z[..., at], z[..., bt] = a * c - b * s, b * c + a * s
    for place in (at, bt):
        off[..., place] = (ao + bo) * max(1.0, abs(scale)) + (a.abs() + b.abs()) * (turn + 2.0 ** -22)
    return z, off


def experts64(x, idx, w, gate_up, down, gate_up_bias=None, down_bias=None, shared_gate_up=None, shared_down=None, shared_gate=None, residual=None, act="silu"):
    """the layer of experts in 64 bits, and the most that fp32 sums and the activations' two bf16 terms may move it"""
    t, d = x.shape
    x64 = x.double()
    y = residual.double().clone() if residual is not None else torch.zeros((t, d), dtype=torch.float64, device=x.device)
    off, size = torch.zeros_like(y), y.abs()

    def mlp(rows, up, b1, dn, b2):
        a, a_off = project64(rows, up, b1, None, act, True)
        a_off = a_off + 2.0 ** -16 * a.abs()  # the second term is a bf16 of what the first leaves: 2^-8 of at most 2^-8
        wide = a.abs() + a_off
        z = a @ dn.double().t()
        z_off = a_off @ dn.double().abs().t() + sum_error(2 * dn.shape[1] + 8, wide @ dn.double().abs().t())
        if b2 is not None:
            z_off = z_off + 2.0 ** -24 * (z.abs() + b2.double().abs())
            z = z + b2.double()
        return z, z_off

    for i in range(t):
        for k in range(idx.shape[1]):
            e = int(idx[i, k]) & 0xFFFFFFFF
            if e >= gate_up.shape[0]:
                continue
            z, z_off = mlp(x[i:i + 1], gate_up[e], None if gate_up_bias is None else gate_up_bias[e], down[e], None if down_bias is None else down_bias[e])
            s = w[i, k].double()
            y[i] += s * z[0]
            size[i] += (s * z[0]).abs()
            off[i] += s.abs() * z_off[0]
    if shared_down is not None:
        z, z_off = mlp(x, shared_gate_up, None, shared_down, None)
        if shared_gate is not None:
            logit, l_off = x64 @ shared_gate.double(), sum_error(d, x64.abs() @ shared_gate.double().abs())
            g = torch.sigmoid(logit).unsqueeze(1)
            z_off = z_off * g + z.abs() * (0.25 * l_off + 2.0 ** -22 * logit.abs() + 2.0 ** -21).unsqueeze(1)
            z = z * g
        y, off, size = y + z, off + z_off, size + z.abs()
    return y, off + (idx.shape[1] + 3) * 2.0 ** -24 * size
