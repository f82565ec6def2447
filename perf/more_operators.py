"""The operators of layers that a model keeps in 16 bits, as timed cases: the projection with bias, activation (plain or gated) and
residual in its epilogue, the norms of query and key heads with the rotation of positions of several axes, and the layer of 16-bit
experts for a few tokens.

  own              False: run() computes the plain form; True: it calls the library's operators
  listed()         the cases with names
  draw(rng)        one more case of the same ranges
  prepare(case, seed)  inputs, weights and buffers a program holds before the call
  run(state)       one pass
  work(case)       bytes and operations a pass cannot do without
  exact(case, seed)    what run returns, in 64 bits from the definition
"""
import functools
import math
import random

import torch

own = False

ACTIVATIONS = ("none", "silu", "gelu_tanh", "gelu")


def _project(t, n, m, **more):
    """gated: the weight has 2 m rows, gate rows first, and the result is act(gate) * up.  part: x is a column range of a wider buffer."""
    c = dict(kind="project", t=t, n=n, m=m, act="none", gated=False, bias=False, residual=False, y32=False, part=False)
    c.update(more)
    return c


def _heads(t, q, k, dim, **more):
    """q and k heads of `dim` in one buffer of a row a token (with as many value heads as key heads behind them), normed and rotated in
    place; rot: how much of a head is rotated; axes: positions a token; order: how the pairs of a head take turns among the axes"""
    c = dict(kind="heads", t=t, q=q, k=k, dim=dim, rot=dim, axes=1, order="blocks", interleaved=False, norm=True, weight_bias=0.0, offset=0, base=1e6)
    c.update(more)
    return c


def _experts(t, d, f, experts, top_k, **more):
    c = dict(kind="experts", t=t, d=d, f=f, experts=experts, top_k=top_k, shared_f=0, act="silu", bias=False, residual=True)
    c.update(more)
    return c


def listed():
    return [
        # one token: queries, keys and values of the benchmark's hidden size in one product with its bias
        dict(_project(1, 2048, 5120, bias=True), name="project-token"),
        # a draft of three tokens being verified: the dense MLP's gate and up halves with silu(gate) * up
        dict(_project(4, 5120, 17408, gated=True, act="silu"), name="project-verify-4"),
        # eight requests decoded together: the dense MLP's down projection and the residual add behind it
        dict(_project(8, 17408, 5120, residual=True), name="project-down-8"),
        # a decode batch of many requests, fp32 results (a head over a part of the vocabulary), x inside a wider buffer
        dict(_project(200, 2816, 2113, y32=True, part=True), name="project-batch-200"),
        # patches of an image through an encoder's MLP with bias and gelu
        dict(_project(777, 1280, 5120, bias=True, act="gelu_tanh"), name="project-patches-777"),
        # a long prompt chunk through the dense model's gate and up
        dict(_project(4096, 5120, 17408, gated=True, act="silu"), name="project-prompt-4096"),
        # one token far into its text, rotation of a quarter of every head, weights stored as differences from one
        dict(_heads(1, 16, 2, 256, rot=64, weight_bias=1.0, offset=200000, base=1e7), name="heads-token"),
        # image and text rows: time, height and width take turns among the pairs
        dict(_heads(777, 32, 8, 128, axes=3, order="turns"), name="heads-mixed-777"),
        # a long prompt chunk
        dict(_heads(8192, 40, 8, 128, offset=50000), name="heads-chunk-8192"),
        # one token of the benchmark's layer, kept in 16 bits
        dict(_experts(1, 2048, 512, 256, 8, shared_f=512), name="experts-token"),
        # a decode batch of eight
        dict(_experts(8, 2816, 704, 128, 8, act="gelu_tanh", shared_f=2112), name="experts-batch-8"),
        # a decode batch of many requests, experts with biases
        dict(_experts(61, 2048, 1024, 64, 8, bias=True), name="experts-batch-61"),
    ]


def _of(name):
    return next(c for c in listed() if c["name"] == name)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _size(rng, lo, hi, odd):
    v = _log_int(rng, lo, hi)
    return v if rng.random() < odd else max(lo, v // 64 * 64)


def draw(rng):
    kind = rng.choice(["project", "project", "heads", "experts"])
    if kind == "project":
        c = _project(_log_int(rng, 1, 4096), _size(rng, 64, 17408, 0.2), _size(rng, 64, 17408, 0.2), act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5,
                     gated=rng.random() < 0.3, residual=rng.random() < 0.4, y32=rng.random() < 0.25, part=rng.random() < 0.2)
        most = work(_of("project-prompt-4096"))["flops"]
        while work(c)["flops"] > most:
            c["t"] = c["t"] * 3 // 4
        return c
    if kind == "heads":
        dim = rng.choice([64, 72, 80, 96, 128, 128, 128, 192, 256, 256])
        k = rng.choice([1, 2, 4, 8, 8, 16])
        c = _heads(_log_int(rng, 1, 8192), k * rng.choice([1, 2, 4, 5, 8]), k, dim, rot=rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]), axes=rng.choice([1, 1, 2, 3, 3]),
                   order=rng.choice(["blocks", "turns"]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.8, weight_bias=rng.choice([0.0, 0.0, 1.0]),
                   offset=rng.choice([0, 0, 1000, 200000, 1000000]), base=rng.choice([1e4, 1e6, 1e7]))
        most = work(_of("heads-chunk-8192"))["bytes"]
        while work(c)["bytes"] > most:
            c["t"] = c["t"] * 3 // 4
        return c
    d, f = _log_int(rng, 256, 5120) // 8 * 8, _log_int(rng, 64, 2048) // 8 * 8
    if rng.random() < 0.7:
        d, f = max(256, d // 64 * 64), max(64, f // 64 * 64)
    experts = _log_int(rng, 8, 256)
    while 3 * experts * d * f > 400_000_000:
        experts = experts * 3 // 4
    top_k = min(rng.choice([1, 2, 4, 6, 8, 8]), experts)
    return _experts(_log_int(rng, 1, 64), d, f, experts, top_k, shared_f=rng.choice([0, 0, f, 2 * f]), act=rng.choice(["silu", "silu", "gelu_tanh", "gelu"]),
                    bias=rng.random() < 0.3, residual=rng.random() < 0.7)


# ------------------------------------------------------------------ preparation

def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _bf16(t):
    return t.to(torch.bfloat16)


def _weights(gen, *shape):
    """bf16 weights of a spread that keeps the size of what they are multiplied with, made a part at a time"""
    w = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    rows = w.view(-1, shape[-1])
    for part in rows.split(max(1, (1 << 28) // shape[-1])):
        part.copy_(_randn(gen, *part.shape) * shape[-1] ** -0.5)
    return w


def _positions(case, salt):
    """[axes][t] whole numbers.  The first axis counts on (a run of image rows shares its place in time), the others walk a grid."""
    rng = random.Random(31 * salt + 11)
    t, axes = case["t"], case["axes"]
    start = case["offset"] + rng.randint(0, 1000)
    if axes == 1:
        return [[start + i for i in range(t)]]
    rows, at = [], start
    while len(rows) < t:
        wide, high = rng.randint(4, 40), rng.randint(4, 40)
        rows += [(at, at + y, at + x)[:axes] for y in range(high) for x in range(wide)]
        at += max(wide, high)
        text = rng.randint(1, 200)
        rows += [(at + i,) * axes for i in range(text)]
        at += text
    return [list(axis) for axis in zip(*rows[:t])]


def _axis_of_pair(case):
    pairs, axes = case["rot"] // 2, case["axes"]
    return [p % axes if case["order"] == "turns" else min(p * axes // pairs, axes - 1) for p in range(pairs)]


def _routes(case, salt):
    """the experts of every token, in a plain list, so that work() can count what is live (salt 0) without a GPU: some experts are asked for more often"""
    rng = random.Random(57 * salt + 7)
    liked = [rng.expovariate(1.0) + 0.05 for _ in range(case["experts"])]
    return [sorted(range(case["experts"]), key=lambda e: -liked[e] * rng.random())[:case["top_k"]] for _ in range(case["t"])]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1_000_003 * int(seed) + 41)
    s, t = {"case": case}, case["t"]
    if case["kind"] == "project":
        n, m = case["n"], case["m"]
        rows = 2 * m if case["gated"] else m
        s["x"] = _bf16(_randn(gen, t, n + 64))[:, 64:] if case["part"] else _bf16(_randn(gen, t, n))
        s["w"] = _weights(gen, rows, n)
        s["bias"] = _bf16(0.3 * _randn(gen, rows)) if case["bias"] else None
        kind = torch.float32 if case["y32"] else torch.bfloat16
        s["residual"] = _randn(gen, t, m).to(kind) if case["residual"] else None
        s["y"] = torch.zeros((t, m), dtype=kind, device="cuda")
        return s
    if case["kind"] == "heads":
        q, k, dim = case["q"], case["k"], case["dim"]
        s["buffer"] = _bf16(_randn(gen, t, q + 2 * k, dim) * 1.5)
        shift = 1.0 - case["weight_bias"]
        for name in ("q_weight", "k_weight"):
            s[name] = _bf16(shift + 0.2 * _randn(gen, dim)) if case["norm"] else None
        pairs = case["rot"] // 2
        s["inv_freq"] = torch.tensor([case["base"] ** (-p / pairs) for p in range(pairs)], dtype=torch.float32, device="cuda")
        s["axis_of_pair"] = torch.tensor(_axis_of_pair(case), dtype=torch.uint8, device="cuda")
        s["positions"] = torch.tensor(_positions(case, int(seed)), dtype=torch.int32, device="cuda")
        return s
    d, f, fs, e = case["d"], case["f"], case["shared_f"], case["experts"]
    s["x"] = _bf16(_randn(gen, t, d))
    s["gate_up"], s["down"] = _weights(gen, e, 2 * f, d), _weights(gen, e, d, f)
    s["gate_up_bias"] = _bf16(0.2 * _randn(gen, e, 2 * f)) if case["bias"] else None
    s["down_bias"] = _bf16(0.2 * _randn(gen, e, d)) if case["bias"] else None
    s["shared_gate_up"] = _weights(gen, 2 * fs, d) if fs else None
    s["shared_down"] = _weights(gen, d, fs) if fs else None
    s["shared_gate"] = _weights(gen, d) if fs else None
    s["indices"] = torch.tensor(_routes(case, int(seed)), dtype=torch.int32, device="cuda")
    s["weights"] = torch.softmax(_randn(gen, t, case["top_k"]), 1)
    s["residual"] = _bf16(_randn(gen, t, d)) if case["residual"] else None
    s["y"] = torch.zeros((t, d), dtype=torch.bfloat16, device="cuda")
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------ the plain forms

def _act(z, kind):
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    return z


def _plain_project(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().t()
    if c["bias"]:
        z = z + s["bias"].float()
    a = _act(z[:, :c["m"]], c["act"]) * z[:, c["m"]:] if c["gated"] else _act(z, c["act"])
    if c["residual"]:
        a = s["residual"].float() + a
    s["y"].copy_(a)
    return {"y": s["y"]}


def _plain_heads(s):
    c = s["case"]
    rot, pairs = c["rot"], c["rot"] // 2
    at = s["positions"].double()[s["axis_of_pair"].long()]  # [pairs, t]
    angle = (at * s["inv_freq"].double().unsqueeze(1)).t()  # far positions: in 64 bits
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def one(heads, weight):
        z = heads.float()
        if c["norm"]:
            z = z * torch.rsqrt(z.square().mean(2, keepdim=True) + 1e-6) * (weight.float() + c["weight_bias"])
        out = z.clone()
        if c["interleaved"]:
            a, b = z[..., 0:rot:2], z[..., 1:rot:2]
            out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = z[..., :pairs], z[..., pairs:rot]
            out[..., :pairs], out[..., pairs:rot] = a * cos - b * sin, b * cos + a * sin
        heads.copy_(out)

    one(s["buffer"][:, :c["q"]], s["q_weight"])
    one(s["buffer"][:, c["q"]:c["q"] + c["k"]], s["k_weight"])
    return {"heads": s["buffer"]}


def _plain_experts(s):
    """every token through every expert, the results of those it did not ask for left out"""
    c = s["case"]
    t, d, f, fs, e = c["t"], c["d"], c["f"], c["shared_f"], c["experts"]
    x = s["x"].float()
    share = torch.zeros((t, e), device="cuda").scatter_(1, s["indices"].long(), s["weights"])
    z = (x @ s["gate_up"].float().view(e * 2 * f, d).t()).view(t, e, 2 * f)
    if c["bias"]:
        z = z + s["gate_up_bias"].float()
    a = _act(z[..., :f], c["act"]) * z[..., f:] * share.unsqueeze(2)
    y = a.view(t, e * f) @ s["down"].float().permute(0, 2, 1).reshape(e * f, d)
    if c["bias"]:
        y = y + share @ s["down_bias"].float()
    if fs:
        z = x @ s["shared_gate_up"].float().t()
        a = _act(z[:, :fs], c["act"]) * z[:, fs:]
        y = y + (a @ s["shared_down"].float().t()) / (1.0 + torch.exp(-(x @ s["shared_gate"].float()))).unsqueeze(1)
    if c["residual"]:
        y = s["residual"].float() + y
    s["y"].copy_(y)
    return {"y": s["y"]}


# ------------------------------------------------------------------ one pass

@functools.lru_cache(maxsize=None)
def _context():
    from mference_amd import operators as ops
    return ops.MetalContext(0)


def _held(s):
    """the operator, views and workspace that a program makes once and keeps"""
    if "held" not in s:
        from mference_amd import operators as ops
        c, ctx, h = s["case"], _context(), {}
        act = dict(zip(ACTIVATIONS, (ops.ACT_NONE, ops.ACT_SILU, ops.ACT_GELU_TANH, ops.ACT_GELU)))
        if c["kind"] == "heads":
            h["op"] = ops.HeadNorms(ctx, c["dim"], inv_freq=s["inv_freq"], axis_of_pair=s["axis_of_pair"] if c["axes"] > 1 else None, interleaved=c["interleaved"],
                                    q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6, weight_bias=c["weight_bias"])
            h["q"], h["k"] = s["buffer"][:, :c["q"]], s["buffer"][:, c["q"]:c["q"] + c["k"]]
        else:
            if c["kind"] == "project":
                h["op"] = ops.Projection(ctx, s["w"], bias=s["bias"], activation=act[c["act"]], gated=c["gated"])
            else:
                h["op"] = ops.Bf16Experts(ctx, s["gate_up"], s["down"], c["top_k"], gate_up_bias=s["gate_up_bias"], down_bias=s["down_bias"], activation=act[c["act"]],
                                          shared_gate_up=s["shared_gate_up"], shared_down=s["shared_down"], shared_gate=s["shared_gate"])
            h["workspace"] = torch.empty(h["op"].workspace_bytes(c["t"]), dtype=torch.uint8, device="cuda")
        s["held"] = h
    return s["held"]


def _own(s):
    c, h = s["case"], _held(s)
    if c["kind"] == "heads":
        h["op"].encode(h["q"], h["k"], positions=s["positions"])
        return {"heads": s["buffer"]}
    if c["kind"] == "project":
        h["op"].encode(s["x"], s["y"], residual=s["residual"], workspace=h["workspace"])
    else:
        h["op"].encode(s["x"], s["indices"], s["weights"], s["y"], residual=s["residual"], workspace=h["workspace"])
    return {"y": s["y"]}


def run(state):
    if own:
        return _own(state)
    return {"project": _plain_project, "heads": _plain_heads, "experts": _plain_experts}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass needs

def work(case):
    t = case["t"]
    if case["kind"] == "project":
        n, m, rows = case["n"], case["m"], case["m"] * (2 if case["gated"] else 1)
        element = 4 if case["y32"] else 2
        return {"bytes": 2 * (t * n + rows * n) + (2 * rows if case["bias"] else 0) + t * m * element * (2 if case["residual"] else 1), "flops": 2 * t * n * rows}
    if case["kind"] == "heads":
        elements = t * (case["q"] + case["k"]) * case["dim"]
        return {"bytes": 4 * elements + 4 * t * case["axes"] + (4 * case["dim"] if case["norm"] else 0) + 3 * case["rot"], "flops": 7 * elements}
    d, f, fs = case["d"], case["f"], case["shared_f"]
    live = len({e for row in _routes(case, 0) for e in row})
    routes = t * case["top_k"]
    return {"bytes": 2 * (live * (3 * d * f + (2 * f + d if case["bias"] else 0)) + 3 * d * fs + (d if fs else 0)) + 8 * routes + 2 * t * d * (3 if case["residual"] else 2),
            "flops": 6 * d * (routes * f + t * fs)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _act64(z, kind):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    if kind == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    return z


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "project":
        m, ys = case["m"], []
        x, bias = s["x"].double(), s["bias"].double() if case["bias"] else torch.zeros(s["w"].shape[0], dtype=torch.float64, device="cuda")
        for at in range(0, m, 4096):
            rows = slice(at, min(m, at + 4096))
            z = torch.nn.functional.linear(x, s["w"][:m][rows].double(), bias[:m][rows])
            z = _act64(z, case["act"])
            if case["gated"]:
                z = z * torch.nn.functional.linear(x, s["w"][m:][rows].double(), bias[m:][rows])
            ys.append(z)
        y = torch.cat(ys, 1)
        return {"y": y + s["residual"].double() if case["residual"] else y}
    if case["kind"] == "heads":
        rot, pairs = case["rot"], case["rot"] // 2
        z = s["buffer"].double()
        angle = torch.stack([s["positions"][axis].double() * s["inv_freq"][p].double() for p, axis in enumerate(_axis_of_pair(case))], 1)
        turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
        for part, weight in ((slice(0, case["q"]), s["q_weight"]), (slice(case["q"], case["q"] + case["k"]), s["k_weight"])):
            h = z[:, part]
            if case["norm"]:
                h = h / torch.sqrt((h * h).sum(2, keepdim=True) / case["dim"] + 1e-6) * (weight.double() + case["weight_bias"])
            first, second = (h[..., 0:rot:2], h[..., 1:rot:2]) if case["interleaved"] else (h[..., :pairs], h[..., pairs:rot])
            turned = torch.complex(first, second) * turn
            if case["interleaved"]:
                h = torch.cat([torch.view_as_real(turned).flatten(2), h[..., rot:]], 2)
            else:
                h = torch.cat([turned.real, turned.imag, h[..., rot:]], 2)
            z[:, part] = h
        return {"heads": z}
    f, fs = case["f"], case["shared_f"]
    x = s["x"].double()
    y = s["residual"].double() if case["residual"] else torch.zeros_like(x)
    for e in sorted(set(s["indices"].flatten().tolist())):
        token, rank = (s["indices"] == e).nonzero(as_tuple=True)
        z = x[token] @ s["gate_up"][e].double().t()
        if case["bias"]:
            z = z + s["gate_up_bias"][e].double()
        z = (_act64(z[:, :f], case["act"]) * z[:, f:]) @ s["down"][e].double().t()
        if case["bias"]:
            z = z + s["down_bias"][e].double()
        y.index_add_(0, token, z * s["weights"][token, rank].double().unsqueeze(1))
    if fs:
        z = x @ s["shared_gate_up"].double().t()
        z = (_act64(z[:, :fs], case["act"]) * z[:, fs:]) @ s["shared_down"].double().t()
        y = y + z * torch.sigmoid(x @ s["shared_gate"].double()).unsqueeze(1)
    return {"y": y}
