"""The operators of an MLP block whose rows carry low-rank adapters, as timed cases: the adapters of many requests beside
shared projections, the grouping of a batch's rows by adapter, and the norms around a block with its gate and residual scale.

  own              False: run() computes the plain form; True: it calls the library's operators
  listed()         the cases with names
  draw(rng)        one more case of the same ranges
  prepare(case, seed)  inputs, adapter pools and buffers a program holds before the call
  run(state)       one pass
  work(case)       bytes and operations a pass cannot do without
  exact(case, seed)    what run returns, in 64 bits from the definition
"""
import functools
import random

import torch

own = False

# kinds of gate of the norm case: none, one logit a row, one logit an element (both through a sigmoid), one factor a channel
GATES = ("none", "row", "element", "channel")


def _adapters(t, n, m0, m1, adapters, rank, **more):
    """m1 = 0: one projection; else two that read the same x.  order: one request ("one"), requests one behind the other
    ("runs"), or single rows of many requests ("mixed").  bare: share of the rows without an adapter.  fused: both results
    are column ranges of one buffer."""
    c = dict(kind="adapters", t=t, n=n, m0=m0, m1=m1, adapters=adapters, rank=rank, ranks="full", order="mixed", bare=0.0, y32=False, fused=False, grouped=False)
    c.update(more)
    return c


def _norm(t, d, **more):
    c = dict(kind="norm", t=t, d=d, gate="none", post=True, pre=True, delta32=False, residual_scale=1.0, branch_scale=1.0, weight_bias=0.0)
    c.update(more)
    return c


def listed():
    return [
        # one token of one request through the gate and up projections of the benchmark's shared expert
        dict(_adapters(1, 2048, 512, 512, 16, 16, order="one"), name="adapters-token"),
        # a draft of three tokens being verified: four rows of one request, gate and up of the dense MLP
        dict(_adapters(4, 5120, 17408, 17408, 8, 32, order="one"), name="adapters-verify-4"),
        # eight requests decoded together, each with its adapter: the dense MLP's down projection, kept in fp32
        dict(_adapters(8, 17408, 5120, 0, 32, 16, y32=True), name="adapters-down-8-f32"),
        # a decode batch of many requests in any order, ranks of several sizes, some rows without an adapter, grouped first
        dict(_adapters(200, 2816, 2112, 2112, 48, 24, ranks="mixed", bare=0.1, grouped=True), name="adapters-batch-200"),
        # a prompt batch of a ragged length, large ranks
        dict(_adapters(777, 4096, 2048, 2048, 5, 64, order="runs", bare=0.05), name="adapters-prompt-777"),
        # a long prompt chunk of a few requests through gate and up of the dense MLP, one buffer for both
        dict(_adapters(4096, 5120, 17408, 17408, 12, 16, order="runs", fused=True), name="adapters-prompt-4096"),
        # the rows of a decode batch, once a step
        dict(kind="group", t=200, adapters=48, order="mixed", bare=0.1, name="group-200"),
        # the rows of a large mixed batch over a large pool
        dict(kind="group", t=16384, adapters=512, order="mixed", bare=0.02, name="group-16384"),
        # between two blocks, one token: residual add, norm in front of the next block, the block's output under a scalar gate
        dict(_norm(1, 2048, gate="row", post=False), name="norm-token"),
        # a decode batch in layers with a norm behind the block too, weights stored as differences from one, scaled stream
        dict(_norm(8, 2816, weight_bias=1.0, residual_scale=0.875, branch_scale=0.875), name="norm-batch-8"),
        # a prompt of a ragged length, gated element by element, the block's output as the fp32 result of its projection
        dict(_norm(777, 4096, gate="element", delta32=True, branch_scale=0.22), name="norm-prompt-777"),
        # a long prompt chunk of the dense model
        dict(_norm(8192, 5120, gate="channel"), name="norm-chunk-8192"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _cost(c):
    """what bounds the two sides of an adapter case: bytes of the rows, and the plain form's products over the whole pool"""
    m = c["m0"] + c["m1"]
    return c["t"] * (c["n"] + 4 * m) + c["adapters"] * c["rank"] * (c["n"] + m) * 4, c["t"] * c["adapters"] * c["rank"] * (c["n"] + m)


def draw(rng):
    kind = rng.choice(["adapters", "adapters", "adapters", "group", "norm", "norm"])
    if kind == "group":
        return dict(kind="group", t=_log_int(rng, 16, 65536), adapters=_log_int(rng, 4, 1024), order=rng.choice(["mixed", "runs"]), bare=rng.choice([0.0, 0.1, 0.5]))
    if kind == "norm":
        d = _log_int(rng, 64, 16384)
        d = d if rng.random() < 0.3 else max(64, d // 64 * 64)
        t = min(_log_int(rng, 1, 8192), 8192 * 5120 // d)
        gate, post = rng.choice(GATES), rng.random() < 0.6
        scale = rng.choice([1.0, 1.0, 0.5, 0.875])
        return _norm(t, d, gate=gate, post=post, pre=rng.random() < 0.85, delta32=rng.random() < 0.3, residual_scale=scale,
                     branch_scale=rng.choice([1.0, scale, 0.22]), weight_bias=rng.choice([0.0, 0.0, 1.0]))
    c = _adapters(_log_int(rng, 1, 4096), 64 * _log_int(rng, 8, 272), 64 * _log_int(rng, 2, 272), 0, _log_int(rng, 1, 64), rng.choice([8, 16, 16, 32, 32, 64, 128]))
    if rng.random() < 0.25:
        c["m0"] += rng.randint(1, 63)
    if rng.random() < 0.5:
        c["m1"] = c["m0"]
        c["fused"] = rng.random() < 0.4
    c.update(ranks=rng.choice(["full", "full", "mixed"]), order=rng.choice(["one", "mixed", "runs"]), bare=rng.choice([0.0, 0.0, 0.1]), y32=rng.random() < 0.25)
    rows, products = _cost(_of(listed(), "adapters-prompt-4096"))
    while _cost(c)[0] > rows or _cost(c)[1] > products:
        if c["adapters"] > 8:
            c["adapters"] = c["adapters"] * 3 // 4
        else:
            c["t"] = c["t"] * 3 // 4
    c["grouped"] = c["order"] == "mixed" and c["t"] > 16
    return c


def _of(cases, name):
    return next(c for c in cases if c["name"] == name)


# ------------------------------------------------------------------ preparation

def _ids(case, salt):
    """the adapter of every row: a plain list, so that work() can count what is live (salt 0) without a GPU"""
    rng = random.Random(9176 * salt + 5)
    t, n = case["t"], case["adapters"]
    if case["order"] == "one":
        ids = [rng.randrange(n)] * t
    elif case["order"] == "mixed":
        ids = [rng.randrange(n) for _ in range(t)]
    else:
        ids = []
        while len(ids) < t:
            ids += [rng.randrange(n)] * rng.randint(max(1, t // 16), max(1, t // 4))
        ids = ids[:t]
    return [-1 if rng.random() < case["bare"] else a for a in ids]


def _ranks(case, salt):
    rng = random.Random(77 * salt + 3)
    full = case["rank"]
    return [full if case["ranks"] == "full" else rng.randint(max(1, full // 3), full) for _ in range(case["adapters"])]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _bf16(t):
    return t.to(torch.bfloat16)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1_000_003 * int(seed) + 29)
    t, s = case["t"], {"case": case}
    if case["kind"] == "norm":
        d = case["d"]
        s["hidden"] = _bf16(_randn(gen, t, d) * 2.0)
        delta = _randn(gen, t, d) * 0.7
        s["delta"] = delta if case["delta32"] else _bf16(delta)
        shift = 1.0 - case["weight_bias"]
        s["post"] = _bf16(shift + 0.2 * _randn(gen, d)) if case["post"] else None
        s["pre"] = _bf16(shift + 0.2 * _randn(gen, d)) if case["pre"] else None
        shape = {"none": None, "row": (t, 1), "element": (t, d), "channel": (d,)}[case["gate"]]
        s["gate"] = None if shape is None else _bf16(_randn(gen, *shape))
        s["out"] = torch.zeros((t, d), dtype=torch.bfloat16, device="cuda") if case["pre"] else None
        return s
    s["ids"] = torch.tensor(_ids(case, int(seed)), dtype=torch.int32, device="cuda")
    if case["kind"] == "group":
        return s
    n, rank, adapters = case["n"], case["rank"], case["adapters"]
    ms = [m for m in (case["m0"], case["m1"]) if m]
    s["x"] = _bf16(_randn(gen, t, n))
    s["a"] = [_bf16(_randn(gen, adapters, rank, n) * n ** -0.5) for _ in ms]
    s["b"] = [_bf16(_randn(gen, adapters, m, rank) * 0.1) for m in ms]
    s["scales"] = 0.25 + 1.75 * torch.rand((adapters,), generator=gen, device="cuda")
    s["ranks"] = torch.tensor(_ranks(case, int(seed)), dtype=torch.int32, device="cuda")
    kind = torch.float32 if case["y32"] else torch.bfloat16
    whole = _randn(gen, t, sum(ms)).to(kind)
    s["y"] = list(whole.split(ms, dim=1)) if case["fused"] else [y.contiguous() for y in whole.split(ms, dim=1)]
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------ the plain forms

def _plain_adapters(s):
    """every row against the whole pool, the products of other adapters than the row's own set to zero"""
    c = s["case"]
    t, n, rank, adapters = c["t"], c["n"], c["rank"], c["adapters"]
    at = torch.arange(adapters, device="cuda")
    mine = s["ids"].unsqueeze(1) == at
    live = torch.arange(rank, device="cuda") < s["ranks"].unsqueeze(1)
    keep = (mine.unsqueeze(2) & live).view(t, adapters * rank)
    by = s["scales"].repeat_interleave(rank)
    any_of = mine.any(1, keepdim=True)
    x = s["x"].float()

    def one(a, b, y):
        v = x @ a.float().view(adapters * rank, n).t()
        v = torch.where(keep, v * by, torch.zeros_like(v))
        delta = v @ b.float().permute(0, 2, 1).reshape(adapters * rank, -1)
        y.copy_(torch.where(any_of, y.float() + delta, y.float()))
        return y

    return {"y": [one(*p) for p in zip(s["a"], s["b"], s["y"])]}


def _plain_group(s):
    n = s["case"]["adapters"]
    ids = s["ids"]
    key = torch.where((ids >= 0) & (ids < n), ids, torch.full_like(ids, n))
    ordered, rows = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(n + 1, dtype=torch.int32, device="cuda"))
    return {"rows": rows.to(torch.int32), "offsets": offsets.to(torch.int32)}


def _plain_norm(s):
    c = s["case"]
    h, b = s["hidden"].float(), s["delta"].float()
    if c["post"]:
        b = b * torch.rsqrt(b.square().mean(1, keepdim=True) + 1e-6) * (s["post"].float() + c["weight_bias"])
    if c["gate"] == "channel":
        b = b * s["gate"].float()
    elif c["gate"] != "none":
        b = b / (1.0 + torch.exp(-s["gate"].float()))
    s["hidden"].copy_(c["residual_scale"] * h + c["branch_scale"] * b)
    if not c["pre"]:
        return {"hidden": s["hidden"]}
    h = s["hidden"].float()
    s["out"].copy_(h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * (s["pre"].float() + c["weight_bias"]))
    return {"hidden": s["hidden"], "out": s["out"]}


# ------------------------------------------------------------------ one pass

@functools.lru_cache(maxsize=None)
def _context():
    from mference_amd import operators as ops
    return ops.MetalContext(0)


def _held(s):
    """the operators, plan and workspace that a program makes once and keeps"""
    if "held" not in s:
        from mference_amd import operators as ops
        c, ctx = s["case"], _context()
        h = {}
        if c["kind"] == "norm":
            h["norm"] = ops.BlockNorm(ctx)
            h["gate"] = dict(zip(GATES, (ops.GATE_NONE, ops.GATE_ROW, ops.GATE_ELEMENT, ops.GATE_CHANNEL)))[c["gate"]]
        else:
            h["grouping"] = ops.AdapterGrouping(ctx, c["adapters"])
            h["plan"] = h["grouping"].plan(c["t"]) if c["kind"] == "group" or c["grouped"] else None
        if c["kind"] == "adapters":
            h["adapters"] = ops.LowRankAdapters(ctx, s["a"], s["b"], scales=s["scales"], ranks=s["ranks"])
            h["workspace"] = torch.empty(h["adapters"].workspace_bytes(c["t"]), dtype=torch.uint8, device="cuda")
        s["held"] = h
    return s["held"]


def _own(s):
    c, h = s["case"], _held(s)
    if c["kind"] == "norm":
        h["norm"].encode(s["hidden"], s["delta"], out=s["out"], pre_weight=s["pre"], post_weight=s["post"], gate=s["gate"], gate_kind=h["gate"], eps=1e-6,
                         post_eps=1e-6, residual_scale=c["residual_scale"], branch_scale=c["branch_scale"], weight_bias=c["weight_bias"])
        return {"hidden": s["hidden"], "out": s["out"]} if c["pre"] else {"hidden": s["hidden"]}
    if h["plan"] is not None:
        h["grouping"].encode(s["ids"], h["plan"])
    if c["kind"] == "group":
        return {"rows": h["plan"].rows, "offsets": h["plan"].offsets}
    h["adapters"].encode(s["x"], s["ids"], s["y"], plan=h["plan"], workspace=h["workspace"])
    return {"y": s["y"]}


def run(state):
    if own:
        return _own(state)
    return {"adapters": _plain_adapters, "group": _plain_group, "norm": _plain_norm}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass needs

def work(case):
    t = case["t"]
    if case["kind"] == "group":
        return {"bytes": 8 * t + 4 * (case["adapters"] + 1), "flops": 2 * t}
    if case["kind"] == "norm":
        d = case["d"]
        element = 4 + (4 if case["delta32"] else 2) + (2 if case["pre"] else 0) + (2 if case["gate"] == "element" else 0)
        return {"bytes": t * d * element + 2 * d * (case["post"] + case["pre"]), "flops": 12 * t * d}
    ids, ranks = _ids(case, 0), _ranks(case, 0)
    rows = sum(a >= 0 for a in ids)
    n, m = case["n"], case["m0"] + case["m1"]
    targets = 2 if case["m1"] else 1
    pool = sum(ranks[a] for a in set(ids) - {-1}) * (targets * n + m) * 2
    return {"bytes": pool + 4 * t + rows * (2 * n + (8 if case["y32"] else 4) * m),
            "flops": 2 * sum(ranks[a] for a in ids if a >= 0) * (targets * n + m)}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "group":
        ids = s["ids"].tolist()
        n = case["adapters"]
        rows = sorted(range(len(ids)), key=lambda i: (ids[i] if 0 <= ids[i] < n else n, i))
        count = [0] * (n + 1)
        for a in ids:
            if 0 <= a < n:
                count[a + 1] += 1
        for a in range(n):
            count[a + 1] += count[a]
        return {"rows": torch.tensor(rows, dtype=torch.int32), "offsets": torch.tensor(count, dtype=torch.int32)}
    if case["kind"] == "norm":
        h, b, bias = s["hidden"].double(), s["delta"].double(), case["weight_bias"]
        if case["post"]:
            b = b / torch.sqrt((b * b).sum(1, keepdim=True) / case["d"] + 1e-6) * (s["post"].double() + bias)
        if case["gate"] in ("row", "element"):
            b = b * torch.sigmoid(s["gate"].double())
        elif case["gate"] == "channel":
            b = b * s["gate"].double()
        h = case["residual_scale"] * h + case["branch_scale"] * b
        if not case["pre"]:
            return {"hidden": h}
        z = h.to(torch.bfloat16).double()  # the stream is stored in 16 bits, and the norm is of what is stored
        return {"hidden": h, "out": z / torch.sqrt((z * z).sum(1, keepdim=True) / case["d"] + 1e-6) * (s["pre"].double() + bias)}
    ys = []
    for a, b, y in zip(s["a"], s["b"], s["y"]):
        y = y.double()
        for k, r in enumerate(s["ranks"].tolist()):
            at = (s["ids"] == k).nonzero()[:, 0]
            if at.numel():
                v = s["x"][at].double() @ a[k, :r].double().t()
                y[at] += s["scales"][k].double() * (v @ b[k, :, :r].double().t())
        ys.append(y)
    return {"y": ys}
