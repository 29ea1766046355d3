"""What matrix products in 8 bits are timed on: rows brought to 8 bits (e4m3) with a scale each, out of the residual stream through
its norm or as they are, and products of such rows with 8-bit weights, dense and grouped by expert.

A case is one operator at one size.  `run` makes one pass through it: with `own` the calls a program makes of
`lastengine_b200.ops.kernels`, without it the same numbers from elementary torch operations in 32 bits.

The formulas, a row of 8-bit numbers q with its scale s standing for s q:
  quantize   a = max(max |x|, 2^-100), q = round(448 x / a), s = a / 448; rows may be gathered (row p is x[rows[p] // div]) and
             weighted (s times weights[rows[p]])
  norm       x += y, g = x w, r = 1 / sqrt(mean(x^2) + eps), a = max(max |g|, 2^-100), q = round(448 g / a), s = r a / 448; h = r g
  linear     z = (sum_k x[m, k] w[n, k]) sx[m] sw[n], stored, added into out, or gated: columns in blocks of 16 gate and 16 up
             values, out = silu(gate) up
  grouped    the same, rows [offsets[e], offsets[e + 1]) with expert e's weights; rows behind the last offset stay as they are
"""
from __future__ import annotations

import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "": None}
E4M3, TOP, LEAST = torch.float8_e4m3fn, 448.0, 2.0 ** -100


# ---- the cases -------------------------------------------------------------------------------------------------------
def _norm(name, rows=1, dim=2048, y="f32", h=""):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "y": y, "h": h}


def _quantize(name, rows=1, dim=2048, type="bf16", times=0, weighted=False):
    return {"name": name, "op": "quantize", "rows": rows, "dim": dim, "type": type, "times": times, "weighted": weighted}


def _linear(name, rows=1, n=2048, k=2048, out="bf16", epilogue="store"):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "out": out, "epilogue": epilogue}


def _grouped(name, rows=4, experts=32, n=2048, k=2048, out="bf16", epilogue="store", skew=1.0, behind=0):
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "n": n, "k": k, "out": out, "epilogue": epilogue,
            "skew": skew, "behind": behind}


def listed():
    return [
        # a decode step of one sequence: every call's fixed cost counts
        _norm("norm, one row", y="bf16"),
        # a batch's decode step in front of experts, whose router reads the normed rows; a width that no vector divides
        _norm("norm, 61 rows of 1999", rows=61, dim=1999, h="bf16"),
        # a prompt's rows, the sublayer's result added on the way
        _norm("norm, prompt", rows=16000),
        # the rows of a decode step's experts, gathered in the experts' order
        _quantize("rows of experts, 64 tokens", rows=64, times=4),
        # what a wide feed-forward hands its last product
        _quantize("feed-forward rows, prompt", rows=8191, dim=8192),
        # a decode step of one sequence, the feed-forward's first product
        _linear("gate and up, one token", n=16384, epilogue="gated"),
        # a serving batch, the feed-forward's last product into the residual stream
        _linear("down, 61 tokens", rows=61, k=8192, out="f32", epilogue="add"),
        # logits of a batch
        _linear("head, 17 rows", rows=17, n=65536, out="f32"),
        # a chunk of a prompt, sizes that no tile divides (rows lie 16 bytes apart or a multiple of that)
        _linear("777 rows of 1001", rows=777, n=1000, k=1001),
        # a prompt through a wide feed-forward
        _linear("gate and up, prompt", rows=8191, n=21504, epilogue="gated"),
        # a decode step's experts
        _grouped("experts, 64 tokens", rows=256, n=3584, epilogue="gated", behind=4),
        # a prompt's experts, the products that are then weighed and added
        _grouped("experts, prompt", rows=32768, k=1792, out="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A width, as a rule a multiple of 64 or 16, at times any."""
    step = rng.choice([64, 64, 16, 1])
    return min(hi, max(1, round(_log_int(rng, lo, hi) / step)) * step)


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "quantize", "linear", "linear", "linear", "grouped", "grouped"])
    if op in ("norm", "quantize"):
        dim = _width(rng, 64, 12000)
        rows = _log_int(rng, 1, max(1, min(16000, 30_000_000 // dim)))
        if op == "norm":
            c = _norm("", rows=rows, dim=dim, y=rng.choice(["f32", "bf16", ""]), h=rng.choice(["", "", "bf16", "f32"]))
        else:
            times = rng.choice([0, 0, 1, 2, 4, 8])
            c = _quantize("", rows=max(1, rows // max(1, times)), dim=dim, type=rng.choice(["bf16", "bf16", "f32"]), times=times,
                          weighted=times > 0 and rng.random() < 0.4)
    else:
        k = _width(rng, 64, 12000)
        epilogue = rng.choice(["store", "add", "gated"])
        out = "f32" if epilogue == "add" else rng.choice(["bf16", "bf16", "f32"])
        n = _width(rng, 32, 24000)
        if op == "linear":
            rows = _log_int(rng, 1, max(1, min(16000, 150_000_000 // n, 300_000_000_000 // (n * k))))
        else:
            experts = _log_int(rng, 2, 128)
            n = min(n, 6000)
            k = min(k, max(64, 400_000_000 // (experts * n)))
            rows = _log_int(rng, 1, max(1, min(32768, 60_000_000 // n, 100_000_000_000 // (n * k))))
        if epilogue == "gated":
            n = max(32, n // 32 * 32)
        if op == "linear":
            c = _linear("", rows=rows, n=n, k=k, out=out, epilogue=epilogue)
        else:
            c = _grouped("", rows=rows, experts=experts, n=n, k=k, out=out, epilogue=epilogue, skew=rng.choice([0.0, 1.0, 3.0]),
                         behind=rng.choice([0, 0, 3]))
    del c["name"]
    return c


def _counts(case):
    """Rows of every expert: popular ones first and last, with a skew of 0 as many for all."""
    E, P = case["experts"], case["rows"]
    v = [math.exp(case["skew"] * math.cos(2.4 * e)) for e in range(E)]
    edges = [int(round(P * sum(v[:e]) / sum(v))) for e in range(E + 1)]
    return [b - a for a, b in zip(edges, edges[1:])]


def work(case):
    size = {"bf16": 2, "f32": 4, "": 0}
    if case["op"] == "norm":
        M, D = case["rows"], case["dim"]
        y, h = size[case["y"]], size[case["h"]]
        return {"bytes": M * D * (4 + (y + 4 if y else 0) + h + 1) + 4 * D + 4 * M, "flops": 0}
    if case["op"] == "quantize":
        M, D, P = case["rows"], case["dim"], case["rows"] * max(1, case["times"])
        return {"bytes": M * D * size[case["type"]] + P * (D + 4 + (4 if case["times"] else 0)), "flops": 0}
    M, N, K = case["rows"], case["n"], case["k"]
    n_out = N // 2 if case["epilogue"] == "gated" else N
    E = sum(c > 0 for c in _counts(case)) if case["op"] == "grouped" else 1
    out = M * n_out * size[case["out"]] * (2 if case["epilogue"] == "add" else 1)
    return {"bytes": M * K + E * N * K + out + 4 * M + 4 * E * N, "flops": 2 * M * N * K}


# ---- what a program has in hand --------------------------------------------------------------------------------------
def _pitch(k):
    return -(-k // 16) * 16


def _eight(rows, k):
    """Room for rows of 8-bit numbers, 16 bytes apart or a multiple of that."""
    return torch.zeros((*rows, _pitch(k)), dtype=torch.uint8, device="cuda").view(E4M3)[..., :k]


def _to_eight(x):
    """x in 8 bits and the scales of its rows, as a program holds them."""
    a = x.abs().amax(-1).clamp_(min=LEAST)
    q = _eight(x.shape[:-1], x.shape[-1])
    q.copy_((x * (TOP / a)[..., None]).to(E4M3))
    return q, a / TOP


def _activations(gen, rows, dim):
    """Rows as models have them: a few channels far wider than the others, rows of different sizes."""
    wide = 1 + 15 * (torch.rand(dim, generator=gen, device="cuda") < 0.005).float()
    size = torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    return torch.randn((rows, dim), generator=gen, device="cuda").mul_(wide).mul_(size)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = types.SimpleNamespace(case=case)
    if case["op"] == "norm":
        M, D = case["rows"], case["dim"]
        s.x = _activations(gen, M, D)
        s.w = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
        s.y = torch.randn((M, D), generator=gen, device="cuda").to(TYPES[case["y"]]) if case["y"] else None
        s.h = torch.zeros((M, D), dtype=TYPES[case["h"]], device="cuda") if case["h"] else None
        s.q, s.scale = _eight((M,), D), torch.zeros(M, device="cuda")
        return s
    if case["op"] == "quantize":
        M, D, k = case["rows"], case["dim"], case["times"]
        s.x = _activations(gen, M, D).to(TYPES[case["type"]])
        s.rows = torch.randperm(M * k, generator=gen, device="cuda").to(torch.int32) if k else None
        s.weights = torch.rand(M * k, generator=gen, device="cuda") if case["weighted"] else None
        s.q, s.scale = _eight((M * max(1, k),), D), torch.zeros(M * max(1, k), device="cuda")
        return s
    M, N, K = case["rows"], case["n"], case["k"]
    grouped = case["op"] == "grouped"
    behind = case["behind"] if grouped else 0
    s.x, s.x_scale = _to_eight(_activations(gen, M + behind, K))
    shape = (case["experts"], N, K) if grouped else (N, K)
    s.w, s.w_scale = _to_eight(torch.randn(shape, generator=gen, device="cuda").mul_(K ** -0.5))
    s.offsets = None
    if grouped:
        counts = _counts(case)
        s.most = max(counts)
        s.offsets = torch.tensor([sum(counts[:e]) for e in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    n_out = N // 2 if case["epilogue"] == "gated" else N
    s.out = torch.randn((M + behind, n_out), generator=gen, device="cuda").to(TYPES[case["out"]])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def _own_pass(s):
    from lastengine_b200.ops import kernels
    c = s.case
    if c["op"] == "norm":
        kernels.rmsnorm_e4m3(s.q, s.scale, s.x, s.w, 1e-5, y=s.y, h=s.h)
    elif c["op"] == "quantize":
        kernels.quantize_e4m3(s.q, s.scale, s.x, rows=s.rows, div=max(1, c["times"]), weights=s.weights)
    else:
        epilogue = {"store": kernels.STORE, "add": kernels.ACCUMULATE, "gated": kernels.gated_epilogue(kernels.SILU)}[c["epilogue"]]
        kernels.linear_e4m3(s.out, s.x, s.x_scale, s.w, s.w_scale, epilogue, group_offsets=s.offsets)


def _plain_norm(s):
    if s.y is not None:
        s.x.add_(s.y)
    r = torch.rsqrt(s.x.square().mean(-1) + 1e-5)
    g = s.x * s.w
    a = g.abs().amax(-1).clamp_(min=LEAST)
    if s.h is not None:
        s.h.copy_(g * r[:, None])
    s.q.copy_(g * (TOP / a)[:, None])
    torch.mul(a, r / TOP, out=s.scale)


def _plain_quantize(s):
    at = s.rows.long() // max(1, s.case["times"]) if s.rows is not None else None
    x = s.x.float() if at is None else s.x[at].float()
    a = x.abs().amax(-1).clamp_(min=LEAST)
    s.q.copy_(x * (TOP / a)[:, None])
    scale = a / TOP
    s.scale.copy_(scale if s.weights is None else scale * s.weights[s.rows.long()])


def _plain_products(s):
    c = s.case
    x, w = s.x.float(), s.w.float()
    if s.offsets is None:
        z = torch.matmul(x, w.t()) * s.x_scale[:, None] * s.w_scale
    else:
        # every expert's rows in a block of the largest one's size, and back
        first = s.offsets[:-1].long()
        rows = (first[:, None] + torch.arange(s.most, device="cuda")).clamp_(max=x.shape[0] - 1)
        z = torch.bmm(x[rows], w.transpose(1, 2)) * s.x_scale[rows][..., None] * s.w_scale[:, None]
        r = torch.arange(x.shape[0], device="cuda")
        e = torch.searchsorted(s.offsets[1:].long(), r, right=True).clamp_(max=c["experts"] - 1)
        z = z[e, (r - first[e]).clamp_(max=s.most - 1)]
    if c["epilogue"] == "gated":
        z = z.view(z.shape[0], -1, 2, 16)
        gate = z[:, :, 0]
        z = (gate / (1 + torch.exp(-gate)) * z[:, :, 1]).reshape(z.shape[0], -1)
    elif c["epilogue"] == "add":
        z = z + s.out
    s.out.copy_(z if s.offsets is None else torch.where((r < s.offsets[-1])[:, None], z, s.out.float()))


def run(state):
    s = state
    if own:
        _own_pass(s)
    else:
        {"norm": _plain_norm, "quantize": _plain_quantize, "linear": _plain_products, "grouped": _plain_products}[s.case["op"]](s)
    if s.case["op"] == "norm":
        return {"q": s.q, "scale": s.scale, "x": s.x, **({} if s.h is None else {"h": s.h})}
    return {"q": s.q, "scale": s.scale} if s.case["op"] == "quantize" else s.out


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    """8-bit numbers before their rounding."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s.x.double() + (0 if s.y is None else s.y.double())
        root = torch.sqrt((x * x).sum(1, keepdim=True) / case["dim"] + 1e-5)
        h = x / root * s.w.double()
        scale = h.abs().max(1, keepdim=True).values / 448
        return {"q": h / scale, "scale": scale[:, 0], "x": x, **({} if s.h is None else {"h": h})}
    if case["op"] == "quantize":
        x = s.x.double()
        if s.rows is not None:
            x = x[torch.div(s.rows, case["times"], rounding_mode="floor").long()]
        scale = x.abs().max(1, keepdim=True).values / 448
        q = x / scale
        return {"q": q, "scale": scale[:, 0] if s.weights is None else scale[:, 0] * s.weights.double()[s.rows.long()]}
    out = s.out.double()
    counts = _counts(case) if case["op"] == "grouped" else [case["rows"]]
    row = 0
    for e, m in enumerate(counts):
        for lo in range(row, row + m, 4096):
            hi = min(row + m, lo + 4096)
            w, sw = (s.w[e], s.w_scale[e]) if case["op"] == "grouped" else (s.w, s.w_scale)
            z = (s.x[lo:hi].double() * s.x_scale[lo:hi, None].double()) @ (w.double() * sw[:, None].double()).t()
            if case["epilogue"] == "gated":
                at = torch.arange(out.shape[1], device="cuda")
                gate = at // 16 * 32 + at % 16
                z = z[:, gate] * torch.sigmoid(z[:, gate]) * z[:, gate + 16]
            out[lo:hi] = z + out[lo:hi] if case["epilogue"] == "add" else z
        row += m
    return out
