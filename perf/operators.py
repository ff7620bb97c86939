"""The work of the operators around the quantized projections whose speed is measured.

Three operators of a decoder layer, which follow one another there:

  norm      `ops.add_rms_norm`: v = x + residual in fp32, h = v, u = v * rsqrt(mean(v^2) + eps) * weight, leaving as bf16,
            as mxfp8 rows (e4m3 codes, one power of two for 32 values), or as both
  product   `ops.mxfp8_matmul`: rows in mxfp8 times a weight [out, in] in mxfp8, bf16 out
  adapters  `ops.low_rank_add`: y[t] + scale_a * (x[t] A_a^T) B_a^T for the low-rank adapter a = ids[t] of each row

Where `own` is false, `run` computes them in their plain form, from elementary torch operations in fp32.
Hidden sizes and projections are those of `perf/cases.py` (hidden 2048; 2048 -> 8192, 4096 -> 2048, 2048 -> 512, and the
vocabulary head 2048 -> 152064).
"""
from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-6


def _norm(name, rows, hidden, out, residual=True):
    return dict(name=name, op="norm", rows=rows, hidden=hidden, out=out, residual=residual)


def _product(name, rows, n_in, n_out):
    return dict(name=name, op="product", rows=rows, n_in=n_in, n_out=n_out)


def _adapters(name, tokens, requests, adapters, rank, n_in, n_out, pad=0):
    return dict(name=name, op="adapters", tokens=tokens, requests=requests, adapters=adapters, rank=rank, n_in=n_in,
                n_out=n_out, pad=pad)


def listed():
    return [
        # one user's decode step: the rows of the next projection in 8 bits; latency alone
        _norm("norm-1", 1, 2048, "mxfp8"),
        # a decode batch whose projections carry adapters (they read the bf16 rows)
        _norm("norm-64-both", 64, 2048, "both"),
        # a ragged prompt, no residual (the first layer), a wider hidden size that is no power of two
        _norm("norm-777-first", 777, 5120, "bf16", residual=False),
        # a long prompt
        _norm("norm-8192-both", 8192, 2048, "both"),
        # decode of one user through an attention projection
        _product("product-1", 1, 2048, 8192),
        # the vocabulary head of a decode batch: the weights' bytes count
        _product("product-64-head", 64, 2048, 152064),
        # an output projection of a ragged prompt
        _product("product-777", 777, 4096, 2048),
        # a long prompt: the tensor cores' rate counts
        _product("product-8192", 8192, 2048, 8192),
        # one user with an adapter: latency alone
        _adapters("adapters-1", 1, 1, 1, 16, 2048, 8192),
        # a decode batch in which nearly every user has an adapter, some rows of the batch have none
        _adapters("adapters-48", 48, 42, 40, 32, 4096, 2048, pad=6),
        # prompts of a few users packed one after another, the batch padded
        _adapters("adapters-777", 777, 6, 5, 16, 2048, 8192, pad=33),
        # long prompts, larger rank
        _adapters("adapters-8192", 8192, 14, 12, 64, 2048, 8192),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    op = rng.choice(["norm", "product", "adapters"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "norm":
            case = _norm("", _log_uniform(rng, 1, 16384), 32 * _log_uniform(rng, 4, 512),
                         rng.choice(["bf16", "mxfp8", "both"]), rng.random() < 0.8)
        elif op == "product":
            n_in = 32 * _log_uniform(rng, 4, 256) if rng.random() < 0.5 else 512 * rng.randint(1, 12)
            n_out = _log_uniform(rng, 64, 40000)
            case = _product("", _log_uniform(rng, 1, 12000), n_in, n_out if rng.random() < 0.3 else (n_out + 7) // 8 * 8)
        else:
            tokens = _log_uniform(rng, 1, 8192)
            pad = int(tokens * rng.random() * 0.2) if rng.random() < 0.5 else 0
            requests = tokens - pad if tokens <= 128 and rng.random() < 0.7 else rng.randint(1, min(64, tokens - pad))
            n_out = _log_uniform(rng, 256, 12000)
            case = _adapters("", tokens, requests, rng.randint(1, min(64, requests)), rng.choice([8, 16, 16, 24, 32, 64, 128]),
                             8 * _log_uniform(rng, 32, 1024), n_out if rng.random() < 0.2 else (n_out + 7) // 8 * 8, pad)
        if _cost(case) <= most:
            del case["name"]
            return case


# ── inputs ──────────────────────────────────────────────────────────────────
def _to_mxfp8(v):
    """fp32 [rows, n] -> (e4m3 codes as int32 words [rows, n / 4], powers of two as uint8 [rows, n / 32])."""
    g = v.view(v.shape[0], -1, 32)
    mantissa, e = torch.frexp(g.abs().amax(-1) / 448)
    e = torch.where(mantissa == 0.5, e - 1, e).clamp(-127, 127)
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e)
    # 2^-e as two factors: 2^127 fits fp32, 2^-127 only as a subnormal
    half = torch.div(-e, 2, rounding_mode="floor")
    up = ((half + 127) << 23).view(torch.float32).unsqueeze(-1), ((-e - half + 127) << 23).view(torch.float32).unsqueeze(-1)
    q = (g * up[0] * up[1]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(v.shape[0], -1).view(torch.int32), (e + 127).to(torch.uint8)


def _activations(gen, rows, n):
    """Values as they enter a layer: unit variance, a few channels far larger."""
    x = torch.randn(rows, n, generator=gen, device="cuda")
    big = torch.rand(n, generator=gen, device="cuda") < 0.01
    return x * torch.where(big, 8.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "norm":
        n, h = case["rows"], case["hidden"]
        return {"op": "norm", "out": case["out"], "x": (_activations(gen, n, h) * 0.5).bfloat16(),
                "residual": (_activations(gen, n, h) * 2).bfloat16() if case["residual"] else None,
                "weight": (torch.randn(h, generator=gen, device="cuda") * 0.1 + 1).bfloat16()}
    if case["op"] == "product":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        rows = _to_mxfp8(_activations(gen, m, k))
        # the weight in parts: what quantizes it needs room
        parts = [_to_mxfp8(torch.randn(min(32768, n - i), k, generator=gen, device="cuda") * 0.02) for i in range(0, n, 32768)]
        return {"op": "product", "rows": rows, "w": torch.cat([p[0] for p in parts]), "scales": torch.cat([p[1] for p in parts])}
    t, k, n, r, a = case["tokens"], case["n_in"], case["n_out"], case["rank"], case["adapters"]
    # requests follow one another in the batch, each with one adapter; rows at the end have none
    active = t - case["pad"]
    cuts = torch.randperm(active - 1, generator=gen, device="cuda")[: case["requests"] - 1] + 1
    starts = torch.zeros(t, dtype=torch.int64, device="cuda")
    starts[cuts] = 1
    of_request = torch.randperm(a, generator=gen, device="cuda")[torch.arange(case["requests"], device="cuda") % a]
    ids = of_request[torch.cumsum(starts, 0)].int()
    ids[active:] = -1
    return {"op": "adapters", "ids": ids,
            "x": _activations(gen, t, k).bfloat16(), "y": torch.randn(t, n, generator=gen, device="cuda").bfloat16(),
            "a": (torch.randn(a, r, k, generator=gen, device="cuda") / math.sqrt(k)).bfloat16(),
            "b": (torch.randn(a, n, r, generator=gen, device="cuda") * 0.1).bfloat16(),
            "scale": torch.rand(a, generator=gen, device="cuda") * 1.5 + 0.5}


# ── the operators in their plain form ───────────────────────────────────────
def _from_mxfp8(words, scales):
    s = scales.int()
    factor = torch.where(s == 0, torch.full_like(s, 0x00400000), s << 23).view(torch.float32)
    q = words.view(torch.float8_e4m3fn).float()
    return (q.view(q.shape[0], -1, 32) * factor.unsqueeze(-1)).view(q.shape)


def _plain_norm(state):
    v = state["x"].float()
    if state["residual"] is not None:
        v = v + state["residual"].float()
    u = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * state["weight"].float()
    rows = _to_mxfp8(u) if state["out"] != "bf16" else None
    return (state["x"] if state["residual"] is None else v.bfloat16(), u.bfloat16() if state["out"] != "mxfp8" else None, rows)


def _plain_product(state):
    return (_from_mxfp8(*state["rows"]) @ _from_mxfp8(state["w"], state["scales"]).T).bfloat16()


def _plain_adapters(state):
    a, b, ids, scale = state["a"], state["b"], state["ids"], state["scale"]
    # every adapter's product with every row, those of other rows' adapters taken out
    t = (state["x"].float() @ a.float().flatten(0, 1).T).view(-1, a.shape[0], a.shape[1])
    t = t * torch.where(ids[:, None] == torch.arange(a.shape[0], device=ids.device), scale, 0.0).unsqueeze(-1)
    return (state["y"].float() + t.flatten(1) @ b.float().transpose(1, 2).flatten(0, 1)).bfloat16()


def run(state):
    if own:
        from ironmlx_b200 import ops
    if state["op"] == "norm":
        if own:
            h, y, rows = ops.add_rms_norm(state["x"], state["residual"], state["weight"], _EPS, out=state["out"])
        else:
            h, y, rows = _plain_norm(state)
        # the codes as e4m3 numbers, the scales as powers of two
        return {"h": h, "y": y, "codes": None if rows is None else rows[0].view(torch.float8_e4m3fn),
                "scales": None if rows is None else rows[1].view(torch.float8_e8m0fnu)}
    if state["op"] == "product":
        return ops.mxfp8_matmul(state["rows"], state["w"], state["scales"]) if own else _plain_product(state)
    if own:
        return ops.low_rank_add(state["y"], state["x"], state["a"], state["b"], state["ids"], state["scale"])
    return _plain_adapters(state)


# ── the same from the definitions, in 64 bits ───────────────────────────────
def _e4m3_values(codes):
    """The numbers of e4m3 codes: sign, four bits of exponent (bias 7), three of mantissa."""
    c = torch.arange(256, device=codes.device)
    e, m, sign = (c >> 3) & 15, (c & 7).double(), 1.0 - 2.0 * (c >> 7)
    table = sign * torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2((e - 7).double()))
    return table[codes.long()]


def _exact_values(words, scales):
    q = _e4m3_values(words.contiguous().view(torch.uint8))
    return (q.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def _to_e4m3_grid(v):
    """The nearest e4m3 number to each value of at most 448, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        v = s["x"].double() + (0 if s["residual"] is None else s["residual"].double())
        u = v / torch.sqrt((v ** 2).sum(-1, keepdim=True) / case["hidden"] + _EPS) * s["weight"].double()
        codes = scales = None
        if case["out"] != "bf16":
            g = u.unflatten(-1, (-1, 32))
            scales = torch.exp2(torch.ceil(torch.log2(g.abs().amax(-1) / 448)).clamp(-127, 127))
            codes = _to_e4m3_grid(g / scales[..., None]).flatten(-2)
        return {"h": v, "y": u if case["out"] != "mxfp8" else None, "codes": codes, "scales": scales}
    if case["op"] == "product":
        return torch.einsum("mk,nk->mn", _exact_values(*s["rows"]), _exact_values(s["w"], s["scales"]))
    y, x = s["y"].double(), s["x"].double()
    for j in range(case["adapters"]):
        at = torch.nonzero(s["ids"] == j).flatten()
        low = torch.einsum("tk,rk->tr", x[at], s["a"][j].double())
        y[at] += s["scale"][j].double() * torch.einsum("tr,nr->tn", low, s["b"][j].double())
    return y


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    if case["op"] == "norm":
        n, h = case["rows"], case["hidden"]
        a_value = 2 + (4 if case["residual"] else 0) + {"bf16": 2, "mxfp8": 1 + 1 / 32, "both": 3 + 1 / 32}[case["out"]]
        return {"bytes": n * h * a_value + 2 * h, "flops": 8 * n * h}
    if case["op"] == "product":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        return {"bytes": (m + n) * k * (1 + 1 / 32) + 2 * m * n, "flops": 2 * m * k * n}
    t, k, n, r = case["tokens"], case["n_in"], case["n_out"], case["rank"]
    active = t - case["pad"]
    return {"bytes": 2 * active * k + 4 * t * n + 2 * min(case["adapters"], case["requests"]) * r * (k + n) + 4 * t,
            "flops": 2 * active * r * (k + n)}
