"""The decoder-layer operators at the sizes they are measured at.

Three operators that a decoder stack runs around the tree attention and the LM
head of this library:

* ``norm``    add_rms_norm: h = x + residual, y = h * rsqrt(mean(h^2) + eps) * w,
              y in the input's type or in e4m3 with one scale per row
* ``linear``  y = act(x W^T + bias) + residual, or act(x G^T + gate_bias) *
              (x W^T + bias) + residual, on bf16 or on e4m3 with row scales
* ``attn``    chunk_attention: up to n new tokens per sequence over the 16-token
              paged K/V cache, each seeing the context and the chunk up to itself

``run`` computes them with elementary torch operations in fp32, or through
a11spec where ``own`` is set. ``exact`` gives the same results in fp64.
"""
import math
import os
import sys

import torch

own = False

PAGE = 16
DEV = "cuda"


def _case(op, name=None, **kw):
    c = {"op": op, **kw}
    if name is not None:
        c["name"] = name
    return c


def _norm(rows, dim, dtype="bf16", e4m3=False, add=True, **kw):
    return _case("norm", rows=rows, dim=dim, dtype=dtype, e4m3=e4m3, add=add, **kw)


def _linear(rows, k, n, dtype="bf16", gated=False, act="none", bias=False, residual=False, **kw):
    return _case("linear", rows=rows, k=k, n=n, dtype=dtype, gated=gated, act=act, bias=bias, residual=residual, **kw)


def _attn(batch, n, ctx, hq=32, hkv=4, d=128, ragged=False, lse=False, **kw):
    return _case("attn", batch=batch, n=n, ctx=ctx, hq=hq, hkv=hkv, d=d, ragged=ragged, lse=lse, **kw)


def listed():
    return [
        # the norm between two sub-layers when one sequence decodes one token: latency
        _norm(1, 2048, name="norm 1x2048"),
        # 32 sequences x 64 tree nodes, the norm that feeds an e4m3 projection
        _norm(2048, 2048, e4m3=True, name="norm 2048x2048 e4m3"),
        # a long prompt in an fp32 stack, rows of odd length (no row but the first is aligned)
        _norm(8190, 4999, dtype="fp32", name="norm 8190x4999 fp32"),
        # one decoded token through the gate and up projections
        _linear(1, 2048, 8192, gated=True, act="silu", name="gated 1x2048x8192"),
        # one token each of 32 sequences through a fused q, k, v projection (32 + 2 x 4 heads of 128) in e4m3
        _linear(32, 2048, 5120, dtype="e4m3", bias=True, name="linear 32x2048x5120 e4m3"),
        # an odd batch between the single-token and the prompt sizes: odd rows and columns, everything in the epilogue
        _linear(197, 1000, 1531, act="gelu", bias=True, residual=True, name="linear 197x1000x1531"),
        # 32 x 64 tree nodes through the down projection, added to the residual stream
        _linear(2048, 8192, 2048, residual=True, name="linear 2048x8192x2048"),
        # a prompt chunk of 8192 tokens through the gate and up projections in e4m3
        _linear(8192, 2048, 8192, dtype="e4m3", gated=True, act="silu", name="gated 8192x2048x8192 e4m3"),
        # one sequence decodes one token over a long context: work split along the cache
        _attn(1, 1, 32767, name="attn 1x1 ctx 32767"),
        # 32 sequences of different lengths decode one token each
        _attn(32, 1, 4096, ragged=True, name="attn 32x1 ctx 4096"),
        # ragged prompt chunks over ragged contexts, heads of 64 in groups of three, with the log sum of exponentials
        _attn(4, 300, 2000, hq=24, hkv=8, d=64, ragged=True, lse=True, name="attn 4x300 ctx 2000 d64"),
        # the last chunk of a 16384-token prompt
        _attn(1, 4096, 12288, name="attn 1x4096 ctx 12288"),
    ]


#: What a drawn case of an operator may cost: the largest listed one's.
_MOST = {"norm": 8190 * 4999, "linear": 8192 * 2048 * 8192 * 2, "attn": 32 * 4096 * 16384 * 128}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "attn", "attn"])
    if op == "norm":
        e4m3 = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        dim = _log(rng, 64, 8192)
        if rng.random() < 0.5:
            dim = -(-dim // 8) * 8
        rows = min(_log(rng, 1, 16384), max(1, _MOST["norm"] // dim))
        return _norm(rows, dim, dtype=dtype, e4m3=e4m3, add=rng.random() < 0.75)
    if op == "linear":
        dtype = rng.choice(["bf16", "bf16", "e4m3"])
        k = -(-_log(rng, 64, 8192) // 16) * 16
        n = _log(rng, 16, 16384)
        if rng.random() < 0.7:
            n = -(-n // 8) * 8
        gated = rng.random() < 0.4
        rows = min(_log(rng, 1, 8192), max(1, _MOST["linear"] // (k * n * (2 if gated else 1))))
        act = rng.choice(["silu", "gelu"]) if gated else rng.choice(["none", "none", "silu", "gelu"])
        return _linear(rows, k, n, dtype=dtype, gated=gated, act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8, 8])
    ctx = 0 if rng.random() < 0.1 else _log(rng, 1, 32768)
    n = 1 if rng.random() < 0.3 else _log(rng, 1, 4096)
    batch = _log(rng, 1, 32)
    batch = max(1, min(batch, _MOST["attn"] // (hq * n * (ctx + n) * d), (1 << 20) // (ctx + n)))
    n = max(1, min(n, _MOST["attn"] // (hq * (ctx + n) * d)))
    return _attn(batch, n, ctx, hq=hq, hkv=hkv, d=d, ragged=rng.random() < 0.7, lse=rng.random() < 0.5)


def _lengths(c):
    """(context, new tokens) of each sequence: a function of the case alone, so that its work is known."""
    out = []
    for b in range(c["batch"]):
        ctx, n = c["ctx"], c["n"]
        if c["ragged"]:
            ctx -= (b * 977) % (ctx // 2 + 1)
            n -= (b * 331) % (n // 2 + 1)
        out.append((ctx, n))
    return out


def _type(name):
    return {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}[name]


def _e4m3_rows(t):
    scale = t.abs().amax(dim=1) / 448.0
    return (t / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * std

    c = dict(case)
    s = {"case": c}
    if c["op"] == "norm":
        dt = _type(c["dtype"])
        rows, dim = c["rows"], c["dim"]
        s["x"] = rnd(rows, dim).to(dt)
        s["residual"] = rnd(rows, dim, std=2.0).to(dt) if c["add"] else None
        s["weight"] = (1.0 + rnd(dim, std=0.1)).to(dt)
        s["y"] = torch.empty(rows, dim, dtype=torch.float8_e4m3fn if c["e4m3"] else dt, device=DEV)
        s["scales"] = torch.empty(rows, device=DEV) if c["e4m3"] else None
        s["sum"] = torch.empty(rows, dim, dtype=dt, device=DEV) if c["add"] else None
    elif c["op"] == "linear":
        rows, k, n = c["rows"], c["k"], c["n"]
        x, w = rnd(rows, k), rnd(n, k, std=k ** -0.5)
        gate = rnd(n, k, std=k ** -0.5) if c["gated"] else None
        for name, t in (("x", x), ("weight", w), ("gate", gate)):
            if t is not None and c["dtype"] == "e4m3":
                s[name], s[name + "_scale"] = _e4m3_rows(t)
            else:
                s[name], s[name + "_scale"] = None if t is None else t.to(torch.bfloat16), None
        s["bias"] = rnd(n, std=0.1).to(torch.bfloat16) if c["bias"] else None
        s["gate_bias"] = rnd(n, std=0.1).to(torch.bfloat16) if c["bias"] and c["gated"] else None
        s["residual"] = rnd(rows, n, std=2.0).to(torch.bfloat16) if c["residual"] else None
        s["y"] = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
    else:
        lens = _lengths(c)
        batch, n, d = c["batch"], c["n"], c["d"]
        need = [(a + b + PAGE - 1) // PAGE for a, b in lens]
        s["max_kv_len"] = max(a + b for a, b in lens)
        max_pages = max(need)
        pages = sum(need) + 7
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = perm[at:at + m]
            at += m
        s["q"] = rnd(batch, n, c["hq"], d, std=1.5).to(torch.bfloat16)
        s["k_pool"] = rnd(pages, PAGE, c["hkv"], d).to(torch.bfloat16)
        s["v_pool"] = rnd(pages, PAGE, c["hkv"], d).to(torch.bfloat16)
        s["page_table"] = table
        s["ctx_lens"] = torch.tensor([a for a, _ in lens], dtype=torch.int32, device=DEV)
        s["n_new"] = torch.tensor([b for _, b in lens], dtype=torch.int32, device=DEV)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(batch, n, c["hq"], device=DEV) if c["lse"] else None
    return s


def _act(t, act):
    if act == "silu":
        return t / (1.0 + torch.exp(-t))
    if act == "gelu":
        return 0.5 * t * (1.0 + torch.erf(t * math.sqrt(0.5)))
    return t


def _plain_norm(s):
    c = s["case"]
    h = s["x"].float()
    if c["add"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * s["weight"].float()
    out = {}
    if c["e4m3"]:
        scale = (y.abs().amax(dim=1) / 448.0).clamp_min(2.0 ** -100)
        out["y"], out["scales"] = (y / scale[:, None]).to(torch.float8_e4m3fn), scale
    else:
        out["y"] = y.to(s["x"].dtype)
    if c["add"]:
        out["sum"] = h.to(s["x"].dtype)
    return out


def _plain_linear(s):
    c = s["case"]

    def values(name):
        t = s[name].float()
        return t if s[name + "_scale"] is None else t * s[name + "_scale"][:, None]

    x = values("x")
    y = x @ values("weight").t()
    if c["bias"]:
        y = y + s["bias"].float()
    if c["gated"]:
        u = x @ values("gate").t()
        if c["bias"]:
            u = u + s["gate_bias"].float()
        y = _act(u, c["act"]) * y
    else:
        y = _act(y, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


def _plain_attn(s):
    c = s["case"]
    batch, n, hq, hkv, d = c["batch"], c["n"], c["hq"], c["hkv"], c["d"]
    pages = s["page_table"].clamp_min(0).long()
    k = s["k_pool"][pages].reshape(batch, -1, hkv, d).float()
    v = s["v_pool"][pages].reshape(batch, -1, hkv, d).float()
    q = s["q"].float().view(batch, n, hkv, hq // hkv, d)
    p = torch.einsum("bnkgd,bskd->bkgns", q, k).mul_(d ** -0.5)
    i = torch.arange(n, device=DEV).view(1, n, 1)
    j = torch.arange(k.shape[1], device=DEV).view(1, 1, -1)
    seen = (j <= s["ctx_lens"].view(-1, 1, 1) + i) & (i < s["n_new"].view(-1, 1, 1))
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.einsum("bkgns,bskd->bnkgd", p, v)
    live = (total > 0).permute(0, 3, 1, 2, 4)
    o = torch.where(live, o / total.permute(0, 3, 1, 2, 4), torch.zeros_like(o))
    out = {"out": o.reshape(batch, n, hq, d).to(torch.bfloat16)}
    if c["lse"]:
        lse = torch.where(total > 0, top + torch.log(total), torch.zeros_like(total))
        out["lse"] = lse[..., 0].permute(0, 3, 1, 2).reshape(batch, n, hq)
    return out


def _a11spec():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a11-llm-optimizer_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import a11spec
    return a11spec


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "attn": _plain_attn}[c["op"]](s)
    a11spec = _a11spec()
    if c["op"] == "norm":
        y, scales, total = a11spec.add_rms_norm(s["x"], s["weight"], residual=s["residual"], eps=1e-6, out=s["y"],
                                                scales=s["scales"], sum_out=s["sum"])
        return {k: t for k, t in (("y", y), ("scales", scales), ("sum", total)) if t is not None}
    if c["op"] == "linear":
        return a11spec.linear(s["x"], s["weight"], bias=s["bias"], gate=s["gate"], gate_bias=s["gate_bias"],
                              activation=None if c["act"] == "none" else c["act"], residual=s["residual"],
                              x_scale=s["x_scale"], weight_scale=s["weight_scale"], gate_scale=s["gate_scale"],
                              out=s["y"])
    out, lse, s["ws"] = a11spec.chunk_attention(s["q"], s["k_pool"], s["v_pool"], s["page_table"], s["ctx_lens"],
                                                s["n_new"], max_kv_len=s["max_kv_len"], want_lse=c["lse"],
                                                out=s["out"], lse=s["lse"], ws=s.get("ws"))
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def work(case):
    c = case
    if c["op"] == "norm":
        e = 2 if c["dtype"] == "bf16" else 4
        values = c["rows"] * c["dim"]
        moved = values * (e + (2 * e if c["add"] else 0) + (1 if c["e4m3"] else e))
        return {"bytes": moved + c["dim"] * e + (4 * c["rows"] if c["e4m3"] else 0), "flops": 5 * values}
    if c["op"] == "linear":
        e = 1 if c["dtype"] == "e4m3" else 2
        products = 2 if c["gated"] else 1
        moved = (c["rows"] * c["k"] + products * c["n"] * c["k"]) * e
        moved += c["rows"] * c["n"] * 2 * (2 if c["residual"] else 1)
        if c["bias"]:
            moved += 2 * products * c["n"]
        if c["dtype"] == "e4m3":
            moved += 4 * (c["rows"] + products * c["n"])
        return {"bytes": moved, "flops": 2 * products * c["rows"] * c["k"] * c["n"]}
    lens = _lengths(c)
    rows = c["batch"] * c["n"] * c["hq"]
    moved = rows * c["d"] * 2 + sum(n for _, n in lens) * c["hq"] * c["d"] * 2 + (rows * 4 if c["lse"] else 0)
    moved += sum(a + n for a, n in lens) * c["hkv"] * c["d"] * 2 * 2
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in lens)
    return {"bytes": moved, "flops": 4 * c["hq"] * c["d"] * pairs}


def exact(case, seed):
    """fp64, row by row or head by head from the definitions."""
    s, c = prepare(case, seed), case
    if c["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if c["add"] else 0.0)
        rms = torch.sqrt(torch.sum(h * h, dim=1) / c["dim"] + 1e-6)
        y = h / rms[:, None] * s["weight"].double()[None]
        out = {}
        if c["e4m3"]:
            out["scales"] = torch.clamp(torch.max(torch.abs(y), dim=1).values / 448.0, min=2.0 ** -100)
            y = y / out["scales"][:, None]
        out["y"] = y
        if c["add"]:
            out["sum"] = h
        return out
    if c["op"] == "linear":
        one = torch.ones(1, device=DEV, dtype=torch.float64)

        def product(name, bias):
            sx = one if s["x_scale"] is None else s["x_scale"].double()
            sw = one if s[name + "_scale"] is None else s[name + "_scale"].double()
            t = torch.mm(s["x"].double(), s[name].double().T) * sx[:, None] * sw[None, :]
            return t if s[bias] is None else t + s[bias].double()[None, :]

        def activation(t):
            if c["act"] == "silu":
                return t * torch.special.expit(t)
            if c["act"] == "gelu":
                return t * torch.special.ndtr(t)
            return t

        y = product("weight", "bias")
        y = activation(product("gate", "gate_bias")) * y if c["gated"] else activation(y)
        return y if s["residual"] is None else y + s["residual"].double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device=DEV)
    group = c["hq"] // c["hkv"]
    for b, (ctx, n) in enumerate(_lengths(c)):
        pos = torch.arange(ctx + n, device=DEV)
        page, slot = s["page_table"][b].long()[pos // PAGE], pos % PAGE
        unseen = pos[None, :] > ctx + torch.arange(n, device=DEV)[:, None]
        for kv in range(c["hkv"]):
            keys, vals = s["k_pool"][page, slot, kv].double(), s["v_pool"][page, slot, kv].double()
            for h in range(kv * group, (kv + 1) * group):
                score = torch.mm(s["q"][b, :n, h].double(), keys.T) / math.sqrt(c["d"])
                score[unseen] = -math.inf
                lse[b, :n, h] = torch.logsumexp(score, dim=1)
                out[b, :n, h] = torch.mm(torch.exp(score - lse[b, :n, h, None]), vals)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
