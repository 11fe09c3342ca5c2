"""fp64 forms of the decoder-layer operators (K8, K9, K10) and what their
results may be off by (test helper).

Roundings count half a step, relative: u(bf16) = 2^-8, u(fp32) = 2^-24,
u(e4m3) = 2^-4 (half its smallest step, 2^-10, near zero).

norm: the sum of squares runs through at most 16 products a thread and 10
shuffle steps (all terms positive: relative error below 28 u), of which the
square root takes half; the reciprocal square root is good to 2 ulp, and three
products follow: below 32 u(fp32) = 2^-19 in all, then the output's rounding.

linear: every addition of the fp32 sum may be off by 2^-23 of the running sum
of magnitudes (tensor cores may truncate): K 2^-23 sum|x w|. The activations
have slopes below 1.13 and are good to 2^-19 of their value; then one rounding
to bf16.

attention: the scores as for linear with K = D; a relative change of a
probability by twice the largest score error; the probabilities are rounded to
bf16 before the product with V, independent errors of at most 2^-9 on average
and 2^-8 at most: 8 * 2^-9 ||p||_2 rms(v) is about ten standard deviations (as
in attn_tolerance.py); then one rounding to bf16.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def norm(x, w, residual=None, eps=1e-6):
    """(y, h) in fp64."""
    h = x.double() + (0.0 if residual is None else residual.double())
    return h / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + eps) * w.double(), h


def worst(got, ref, tol):
    """Largest |got - ref| / tol; inf where only one is finite."""
    got, ref = got.double(), ref.double()
    same = torch.isfinite(got) == torch.isfinite(ref)
    r = torch.where(torch.isfinite(ref), (got - ref).abs() / tol.clamp_min(1e-300), torch.zeros_like(ref))
    r = torch.where(same, r, torch.full_like(r, math.inf))
    return float(r.max()) if r.numel() else 0.0


def act(t, name):
    return t * torch.sigmoid(t) if name == "silu" else 0.5 * t * (1 + torch.erf(t / math.sqrt(2))) if name == "gelu" else t


def linear(x, w, bias=None, activation=None, gate=None, gate_bias=None, residual=None, sx=None, sw=None, sg=None):
    """(y, tolerance) in fp64; the scales are folded into the operands."""
    def product(m, s, b):
        xd = x.double() if sx is None else x.double() * sx.double()[:, None]
        md = m.double() if s is None else m.double() * s.double()[:, None]
        t = xd @ md.T
        off = x.shape[1] * 2.0 ** -23 * (xd.abs() @ md.abs().T) + 2.0 ** -22 * t.abs()
        return (t, off) if b is None else (t + b.double(), off + 2.0 ** -23 * (t.abs() + b.double().abs()))

    v, dv = product(w, sw, bias)
    if gate is None:
        y, dy = act(v, activation), (1.13 if activation else 1.0) * dv
        dy = dy + 2.0 ** -19 * y.abs()
    else:
        u, du = product(gate, sg, gate_bias)
        a = act(u, activation)
        y = a * v
        dy = (1.13 * du + 2.0 ** -19 * a.abs()) * (v.abs() + dv) + a.abs() * dv + 2.0 ** -23 * y.abs()
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy + (y.abs() + dy) * 2.0 ** -8 + 2.0 ** -134


def attention(q, k_pool, v_pool, page_table, ctx, n_new, scale=None):
    """(out, its tolerance, lse, its tolerance) in fp64; rows without work are zero."""
    B, N, Hq, D = q.shape
    Hkv = k_pool.shape[2]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, 1e-300)
    lse = torch.zeros(B, N, Hq, dtype=torch.float64, device=q.device)
    ltol = torch.full_like(lse, 1e-300)
    for b in range(B):
        c, n = int(ctx[b]), int(n_new[b])
        if n == 0:
            continue
        pos = torch.arange(c + n, device=q.device)
        page = page_table[b].long()[pos // 16]
        k, v = k_pool[page, pos % 16].double(), v_pool[page, pos % 16].double()  # [S, Hkv, D]
        seen = pos[None] <= c + torch.arange(n, device=q.device)[:, None]
        for h in range(Hkv):
            qh = q[b, :n, h * G:(h + 1) * G].double().permute(1, 0, 2)  # [G, n, D]
            s = (qh @ k[:, h].T * scale).masked_fill(~seen, -math.inf)
            mag = (qh.abs() @ k[:, h].abs().T * scale).masked_fill(~seen, 0).amax(-1)  # [G, n]
            ds = D * 2.0 ** -23 * mag + 2.0 ** -20 * (1 + s.amax(-1).abs())
            p = torch.softmax(s, dim=-1)
            o = p @ v[:, h]
            floor = 8 * 2.0 ** -9 * p.square().sum(-1).sqrt() * v[:, h].square().mean().sqrt()
            small = (2 * ds + (c + n) * 2.0 ** -23)[..., None] * (p @ v[:, h].abs())
            out[b, :n, h * G:(h + 1) * G] = o.permute(1, 0, 2)
            tol[b, :n, h * G:(h + 1) * G] = (floor[..., None] + small + 2.0 ** -8 * o.abs()).permute(1, 0, 2)
            lse[b, :n, h * G:(h + 1) * G] = torch.logsumexp(s, dim=-1).T
            ltol[b, :n, h * G:(h + 1) * G] = (2 * ds + 2.0 ** -20 * (1 + torch.logsumexp(s, dim=-1).abs())).T
    return out, tol, lse, ltol
