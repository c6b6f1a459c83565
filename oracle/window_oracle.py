"""Windowed attention, rotary positions and the rolling cache from their definitions, in 64 bits, on the device of
the inputs (test infrastructure).

Every result comes with `*_abs`, the sum of the absolute values of its terms, and `*_sq`, the root of the sum of their squares, from
which a test derives how far a result of 16-bit operands may be off."""
import math

import torch


def rope(x, pos, sections, theta, shared=False, interleaved=False, inverse=False):
    """x [M, heads, dim], pos [M, axes] -> turned x (64 bits)."""
    x = x.double()
    y, R, p = x.clone(), sum(sections), 0
    for a, d in enumerate(sections):
        for i in range(d // 2):
            w = theta ** (-2.0 * p / R if shared else -2.0 * i / d)
            ang = (pos[:, a].double() * w)[:, None]
            u, v = (2 * p, 2 * p + 1) if interleaved else (p, p + R // 2)
            c, s = torch.cos(ang), torch.sin(ang) * (-1.0 if inverse else 1.0)
            y[..., u], y[..., v] = x[..., u] * c - x[..., v] * s, x[..., v] * c + x[..., u] * s
            p += 1
    return y


def visible(nq, nk, left, right, sinks, device="cpu"):
    p = torch.arange(nq, device=device)[:, None] + nk - nq
    j = torch.arange(nk, device=device)[None, :]
    see = torch.ones(nq, nk, dtype=torch.bool, device=device)
    if right >= 0:
        see &= j <= p + right
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    return see


def probabilities(q, k, see, scale):
    """q [nq, D], k [nk, D] -> (P [nq, nk], lse [nq]); a row that sees nothing: zeros and -inf"""
    s = (q @ k.t() * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, 1) if s.shape[1] else torch.full((s.shape[0],), -math.inf, dtype=torch.float64, device=s.device)
    P = torch.where(see, (s - torch.where(lse > -math.inf, lse, torch.zeros_like(lse))[:, None]).exp(), torch.zeros_like(s))
    return P, lse


def attention(q, k, v, seqs, heads, kv_heads, D, left, right, sinks, scale, dout=None, out=None):
    """q [Mq, heads * D], k, v [Mk, kv_heads * D]; seqs: list of (q0, nq, k0, nk).  -> dict of out, lse and - with dout - dq, dk, dv, each
    with its `_abs`; `seen_q` / `seen_k`: rows of some sequence.  out: the 16-bit forward result that a backward pass reads (its
    distance from the exact one enters delta, see ds_abs below)."""
    q, k, v = q.double(), k.double(), v.double()
    G = heads // kv_heads
    Mq, Mk = q.shape[0], k.shape[0]
    z = lambda m, h: torch.zeros(m, h * D, dtype=torch.float64, device=q.device)
    r = {"out": z(Mq, heads), "out_abs": z(Mq, heads), "lse": torch.zeros(Mq, heads, dtype=torch.float64, device=q.device),
         "dq": z(Mq, heads), "dq_abs": z(Mq, heads), "dk": z(Mk, kv_heads), "dk_abs": z(Mk, kv_heads), "dv": z(Mk, kv_heads),
         "dv_abs": z(Mk, kv_heads), "out_sq": z(Mq, heads), "dq_sq": z(Mq, heads), "dk_sq": z(Mk, kv_heads), "dv_sq": z(Mk, kv_heads),
         "dq_off": z(Mq, heads), "dk_off": z(Mk, kv_heads),
         "seen_q": torch.zeros(Mq, dtype=torch.bool, device=q.device), "seen_k": torch.zeros(Mk, dtype=torch.bool, device=q.device)}
    for q0, nq, k0, nk in seqs:
        see = visible(nq, nk, left, right, sinks, q.device)
        r["seen_q"][q0:q0 + nq] = True
        r["seen_k"][k0:k0 + nk] = True
        for h in range(heads):
            cq, ck = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            Q, K, V = q[q0:q0 + nq, cq], k[k0:k0 + nk, ck], v[k0:k0 + nk, ck]
            P, lse = probabilities(Q, K, see, scale)
            O = P @ V
            r["out"][q0:q0 + nq, cq], r["out_abs"][q0:q0 + nq, cq] = O, P @ V.abs()
            r["out_sq"][q0:q0 + nq, cq] = (P.square() @ V.square()).sqrt()
            r["lse"][q0:q0 + nq, h] = lse
            if dout is None:
                continue
            dO = dout[q0:q0 + nq, cq].double()
            dP = dO @ V.t()
            dS = P * (dP - (dO * O).sum(1, keepdim=True))
            size = P * (dO.abs() @ V.abs().t() + (dO.abs() * (P @ V.abs())).sum(1, keepdim=True))   # the terms that cancel in dS
            # delta is formed from the rounded out: what that rounding moves
            off = P * (dO * (out[q0:q0 + nq, cq].double() - O)).sum(1, keepdim=True).abs() if out is not None else torch.zeros_like(P)
            r["dq"][q0:q0 + nq, cq], r["dq_abs"][q0:q0 + nq, cq] = scale * dS @ K, scale * dS.abs() @ K.abs()
            r["dk"][k0:k0 + nk, ck] += scale * dS.t() @ Q
            r["dk_abs"][k0:k0 + nk, ck] += scale * dS.abs().t() @ Q.abs()
            r["dv"][k0:k0 + nk, ck] += P.t() @ dO
            r["dv_abs"][k0:k0 + nk, ck] += P.t() @ dO.abs()
            r["dq_sq"][q0:q0 + nq, cq] = scale * (dS.square() @ K.square()).sqrt()
            r["dk_sq"][k0:k0 + nk, ck] += scale * (dS.square().t() @ Q.square()).sqrt()
            r["dv_sq"][k0:k0 + nk, ck] += (P.square().t() @ dO.square()).sqrt()
            # 2^-16 of the terms that cancel: sums in 32 bits, exp2 and the log-sum-exp in 32 bits
            r["dq_off"][q0:q0 + nq, cq] = scale * (off + 2.0 ** -16 * size) @ K.abs()
            r["dk_off"][k0:k0 + nk, ck] += scale * (off + 2.0 ** -16 * size).t() @ Q.abs()
    return r


def slot(t, cap, sinks, rolling):
    return t if not rolling or t < sinks else sinks + (t - sinks) % (cap - sinks)


def step(q, k_cache, v_cache, past, left, sinks, rolling, scale):
    """q [heads, D] of one sequence, caches [cap, kv_heads, D] that already hold the new token in its slot -> (out [heads, D], abs, sq)."""
    cap, kv_heads, D = k_cache.shape
    first = 0 if left < 0 else max(0, past - left)
    tokens = list(range(min(sinks, first))) + list(range(first, past + 1))
    at = torch.tensor([slot(t, cap, sinks, rolling) for t in tokens], device=q.device)
    heads = q.shape[0]
    out, size, sq = (torch.zeros(heads, D, dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(heads):
        K, V = k_cache[at, h // (heads // kv_heads)].double(), v_cache[at, h // (heads // kv_heads)].double()
        P = torch.softmax(K @ q[h].double() * scale, 0)
        out[h], size[h], sq[h] = P @ V, P @ V.abs(), (P.square() @ V.square()).sqrt()
    return out, size, sq
