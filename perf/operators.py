"""Cases, plain forms and 64-bit definitions of the windowed-attention operators (rotary positions over several axes, attention
over a sliding window with sinks, and its one-token form over a key / value cache).

`own` chooses what `run` calls: the framework's kernels (True) or the plain torch form (False)."""
import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of eight captions: one axis, latency
        dict(name="rope_8_tokens", op="rope", B=1, L=8, heads=12, kv=12, dim=64, sections="64", shared=False, inter=False,
             inverse=False, dtype="bf16", theta=10000.0),
        # queries and keys of a batch of 32 clips: 8 frames of 14 x 14 patches and the class token (the headline workload's rows)
        dict(name="rope_32_clips_8f", op="rope", B=32, L=1569, heads=12, kv=12, dim=64, sections="16,24,24", shared=False,
             inter=False, inverse=False, dtype="bf16", theta=10000.0),
        # the gradient's way back for four clips of 16 frames of 21 x 21 patches, kept in 32 bits, neighbouring pairs
        dict(name="rope_back_4_clips_16f", op="rope", B=4, L=7057, heads=12, kv=12, dim=64, sections="16,24,24", shared=True,
             inter=True, inverse=True, dtype="fp32", theta=100.0),
        # eight short captions read once and left in a cache (causal, everything visible)
        dict(name="prompt_8_captions", op="prompt", B=8, L=77, heads=12, kv=12, dim=64, left=-1, sinks=0, sections="64", shared=False,
             dtype="fp16", theta=10000.0),
        # a long prompt with shared key heads: a window of 1024 and four sinks, a cache that holds just these
        dict(name="prompt_8191", op="prompt", B=1, L=8191, heads=32, kv=8, dim=128, left=1023, sinks=4, sections="128", shared=False,
             dtype="bf16", theta=500000.0),
        # eight clips without a gradient: two frames to each side and the class token
        dict(name="clips_8f", op="attend", B=8, L=1569, heads=12, kv=12, dim=64, left=392, right=392, sinks=1, dtype="bf16"),
        # a training step's attention over ragged captions, both directions visible
        dict(name="train_captions", op="train", B=32, L=512, heads=12, kv=12, dim=64, left=-1, right=-1, sinks=0, sections="64",
             shared=False, dtype="bf16", theta=10000.0),
        # two clips of 16 frames of 21 x 21 patches: two frames to each side, the class token, positions of time, height and width
        dict(name="train_clips_16f", op="train", B=2, L=7057, heads=12, kv=12, dim=64, left=882, right=882, sinks=1,
             sections="16,24,24", shared=False, dtype="bf16", theta=10000.0),
        # causal training on packed texts of many lengths with shared key heads
        dict(name="train_shared_heads", op="train", B=6, L=2048, heads=16, kv=4, dim=128, left=511, right=0, sinks=4, sections="128",
             shared=False, dtype="fp16", theta=10000.0),
        # one caption being written: a rolling cache of 512 rows
        dict(name="step_1_rolling", op="step", B=1, cap=512, heads=12, kv=12, dim=64, left=507, sinks=4, rolling=True, past=700, spread=0,
             sections="64", shared=False, dtype="bf16", theta=10000.0),
        # 64 answers being written, each of its own length up to 4096
        dict(name="step_64", op="step", B=64, cap=4096, heads=32, kv=8, dim=128, left=-1, sinks=0, rolling=False, past=4095, spread=4095,
             sections="128", shared=False, dtype="bf16", theta=500000.0),
        # two very long videos being followed: 64 k visible tokens of 128 k, positions of time, height and width
        dict(name="step_2_long", op="step", B=2, cap=131072, heads=32, kv=8, dim=128, left=65535, sinks=4, rolling=False, past=131071,
             spread=100, sections="32,48,48", shared=True, dtype="fp16", theta=500000.0),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "attend", "train", "step"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv * rng.choice([1, 1, 2, 4, 5, 8])
    sections = rng.choice(["64", "16,24,24", "32,32", "48"] if dim == 64 else ["128", "32,48,48", "64,64", "64"])
    c = dict(op=op, heads=heads, kv=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]), sections=sections,
             shared=rng.choice([False, True]), theta=rng.choice([100.0, 10000.0, 500000.0]))
    if op == "rope":
        c.update(B=_spread(rng, 1, 48), L=_spread(rng, 1, 8000), inter=rng.choice([False, True]), inverse=rng.choice([False, True]),
                 dtype=rng.choice(["bf16", "fp16", "fp32"]))
        while c["B"] * c["L"] * (heads + kv) * dim > 120_000_000:
            c["B"], c["L"] = (c["B"] + 1) // 2, (c["L"] + 1) // 2
        return c
    if op == "step":
        c.update(B=_spread(rng, 1, 64), cap=_spread(rng, 16, 131072), rolling=rng.choice([False, True]), sinks=rng.choice([0, 1, 4, 16]))
        while c["B"] * c["cap"] * kv * dim > 300_000_000:
            c["cap"] = (c["cap"] + 1) // 2
        c["sinks"] = min(c["sinks"], c["cap"] // 2)
        if c["rolling"]:
            c["left"], c["past"] = c["cap"] - c["sinks"] - 1, _spread(rng, 1, 4 * c["cap"])
        else:
            c["left"], c["past"] = rng.choice([-1, _spread(rng, 1, c["cap"])]), rng.randint(0, c["cap"] - 1)
        c["spread"] = rng.randint(0, c["past"])
        return c
    c.update(B=_spread(rng, 1, 32), L=_spread(rng, 1, 8000), sinks=rng.choice([0, 0, 1, 4, 33]))
    top = 800_000_000 if op == "train" else 1_600_000_000
    while c["B"] * heads * c["L"] * c["L"] > top:
        if c["B"] > 1 and rng.random() < 0.7:
            c["B"] = (c["B"] + 1) // 2
        else:
            c["L"] = (3 * c["L"] + 3) // 4
    c["left"] = rng.choice([-1, _spread(rng, 1, 4096), _spread(rng, 1, 512)])
    if op != "prompt":
        c["right"] = rng.choice([0, 0, -1, _spread(rng, 1, 512)])
    return c


def _lengths(case):
    """Tokens of each sequence, of the case alone: a fixed clip's, or texts from a fourth of the longest up."""
    B, L = case["B"], case["L"]
    if case.get("sections", "").count(",") == 2 or case["op"] == "attend":
        return [L] * B
    r = random.Random(1000 * B + L)
    return [L] + [r.randint(max(1, L // 4), L) for _ in range(B - 1)]


def _visible(lens, left, right, sinks):
    """Pairs of a query and a key that sees it, over all sequences: key j for query i if j <= i + right and (j >= i - left or j < sinks)."""
    total = 0
    for n in lens:
        i = np.arange(n, dtype=np.int64)
        hi = np.minimum(n - 1, i + right) if right >= 0 else np.full(n, n - 1)
        lo = np.maximum(0, i - left) if left >= 0 else np.zeros(n, dtype=np.int64)
        total += int(np.maximum(0, hi - lo + 1).sum() + np.minimum(np.minimum(lo, sinks), hi + 1).clip(0).sum())
    return total


def work(case):
    Hq, Hk, D = case["heads"], case["kv"], case["dim"]
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "rope":
        # q and k are read and written; six operations for each pair of values
        n = case["B"] * case["L"] * (Hq + Hk) * D
        return {"bytes": 2 * n * size, "flops": 3 * n}
    if op == "step":
        past = _past(case)
        S, left = case["sinks"], case["left"]
        seen = int(sum(min(p + 1, S + left + 1) if left >= 0 else p + 1 for p in past))
        row = (Hq + 2 * Hk) * D
        return {"bytes": size * (2 * seen * Hk * D + case["B"] * (row + Hq * D)), "flops": 4 * seen * Hq * D}
    lens = _lengths(case)
    M = sum(lens)
    pairs = _visible(lens, case["left"], case.get("right", 0), case["sinks"]) * Hq * D
    if op == "attend":
        return {"bytes": size * M * (2 * Hq + 2 * Hk) * D, "flops": 4 * pairs}
    if op == "prompt":
        # the attention, and the keys and values that the cache keeps
        kept = min(max(lens), _cap(case)) if len(lens) == 1 else sum(min(n, _cap(case)) for n in lens)
        return {"bytes": size * (M * (2 * Hq + 2 * Hk) + 2 * kept * Hk) * D, "flops": 4 * pairs}
    # forward: qkv read, out written; backward: qkv, out and its gradient read, dqkv written; two products forward, five backward
    return {"bytes": size * M * ((2 * Hq + 2 * Hk) + (3 * Hq + 2 * Hk) + (Hq + 2 * Hk)) * D, "flops": 14 * pairs}


def _cap(case):
    return case["sinks"] + case["left"] + 1 if case["left"] >= 0 else case["L"]


def _past(case):
    r = random.Random(case["B"] * 7919 + case["cap"])
    return [case["past"] - (r.randint(0, case["spread"]) if b else 0) for b in range(case["B"])]


# ---------------------------------------------------------------------------------------------- inputs
def _positions(case, n):
    """Positions of n tokens of one sequence, by axes: a text's count up; a clip has a class token at 0 and then frames of a square."""
    axes = case["sections"].count(",") + 1
    i = np.arange(n)
    if axes == 1:
        return i[:, None]
    side = max(1, min(21, int(math.sqrt(n))))
    j = np.maximum(i - 1, 0)
    grid = np.stack([j // (side * side), j // side % side, j % side], 1)
    return grid[:, 3 - axes:]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    Hq, Hk, D = case["heads"], case["kv"], case["dim"]

    def normal(*shape):
        out = torch.empty(shape, dtype=dt, device=dev)
        flat, step = out.view(-1), 1 << 27
        for a in range(0, flat.numel(), step):
            b = min(a + step, flat.numel())
            flat[a:b] = torch.randn(b - a, generator=g, device=dev).to(dt)
        return out

    s = dict(case)
    op = case["op"]
    if op == "step":
        B = case["B"]
        s["qkv"] = normal(B, (Hq + 2 * Hk) * D)
        s["k"], s["v"] = normal(B, case["cap"], Hk, D), normal(B, case["cap"], Hk, D)
        past = _past(case)
        s["past"] = torch.tensor(past, dtype=torch.int32, device=dev)
        axes = case["sections"].count(",") + 1
        pos = np.array([[p] if axes == 1 else [p // 441, p % 441 // 21, p % 21][3 - axes:] for p in past])
        s["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
        # room for the pieces that a long cache is split into, and their tickets
        s["pieces"] = torch.zeros(B * Hq * min(256, 1 + 1024 // (B * Hk)) * (D + 2) + B * Hk, dtype=torch.float32, device=dev)
        return s
    if op == "rope":
        # the query and key columns of packed rows, and one sequence's positions for every sequence of the batch
        s["x"] = normal(case["B"] * case["L"], (Hq + 2 * Hk) * D)[:, :(Hq + Hk) * D]
        s["pos"] = torch.tensor(_positions(case, case["L"]), dtype=torch.int32, device=dev)
        return s
    lens = _lengths(case)
    M = sum(lens)
    s["qkv"] = normal(M, (Hq + 2 * Hk) * D)
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    s["seqs"] = torch.tensor(np.stack([starts, lens, starts, lens], 1), dtype=torch.int32, device=dev)
    s["longest"] = max(lens)
    if op != "attend":
        s["pos"] = torch.tensor(np.concatenate([_positions(case, n) for n in lens]), dtype=torch.int32, device=dev)
    if op == "train":
        s["qkv"].requires_grad_(True)
        s["dout"] = normal(M, Hq * D)
    if op == "prompt":
        s["k"] = torch.zeros(case["B"], _cap(case), Hk, D, dtype=dt, device=dev)
        s["v"] = torch.zeros_like(s["k"])
    return s


# ---------------------------------------------------------------------------------------------- the plain form
@functools.lru_cache(maxsize=None)
def _ladder(sections, theta, shared):
    """Axis and frequency of every rotated pair."""
    dims = [int(t) for t in sections.split(",")]
    axis = np.concatenate([np.full(d // 2, a) for a, d in enumerate(dims)])
    if shared:
        freq = theta ** (-2.0 * np.arange(sum(dims) // 2) / sum(dims))
    else:
        freq = np.concatenate([theta ** (-2.0 * np.arange(d // 2) / d) for d in dims])
    return torch.tensor(axis, device="cuda"), torch.tensor(freq, dtype=torch.float64, device="cuda")


def _rotate(x, pos, s, inverse=False):
    """x [..., tokens, heads, dim] in 32 bits, rotated by pos [tokens, axes]; the angles in 64 bits."""
    axis, freq = _ladder(s["sections"], s["theta"], s["shared"])
    angle = pos.double()[:, axis] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if inverse:
        sin = -sin
    R = 2 * freq.numel()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if s.get("inter") else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if s.get("inter") else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _split(qkv, s):
    Hq, Hk, D = s["heads"], s["kv"], s["dim"]
    x = qkv.float().view(qkv.shape[0], Hq + 2 * Hk, D)
    return x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]


def _padded(x, rows, heads):
    """[M, H, D] -> [B, heads, H / heads * L, D]"""
    y = x[rows]                                                        # [B, L, H, D]
    B, L, H, D = y.shape
    return y.view(B, L, heads, H // heads, D).permute(0, 2, 3, 1, 4).reshape(B, heads, H // heads * L, D)


def _rows(x, rows, valid, M):
    """[B, heads, G * L, D] -> [M, heads * G, D]; rows of no sequence are zero"""
    B, L = rows.shape
    h, D = x.shape[1], x.shape[3]
    G = x.shape[2] // L
    y = x.view(B, h, G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, h * G, D)
    out = torch.zeros(M + 1, h * G, D, device=x.device)
    out[torch.where(valid, rows, M)] = y
    return out[:M]


def _mask(s, valid, L):
    i = torch.arange(L, device="cuda")
    left, right = s["left"], s.get("right", 0)
    see = torch.ones(L, L, dtype=torch.bool, device="cuda")
    if left >= 0:
        see &= (i[None, :] >= i[:, None] - left) | (i[None, :] < s["sinks"])
    if right >= 0:
        see &= i[None, :] <= i[:, None] + right
    return see & valid[:, None, :] & valid[:, :, None]


def _attend(q, k, v, s, scale):
    """-> out [M, Hq, D] and what a gradient needs, all in 32 bits over a padded batch"""
    M, Hk, L = q.shape[0], s["kv"], s["longest"]
    seqs = s["seqs"].long()
    i = torch.arange(L, device="cuda")
    valid = i < seqs[:, 1:2]
    rows = torch.where(valid, seqs[:, :1] + i, 0)
    Q, K, V = _padded(q, rows, Hk), _padded(k, rows, Hk), _padded(v, rows, Hk)
    S = torch.matmul(Q, K.transpose(2, 3).contiguous()) * scale
    B, _, GL, _ = S.shape
    see = _mask(s, valid, L)[:, None, None]
    P = S.view(B, Hk, GL // L, L, L).masked_fill_(~see, float("-inf"))
    P = P - P.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    P = P.exp_()
    P = P.div_(P.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)).view(B, Hk, GL, L)
    O = torch.matmul(P, V)
    return _rows(O, rows, valid, M), (Q, K, V, P, O, rows, valid)


def _gradients(dout, kept, s, scale):
    Q, K, V, P, O, rows, valid = kept
    M, Hk = dout.shape[0], s["kv"]
    dO = _padded(dout, rows, Hk) * valid.repeat(1, O.shape[2] // valid.shape[1])[:, None, :, None]
    dV = torch.matmul(P.transpose(2, 3).contiguous(), dO)
    dS = torch.matmul(dO, V.transpose(2, 3).contiguous())
    dS = dS.sub_((dO * O).sum(-1, keepdim=True)).mul_(P).mul_(scale)
    dQ, dK = torch.matmul(dS, K), torch.matmul(dS.transpose(2, 3).contiguous(), Q)
    return _rows(dQ, rows, valid, M), _rows(dK, rows, valid, M), _rows(dV, rows, valid, M)


def _keep(k, v, s):
    """The rows of a prompt that its cache holds: the sinks, and the last ones in rolling order."""
    seqs, cap, S = s["seqs"].long(), s["k"].shape[1], s["sinks"]
    i = torch.arange(s["longest"], device="cuda")
    n = seqs[:, 1:2]
    held = (i < n) & ((i < S) | (i >= n - (cap - S)))
    slot = torch.where(i < S, i, S + (i - S).clamp_min(0) % max(1, cap - S))
    slot = torch.where(held, slot, cap)
    rows = torch.where(held, seqs[:, :1] + i, 0)
    at = torch.arange(seqs.shape[0], device="cuda")[:, None].expand_as(slot)
    for cache, x in ((s["k"], k), (s["v"], v)):
        wide = torch.cat([cache, cache[:, :1]], 1)
        wide[at, slot] = x[rows].to(cache.dtype)
        cache.copy_(wide[:, :cap])


def _step(s, scale):
    q, k, v = _split(s["qkv"], s)
    q, k = _rotate(q, s["pos"], s), _rotate(k, s["pos"], s)
    B, cap, Hk, D = s["k"].shape
    past, S, left = s["past"].long(), s["sinks"], s["left"]
    at = torch.arange(B, device="cuda")
    slot = torch.where(past < S, past, S + (past - S).clamp_min(0) % (cap - S)) if s["rolling"] else past
    s["k"][at, slot] = k.to(s["k"].dtype)
    s["v"][at, slot] = v.to(s["v"].dtype)
    K = s["k"].permute(0, 2, 3, 1).float()                             # [B, Hk, D, cap]
    S_ = torch.matmul(q.view(B, Hk, -1, D), K.contiguous()) * scale
    del K
    j = torch.arange(cap, device="cuda")[None]
    see = j <= past[:, None]
    if left >= 0 and not s["rolling"]:
        see = see & ((j >= past[:, None] - left) | (j < S))
    P = _softmax(S_, see)
    out = torch.matmul(P, s["v"].permute(0, 2, 1, 3).float().contiguous())
    return out.reshape(B, -1).to(s["qkv"].dtype), s["k"], s["v"]


def _softmax(x, see):
    x = x.masked_fill_(~see[:, None, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    return x.div_(x.sum(-1, keepdim=True))


def _plain(s):
    op, dt, scale = s["op"], DTYPES[s["dtype"]], s["dim"] ** -0.5
    if op == "rope":
        x = s["x"].float().reshape(s["B"], s["L"], s["heads"] + s["kv"], s["dim"])
        return _rotate(x, s["pos"], s, s["inverse"]).to(dt).view(s["x"].shape)
    if op == "step":
        return _step(s, scale)
    with torch.no_grad():
        q, k, v = _split(s["qkv"], s)
        if op != "attend":
            q, k = _rotate(q, s["pos"], s), _rotate(k, s["pos"], s)
        out, kept = _attend(q, k, v, s, scale)
        M = out.shape[0]
        if op == "attend":
            return out.view(M, -1).to(dt)
        if op == "prompt":
            _keep(k, v, s)
            return out.view(M, -1).to(dt), s["k"], s["v"]
        dq, dk, dv = _gradients(s["dout"].float().view(M, s["heads"], s["dim"]), kept, s, scale)
        dq, dk = _rotate(dq, s["pos"], s, True), _rotate(dk, s["pos"], s, True)
        return out.view(M, -1).to(dt), torch.cat([dq, dk, dv], 1).view(M, -1).to(dt)


# ---------------------------------------------------------------------------------------------- the framework's operators
@functools.lru_cache(maxsize=None)
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "oa-transformer_amd"))
    from OATrans.model import window_attention
    from OATrans.ops import hip
    return hip, window_attention


@functools.lru_cache(maxsize=None)
def _rope(sections, theta, shared, inter):
    return _framework()[0].RopeAxes([int(t) for t in sections.split(",")], theta=theta, shared=shared, interleaved=inter)


def _calls(s):
    hip, layers = _framework()
    op, Hq, Hk, D = s["op"], s["heads"], s["kv"], s["dim"]
    rope = _rope(s["sections"], s["theta"], s["shared"], s.get("inter", False)) if op != "attend" else None
    if op == "rope":
        return hip.rope_axes(s["x"], s["pos"], rope, Hq + Hk, D, inverse=s["inverse"])
    if op == "step":
        out = hip.attn_window_step(s["qkv"], s["past"], s["k"], s["v"], Hq, left=s["left"], sinks=s["sinks"], rolling=s["rolling"],
                                   rope=rope, pos=s["pos"], pieces=s["pieces"])
        return out, s["k"], s["v"]
    more = dict(left=s["left"], right=s.get("right", 0), sinks=s["sinks"], longest=s["longest"], packed=True)
    if op == "attend":
        with torch.no_grad():
            return layers.window_attention(s["qkv"], s["seqs"], Hq, Hk, D, **more)
    if op == "prompt":
        with torch.no_grad():
            out = layers.window_attention(s["qkv"], s["seqs"], Hq, Hk, D, rope=rope, pos=s["pos"], cache=(s["k"], s["v"]), **more)
        return out, s["k"], s["v"]
    out = layers.window_attention(s["qkv"], s["seqs"], Hq, Hk, D, rope=rope, pos=s["pos"], **more)
    (grad,) = torch.autograd.grad(out, s["qkv"], s["dout"])
    return out.detach(), grad


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _turned(x, pos, case, sign=1.0):
    """x [tokens, heads, dim] in 64 bits: every pair is a complex number times e^(i angle)."""
    dims = [int(t) for t in case["sections"].split(",")]
    R = sum(dims)
    y = x.clone()
    p = 0
    for a, d in enumerate(dims):
        for e in range(d // 2):
            f = case["theta"] ** (-2.0 * p / R) if case["shared"] else case["theta"] ** (-2.0 * e / d)
            w = torch.polar(torch.ones(pos.shape[0], dtype=torch.float64, device=x.device), sign * pos[:, a].double() * f)[:, None]
            u, v = (2 * p, 2 * p + 1) if case.get("inter") else (p, p + R // 2)
            z = torch.complex(x[..., u], x[..., v]) * w
            y[..., u], y[..., v] = z.real, z.imag
            p += 1
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op, Hq, Hk, D = case["op"], case["heads"], case["kv"], case["dim"]
    scale, G = 1.0 / math.sqrt(D), Hq // Hk
    if op == "rope":
        n = case["L"]
        out = [_turned(s["x"][b * n:(b + 1) * n].double().reshape(n, -1, D), s["pos"], case, -1.0 if case["inverse"] else 1.0)
               for b in range(case["B"])]
        return torch.cat(out).view(s["x"].shape)
    x = s["qkv"].detach().double().view(s["qkv"].shape[0], -1, D)
    if op != "attend":
        x = torch.cat([_turned(x[:, :Hq + Hk], s["pos"], case), x[:, Hq + Hk:]], 1)
    if op == "step":
        out = torch.zeros(case["B"], Hq, D, dtype=torch.float64, device="cuda")
        cap, S = case["cap"], case["sinks"]
        kc, vc = s["k"].double(), s["v"].double()
        for b, p in enumerate(_past(case)):
            at = p if not case["rolling"] or p < S else S + (p - S) % (cap - S)
            kc[b, at], vc[b, at] = x[b, Hq:Hq + Hk], x[b, Hq + Hk:]
            tokens = list(range(p + 1)) if case["left"] < 0 else list(range(min(S, p + 1))) + list(range(max(S, p - case["left"], 0), p + 1))
            slots = [t if not case["rolling"] or t < S else S + (t - S) % (cap - S) for t in tokens]
            slots = torch.tensor(slots, device="cuda")
            for h in range(Hk):
                a = kc[b, slots, h] @ x[b, h * G:(h + 1) * G].T * scale
                w = (a - torch.logsumexp(a, 0)).exp()
                out[b, h * G:(h + 1) * G] = w.T @ vc[b, slots, h]
        return out.view(case["B"], -1), kc, vc
    lens = _lengths(case)
    right = case.get("right", 0)
    out, grad = torch.zeros(x.shape[0], Hq, D, dtype=torch.float64, device="cuda"), torch.zeros_like(x)
    at = 0
    for n in lens:
        i = torch.arange(n, device="cuda")
        gap = i[:, None] - i[None, :]
        hide = torch.zeros(n, n, dtype=torch.bool, device="cuda")
        if case["left"] >= 0:
            hide |= (gap > case["left"]) & (i[None, :] >= case["sinks"])
        if right >= 0:
            hide |= -gap > right
        for h in range(Hq):
            q, k, v = x[at:at + n, h], x[at:at + n, Hq + h // G], x[at:at + n, Hq + Hk + h // G]
            a = (q @ k.T * scale).masked_fill(hide, -math.inf)
            w = (a - torch.logsumexp(a, 1, keepdim=True)).exp()
            out[at:at + n, h] = w @ v
            if op == "train":
                d = s["dout"][at:at + n, h * D:(h + 1) * D].double()
                e = w * (d @ v.T - (d * out[at:at + n, h]).sum(1, keepdim=True)) * scale
                grad[at:at + n, h] = e @ k
                grad[at:at + n, Hq + h // G] += e.T @ q
                grad[at:at + n, Hq + Hk + h // G] += w.T @ d
        at += n
    if op == "attend":
        return out.view(out.shape[0], -1)
    if op == "prompt":
        kc, vc = s["k"].double(), s["v"].double()
        cap, S, at = _cap(case), case["sinks"], 0
        for b, n in enumerate(lens):
            keep = [t for t in range(n) if t < S or t >= n - (cap - S)]
            slots = [t if t < S else S + (t - S) % max(1, cap - S) for t in keep]
            rows = torch.tensor(keep, device="cuda") + at
            kc[b, slots], vc[b, slots] = x[rows, Hq:Hq + Hk], x[rows, Hq + Hk:]
            at += n
        return out.view(out.shape[0], -1), kc, vc
    grad = torch.cat([_turned(grad[:, :Hq + Hk], s["pos"], case, -1.0), grad[:, Hq + Hk:]], 1)
    return out.view(out.shape[0], -1), grad.view(out.shape[0], -1)
