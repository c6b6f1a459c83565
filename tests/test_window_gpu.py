"""Rotary positions, windowed attention (forward, backward) and its one-token form on a real MI355X against their definitions in 64
bits (oracle/window_oracle.py, on the same device) on the same 16-bit inputs.

Tolerances, with u = finfo(dtype).eps / 2 (half a step): an output is rounded once (u |value|), and a product of two 16-bit operands
of which one is a rounded probability (or its gradient) is off by u times the sum of its terms' absolute values (the oracle's
*_abs) at most.  The terms' roundings are independent, each at most u: their sum stays within 6 u times the root of the sum of the terms'
squares (*_sq; six deviations or more), and the smaller of the two bounds is taken.  2^-14 of *_abs stands for sums, exponentials and the log-sum-exp in 32 bits."""
import math

import pytest
import torch

from oracle import window_oracle as wo

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _hip():
    from OATrans.ops import hip
    hip.lib()
    return hip


def rnd(*shape, dtype=BF, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 31 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def terms(r, name, u):
    """how far a sum with 16-bit terms may be off (see above)"""
    return torch.minimum(u * r[name + "_abs"], 6 * u * r[name + "_sq"]) + 2.0 ** -14 * r[name + "_abs"]


def within(got, ref, tol, what):
    got, tol = got.double(), tol.expand_as(ref) if isinstance(tol, torch.Tensor) else tol
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; worst {float(((got - ref).abs() - tol)[bad].max()):.3g} over, "
                           f"at {bad.nonzero()[0].tolist()}: {got[tuple(bad.nonzero()[0])]} for {ref[tuple(bad.nonzero()[0])]}")


# ---------------------------------------------------------------------------------------------- rotary positions
ROPE = [((64,), 10000.0, False, False, 64), ((16, 24, 24), 10000.0, False, False, 64), ((16, 24, 24), 100.0, True, True, 64),
        ((32, 48, 48), 5e5, True, False, 128), ((48,), 10000.0, False, False, 64), ((2, 4), 10.0, False, True, 64),
        ((6, 4, 4, 4), 50.0, False, False, 72), ((2,), 7.0, False, False, 2), ((0, 8), 7.0, False, True, 10)]


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_rope_axes(case, dtype):
    hip = _hip()
    sections, theta, shared, inter, dim = ROPE[case]
    rope = hip.RopeAxes(sections, theta, interleaved=inter, shared=shared)
    for M, P, heads in ((1, 1, 1), (3, 3, 5), (70, 35, 24), (4099, 4099, 3)):
        wide = rnd(M, heads * dim + 8, dtype=dtype, seed=case)
        x = wide[:, :heads * dim]
        g = torch.Generator().manual_seed(case + M)
        pos = torch.randint(-5000, 2_000_000, (P, len(sections)), generator=g, dtype=torch.int32)
        for inverse in (False, True):
            out = hip.rope_axes(x, pos.to(DEV), rope, heads, dim, inverse=inverse)
            ref = wo.rope(x.reshape(M, heads, dim), pos.repeat(M // P, 1).to(DEV), sections,
                          theta, shared, inter, inverse).reshape(M, -1)
            # cos and sin in 32 bits (a few 2^-24 of the pair's length), one rounding of the result
            size = x.double().reshape(M, heads, dim).abs().amax(-1, keepdim=True).expand(M, heads, dim).reshape(M, -1)
            within(out, ref, half_step(dtype) * ref.abs() + 2.0 ** -21 * size + torch.finfo(dtype).tiny, f"rope {M}")
        back = hip.rope_axes(out, pos.to(DEV), rope, heads, dim, out=out)          # in place, the turn back of the inverse
        assert back is out
        within(out, x.double(), 3 * half_step(dtype) * size * 1.5 + 2.0 ** -20 * size, "rope back")
        assert torch.equal(wide[:, heads * dim:], rnd(M, heads * dim + 8, dtype=dtype, seed=case)[:, heads * dim:])


def test_rope_axes_unaligned_rows_and_gradient():
    hip = _hip()
    from OATrans.model import window_attention as wa
    rope = hip.RopeAxes((16, 24, 24))
    flat = rnd(1 + 33 * 193, dtype=torch.float32)
    x = flat[1:].view(33, 193)[:, :192]                                             # 4-byte aligned rows of an odd pitch
    pos = torch.randint(0, 400, (33, 3), dtype=torch.int32)
    out = hip.rope_axes(x, pos.to(DEV), rope, 3, 64)
    ref = wo.rope(x.reshape(33, 3, 64), pos.to(DEV), (16, 24, 24), 10000.0).reshape(33, -1)
    within(out, ref, 2.0 ** -20 * x.double().abs().max().item() * torch.ones_like(ref), "unaligned")
    leaf = x.detach().clone().contiguous().requires_grad_(True)
    w = rnd(33, 192, dtype=torch.float32, seed=5)
    (g,) = torch.autograd.grad((wa.rope_axes(leaf, pos.to(DEV), rope, 3, 64) * w).sum(), leaf)
    ref = wo.rope(w.reshape(33, 3, 64), pos.to(DEV), (16, 24, 24), 10000.0, inverse=True).reshape(33, -1)
    within(g, ref, 2.0 ** -20 * w.double().abs().max().item() * torch.ones_like(ref), "gradient")


@pytest.mark.parametrize("inter", [False, True])
def test_rope_axes_large_output(inter):
    """Over 96 MB of output the stores bypass the caches: the same values, to the last row."""
    hip = _hip()
    rope = hip.RopeAxes((48,), interleaved=inter)                                   # 16 of 64 values pass through
    M, heads = 35000, 24
    x = torch.randn(M, heads * 64, dtype=BF, device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    pos = torch.arange(M, dtype=torch.int32, device=DEV)[:, None].contiguous()
    out = hip.rope_axes(x, pos, rope, heads, 64)
    for a, b in ((0, 10000), (10000, 20000), (20000, 30000), (30000, M)):
        assert torch.equal(out[a:b], hip.rope_axes(x[a:b], pos[a:b], rope, heads, 64))


# ---------------------------------------------------------------------------------------------- attention
# queries, keys, Hq, Hkv, D, left, right, sinks
ATTN = [
    ([1], [1], 1, 1, 64, -1, 0, 0),
    ([0, 5, 0, 1], None, 2, 1, 64, -1, 0, 0),
    ([33, 64, 65], None, 2, 2, 128, -1, -1, 0),
    ([31, 129, 2], None, 4, 2, 64, 7, 0, 0),
    ([200], None, 3, 1, 128, 16, 0, 3),
    ([300, 17], None, 2, 2, 64, 40, 40, 1),
    ([257], None, 2, 1, 64, 0, 0, 0),
    ([150], None, 2, 2, 64, 5, 9, 70),
    ([3, 1, 130], [70, 1, 129], 4, 4, 64, -1, 0, 0),                                  # more keys; as many; fewer (the first query sees nothing)
    ([130, 40], [5, 0], 2, 1, 128, -1, 0, 0),                                         # most rows see nothing; no keys at all
    ([64, 1], [700, 513], 6, 2, 64, 100, 0, 4),
    ([20], [300], 2, 2, 128, 30, 50, 200),
    ([700], None, 8, 1, 64, 64, 0, 2),
    ([520, 130, 90], None, 2, 1, 128, 100, 30, 33),
    ([1100], None, 1, 1, 64, -1, -1, 0),
    ([2300], None, 1, 1, 64, 90, 0, 130),                                             # more sinks than a tile of keys
    ([1500, 1], None, 2, 1, 128, 50, 50, 1),
    ([1300, 700], None, 4, 1, 128, 100, 0, 40),                                       # the sinks' far queries are split over workgroups
    ([900, 20], [1400, 900], 4, 2, 64, 60, 10, 3),
    ([1500], None, 1, 1, 64, 100, 0, 600),                                            # many sinks: their own tiles walk all queries
    ([40] * 9 + [0, 300], None, 3, 3, 64, 20, 5, 2),                                  # a ragged batch: places of the list that are empty
    ([130] * 5, None, 8, 2, 128, -1, 0, 0),                                           # an even one, dealt by key heads
]


def _case(n, dtype, pad=3):
    """Packed rows with `pad` rows of NaN before, between and after the sequences, in buffers of a wider pitch."""
    qn, kn, Hq, Hkv, D, left, right, sinks = ATTN[n]
    kn = qn if kn is None else kn
    seqs, aq, ak = [], pad, pad
    for a, b in zip(qn, kn):
        seqs.append((aq, a, ak, b))
        aq, ak = aq + a + pad, ak + b + pad
    make = lambda rows, heads, seed: rnd(rows, heads * D + 24, dtype=dtype, seed=seed + n)
    q, k, v, do = make(aq, Hq, 1), make(ak, Hkv, 2), make(ak, Hkv, 3), make(aq, Hq, 4)
    for t, which in ((q, 0), (do, 0), (k, 2), (v, 2)):
        own = torch.zeros(t.shape[0], dtype=torch.bool)
        for s in seqs:
            own[s[which]:s[which] + s[which + 1]] = True
        t[~own.to(DEV)] = float("nan")
    cut = lambda t, heads: t[:, 8:8 + heads * D]
    return seqs, cut(q, Hq), cut(k, Hkv), cut(v, Hkv), cut(do, Hq), (Hq, Hkv, D, left, right, sinks), max(qn), max(kn)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", range(len(ATTN)))
def test_attn_window(n, dtype):
    hip = _hip()
    seqs, q, k, v, do, (Hq, Hkv, D, left, right, sinks), mq, mk = _case(n, dtype)
    table = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    scale = 0.9 / math.sqrt(D)
    out = torch.full((q.shape[0], Hq * D), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((q.shape[0], Hq), 7.0, device=DEV)
    hip.attn_window_fwd(q, k, v, table, Hq, Hkv, D, mq, mk, left, right, sinks, scale, out=out, lse=lse)
    dq, dk, dv = (torch.full((t.shape[0], t.shape[1] + 8), 7.0, dtype=dtype, device=DEV)[:, :t.shape[1]] for t in (q, k, v))
    hip.attn_window_bwd(q, k, v, out, lse, do, table, Hq, Hkv, D, mq, mk, left, right, sinks, scale, dq=dq, dk=dk, dv=dv)
    r = wo.attention(q, k, v, seqs, Hq, Hkv, D, left, right, sinks, scale, dout=do, out=out)
    u = half_step(dtype)
    tiny = torch.finfo(dtype).tiny                                                     # what rounds to a subnormal or to zero
    sq, sk = r["seen_q"], r["seen_k"]
    within(out[sq], r["out"][sq], (u * r["out"].abs() + terms(r, "out", u))[sq] + tiny, "out")
    some = r["lse"] > -math.inf
    within(lse[sq[:, None] & some], r["lse"][sq[:, None] & some], 2.0 ** -17 * (4 + r["lse"].abs())[sq[:, None] & some], "lse")
    assert (lse[sq[:, None] & ~some] == -math.inf).all()
    within(dq[sq], r["dq"][sq], (u * r["dq"].abs() + terms(r, "dq", u) + 1.01 * r["dq_off"])[sq] + tiny * D, "dq")
    within(dk[sk], r["dk"][sk], (u * r["dk"].abs() + terms(r, "dk", u) + 1.01 * r["dk_off"])[sk] + tiny * (8 + mq), "dk")
    within(dv[sk], r["dv"][sk], (u * r["dv"].abs() + terms(r, "dv", u))[sk] + tiny * (8 + mq), "dv")
    for t, s in ((out, sq), (lse, sq), (dq, sq), (dk, sk), (dv, sk)):                  # rows of no sequence stay as they were
        assert (t[~s] == 7.0).all()
    # every sum has one order
    again = [torch.zeros_like(t) for t in (dq, dk, dv)]
    hip.attn_window_bwd(q, k, v, out, lse, do, table, Hq, Hkv, D, mq, mk, left, right, sinks, scale, dq=again[0], dk=again[1], dv=again[2])
    for a, b, s in zip(again, (dq, dk, dv), (sq, sk, sk)):
        assert torch.equal(a[s], b[s])


def test_attn_window_large_and_equal_scores():
    """Scores of +-2000 (a single key takes all) and scores all alike (the mean of the values)."""
    hip = _hip()
    table = hip.seq_table([200])
    v = rnd(200, 64, seed=1)
    q = torch.zeros(200, 64, dtype=BF, device=DEV)
    out = hip.attn_window_fwd(q, q, v, table, 1, 1, 64, 200, 200, right=-1)
    mean = v.double().mean(0).expand(200, 64)
    within(out, mean, half_step(BF) * mean.abs() + (half_step(BF) + 2.0 ** -14) * v.double().abs().mean(0), "mean")
    eye = torch.zeros(200, 64, dtype=BF, device=DEV)
    eye[torch.arange(200), torch.arange(200) % 64] = 128.0
    out = hip.attn_window_fwd(eye[:64].contiguous(), eye[:64].contiguous(), v[:64].contiguous(), hip.seq_table([64]), 1, 1, 64, 64, 64, right=-1)
    assert torch.equal(out, v[:64])


def test_attn_window_bad_tables_are_empty():
    """A table on the device cannot be refused by the host: a sequence that does not fit is left out, its rows stay."""
    hip = _hip()
    q = rnd(100, 64)
    for bad in ((-1, 10, 0, 10), (95, 10, 0, 10), (0, -5, 0, 10), (0, 10, 91, 10), (0, 10, 2 ** 31 - 8, 10), (2 ** 31 - 8, 10, 0, 10), (0, 51, 0, 51)):
        table = torch.tensor([bad, (60, 20, 60, 20)], dtype=torch.int32, device=DEV)
        out = torch.full((100, 64), 7.0, dtype=BF, device=DEV)
        hip.attn_window_fwd(q, q, q, table, 1, 1, 64, 50, 50, out=out)
        ok = hip.attn_window_fwd(q, q, q, table[1:], 1, 1, 64, 50, 50, out=torch.full_like(out, 7.0))
        assert torch.equal(out, ok) and (out[:60] == 7.0).all()


def test_attn_window_far_rows():
    """Rows beyond 2^31 elements of a buffer."""
    hip = _hip()
    M = 2 ** 20
    q = torch.empty(M, 2304, dtype=BF, device=DEV)
    q[-150:] = rnd(150, 2304)
    seqs = [(M - 150, 100, M - 150, 100), (M - 50, 50, M - 50, 50)]
    table = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    out = torch.empty(M, 2304, dtype=BF, device=DEV)
    k, v = q[:, 768:1536], q[:, 1536:]
    lse = torch.empty(M, 12, device=DEV)
    hip.attn_window_fwd(q[:, :768], k, v, table, 12, 12, 64, 100, 100, 20, 0, 1, out=out[:, 1536:], lse=lse)
    tail = [(0, 100, 0, 100), (100, 50, 100, 50)]
    small = [t[-150:].contiguous() for t in (q[:, :768], k, v)]
    ref = hip.attn_window_fwd(*small, torch.tensor(tail, dtype=torch.int32, device=DEV), 12, 12, 64, 100, 100, 20, 0, 1)
    assert torch.equal(out[-150:, 1536:], ref)
    g = torch.empty(M, 2304, dtype=BF, device=DEV)
    hip.attn_window_bwd(q[:, :768], k, v, out[:, 1536:], lse, q[:, 768:1536], table, 12, 12, 64, 100, 100, 20, 0, 1, dq=g[:, :768],
                        dk=g[:, 768:1536], dv=g[:, 1536:])
    small_g = hip.attn_window_bwd(*small, ref, lse[-150:].contiguous(), small[1], torch.tensor(tail, dtype=torch.int32, device=DEV), 12, 12, 64, 100,
                                  100, 20, 0, 1)
    for a, b in zip((g[-150:, :768], g[-150:, 768:1536], g[-150:, 1536:]), small_g):
        assert torch.equal(a, b)


@pytest.mark.parametrize("padded", [False, True])
def test_window_attention_gradient_with_rope(padded):
    """The layer: rotary positions, attention and their gradient with respect to the packed q | k | v; rows of padding get zeros."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    Hq, Hkv, D, lens, left, right, sinks = 4, 2, 64, [90, 33], 30, 10, 1
    sections = (16, 24, 24)
    rope = hip.RopeAxes(sections)
    M = 2 * 90 if padded else sum(lens)
    table = hip.seq_table(lens, q_rows=(0, 90) if padded else None)
    qkv = rnd(M, (Hq + 2 * Hkv) * D, seed=3).requires_grad_(True)
    pos = torch.randint(0, 30, (M, 3), dtype=torch.int32)
    out = wa.window_attention(qkv, table, Hq, Hkv, D, left, right, sinks, longest=90, rope=rope, pos=pos.to(DEV), packed=not padded)
    dout = rnd(M, Hq * D, seed=4)
    (g,) = torch.autograd.grad(out, qkv, dout)
    # the oracle takes the turned rows that the rotary operator (tested above) gives
    n = (Hq + Hkv) * D
    qk = hip.rope_axes(qkv.detach()[:, :n], pos.to(DEV), rope, Hq + Hkv, D)
    seqs = [tuple(t) for t in table.tolist()]
    r = wo.attention(qk[:, :Hq * D], qk[:, Hq * D:], qkv.detach()[:, n:], seqs, Hq, Hkv, D, left, right, sinks, D ** -0.5, dout=dout, out=out.detach())
    u = half_step(BF)
    within(out.detach(), r["out"], u * r["out"].abs() + terms(r, "out", u) + 1e-30, "out")
    back = wo.rope(torch.cat([r["dq"], r["dk"]], 1).view(M, Hq + Hkv, D), pos.to(DEV), sections, 10000.0, inverse=True).view(M, n)
    tol = torch.cat([u * r["dq"].abs() + terms(r, "dq", u) + 1.01 * r["dq_off"], u * r["dk"].abs() + terms(r, "dk", u) + 1.01 * r["dk_off"]], 1)
    # the turn mixes a pair's errors (at most their sum) and rounds once more
    pair = tol.view(M, Hq + Hkv, 2, 32)
    tol = (pair + pair.flip(2)).view(M, n) + u * back.abs() * 1.1
    within(g[:, :n], back, tol + 1e-30, "dq | dk")
    within(g[:, n:], r["dv"], u * r["dv"].abs() + terms(r, "dv", u) + 1e-30, "dv")
    if padded:
        assert (out[90 + 33:] == 0).all() and (g[90 + 33:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,Hq,Hkv,D,sections,inter,left,right,sinks,gap", [
    ([90, 33], 4, 2, 64, (16, 24, 24), False, 30, 10, 1, 5), ([1300, 700], 4, 1, 128, (128,), False, 100, 0, 40, 0),
    ([2300], 1, 1, 64, (32, 32), False, 90, 3, 130, 0), ([1500, 1], 2, 2, 128, (32, 48, 48), False, 60, 60, 1, 2), ([70], 2, 1, 64, (48,), False, -1, -1, 0, 0),
    ([70], 2, 1, 64, (64,), True, -1, 0, 3, 1), ([0, 17], 3, 3, 128, (128,), False, -1, 0, 0, 0)])
def test_gradient_turned_back_where_it_is_formed(lens, Hq, Hkv, D, sections, inter, left, right, sinks, gap, dtype):
    """The layer's dq and dk against those of the single operators turned back in 64 bits.  Both have the same 32-bit sums; the operators'
    are rounded before the turn (each of a pair by half a step of its size), the layer's after it."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    M, n, L = sum(lens) + gap * len(lens), (Hq + Hkv) * D, max(lens)
    starts = [sum(lens[:b]) + gap * (b + 1) for b in range(len(lens))]
    table, rope = hip.seq_table(lens, q_rows=starts), hip.RopeAxes(sections, interleaved=inter)
    qkv = rnd(M, n + Hkv * D, dtype=dtype, seed=11).requires_grad_()
    pos = torch.randint(-40, 4000, (M, len(sections)), dtype=torch.int32, generator=torch.Generator().manual_seed(6)).to(DEV)
    dout = rnd(M, Hq * D, dtype=dtype, seed=12)
    out = wa.window_attention(qkv, table, Hq, Hkv, D, left, right, sinks, longest=L, rope=rope, pos=pos)
    (g,) = torch.autograd.grad(out, qkv, dout)
    x = qkv.detach()
    qk, lse = hip.rope_axes(x[:, :n], pos, rope, Hq + Hkv, D), torch.zeros(M, Hq, device=DEV)
    q, k, v = qk[:, :Hq * D], qk[:, Hq * D:], x[:, n:]
    same = hip.attn_window_fwd(q, k, v, table, Hq, Hkv, D, L, L, left, right, sinks, lse=lse)
    assert torch.equal(out, same)
    dq, dk, dv = hip.attn_window_bwd(q, k, v, same, lse, dout, table, Hq, Hkv, D, L, L, left, right, sinks)
    assert torch.equal(g[:, n:], dv)
    d = torch.cat([dq, dk], 1).view(M, Hq + Hkv, D)
    back = wo.rope(d, pos, sections, 10000.0, False, inter, inverse=True).view(M, n)
    R = 2 * rope.pairs
    a = d.double().abs()
    other = a.clone()
    other[..., :R] = a[..., :R].unflatten(-1, (-1, 2)).flip(-1).flatten(-2) if inter else a[..., :R].unflatten(-1, (2, -1)).flip(-2).flatten(-2)
    u = half_step(dtype)
    within(g[:, :n], back, (1.01 * u * (a + other)).view(M, n) + 1.01 * u * back.abs() + 4 * torch.finfo(dtype).tiny, "dq | dk")


def test_window_attention_gradient_by_differences():
    """The directional derivative of the layer against central differences of the 64-bit definition."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    M, D = 40, 64
    table = hip.seq_table([M])
    qkv = rnd(M, 3 * D, dtype=HF, seed=8).requires_grad_(True)
    w, d = rnd(M, D, dtype=HF, seed=9), rnd(M, 3 * D, dtype=torch.float64, seed=10)
    out = wa.window_attention(qkv, table, 1, 1, D, left=11, right=0, sinks=2, longest=M)
    (g,) = torch.autograd.grad(out, qkv, w)

    def f(x):
        return (wo.attention(x[:, :D], x[:, D:2 * D], x[:, 2 * D:], [(0, M, 0, M)], 1, 1, D, 11, 0, 2, D ** -0.5)["out"] * w.double()).sum()
    x, h = qkv.detach().double(), 1e-5
    diff = float(f(x + h * d) - f(x - h * d)) / (2 * h)
    # the gradient's roundings: a few half steps (2^-11) of its size, in random directions
    size = float((g.double() * d).norm())
    assert abs(float((g.double() * d).sum()) - diff) <= 6 * 2.0 ** -11 * size * math.sqrt(3 * M * D) / 8, (diff, float((g.double() * d).sum()))


# ---------------------------------------------------------------------------------------------- one token
# B, cap, Hq, Hkv, D, left, sinks, rolling, past
STEP = [
    (1, 1, 1, 1, 64, -1, 0, False, [0]),
    (3, 40, 4, 2, 64, -1, 0, False, [0, 39, -1]),
    (2, 700, 12, 12, 64, 100, 4, False, [699, 50]),
    (2, 512, 12, 12, 64, 507, 4, True, [511, 5000]),
    (3, 37, 6, 3, 128, 33, 3, True, [2, 37, 1000]),
    (2, 1500, 8, 1, 128, -1, 0, False, [1499, 300]),
    (1, 300, 40, 1, 64, 0, 0, False, [299]),
    (1, 4000, 34, 2, 128, 3000, 700, False, [3999]),
    (2, 129, 5, 5, 128, -1, 0, False, [128, 129]),                                    # the second has no slot left
    (1, 70, 2, 1, 64, 69, 0, True, [10 ** 9]),
    (1, 9000, 2, 2, 64, -1, 0, False, [8999]),
    (4, 260, 16, 8, 128, 30, 250, False, [255, 259, 31, 3]),
]


def _step_ref(qkv, kc, vc, past, Hq, Hkv, D, left, sinks, rolling, scale, rope, sections, pos):
    """-> out, its abs and sq, caches with the new rows as this dtype holds them"""
    B, cap = kc.shape[:2]
    x = qkv.reshape(B, Hq + 2 * Hkv, D)
    kc, vc = kc.clone(), vc.clone()
    out, size, sq = (torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV) for _ in range(3))
    for b, p in enumerate(past):
        if p < 0 or (not rolling and p >= cap):
            continue
        qk = x[b:b + 1, :Hq + Hkv].double()
        if rope is not None:
            qk = wo.rope(qk, pos[b:b + 1].to(DEV), sections, rope.theta, rope.shared, rope.interleaved)
        qk = qk[0].to(kc.dtype)
        s = wo.slot(p, cap, sinks, rolling)
        kc[b, s], vc[b, s] = qk[Hq:], x[b, Hq + Hkv:]
        out[b], size[b], sq[b] = wo.step(qk[:Hq], kc[b], vc[b], p, left, sinks, rolling, scale)
    return out.view(B, -1), {"out_abs": size.view(B, -1), "out_sq": sq.view(B, -1)}, kc, vc


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", range(len(STEP)))
def test_attn_window_step(n, dtype):
    hip = _hip()
    B, cap, Hq, Hkv, D, left, sinks, rolling, past = STEP[n]
    u = half_step(dtype)
    pieces = hip.window_step_workspace(B, Hq, Hkv, D)
    for turn in (None, ((D,), False), ((16, 24, 24), True)):
        qkv = rnd(B, (Hq + 2 * Hkv) * D + 16, dtype=dtype, seed=n)[:, :(Hq + 2 * Hkv) * D]
        kc, vc = rnd(B, cap, Hkv, D, dtype=dtype, seed=n + 1), rnd(B, Hkv, cap, D, dtype=dtype, seed=n + 2).transpose(1, 2)
        rope = hip.RopeAxes(turn[0], interleaved=turn[1]) if turn else None
        pos = torch.randint(0, 3000, (B, len(turn[0])), dtype=torch.int32) if turn else None
        scale = 1.1 / math.sqrt(D)
        ref, r, kr, vr = _step_ref(qkv, kc, vc, past, Hq, Hkv, D, left, sinks, rolling, scale, rope, turn and turn[0], pos)
        # the turned query and key are the operator's own 16-bit values: one of them may fall on the other side of a border (32-bit angles),
        # which moves a score by a step of one term, 2 u |q k| scale <= 2^-5 u of the probabilities' size at these magnitudes
        for _ in range(2):                                                            # the workspace is ready again after a call
            out = hip.attn_window_step(qkv, torch.tensor(past, dtype=torch.int32, device=DEV), kc, vc, Hq, left=left, sinks=sinks, rolling=rolling,
                                       scale=scale, rope=rope, pos=pos.to(DEV) if turn else None, pieces=pieces)
            within(out, ref, u * ref.abs() + terms(r, "out", u) + (2 * u * r["out_abs"] if turn else 0.0) + torch.finfo(dtype).tiny, f"step {turn}")
        assert torch.equal(vc, vr)
        if turn:
            within(kc, kr.double(), 2 * u * kr.double().abs() + 2.0 ** -20, "cache")
        else:
            assert torch.equal(kc, kr)
        same = [b for b, p in enumerate(past) if p < 0 or (not rolling and p >= cap)]
        assert all((out[b] == 0).all() for b in same)


@pytest.mark.parametrize("cap,sinks,rolling", [(1500, 4, True), (1500, 0, True), (1500, 4, False), (4000, 700, True)])
def test_attn_window_step_sees_its_own_token(cap, sinks, rolling):
    """The new token's key points where the query does and takes nearly all of the weight: its value is the output, whichever piece of
    the cache its slot falls into."""
    hip = _hip()
    D = 64
    pieces = hip.window_step_workspace(1, 1, 1, D)
    for past in (0, 3, 255, 256, 700, cap - 1, cap, cap + 255, cap + 900, 3 * cap):
        if not rolling and past >= cap:
            continue
        kc, vc = rnd(1, cap, 1, D, seed=past), rnd(1, cap, 1, D, seed=past + 1)
        qkv = rnd(1, 3 * D, seed=past + 2)
        qkv[:, D:2 * D] = 8 * qkv[:, :D]                     # its score is 8 |q|^2 / 8 ~ 64, the others' ~ 1: e^-50 is left for them
        out = hip.attn_window_step(qkv, torch.tensor([past], dtype=torch.int32, device=DEV), kc, vc, 1, sinks=sinks, rolling=rolling, pieces=pieces)
        v = qkv[:, 2 * D:].double()
        within(out, v, 2.0 ** -20 * v.abs() + 1e-6, f"past {past}")


def test_attn_window_step_far_slots():
    """Slots beyond 2^31 elements of a cache: only the last rows are visible (and written)."""
    hip = _hip()
    cap, Hkv, D = 2_200_000, 8, 128
    kc, vc = torch.empty(1, cap, Hkv, D, dtype=BF, device=DEV), torch.empty(1, cap, Hkv, D, dtype=BF, device=DEV)
    kc[:, -300:], vc[:, -300:] = rnd(1, 300, Hkv, D, seed=1), rnd(1, 300, Hkv, D, seed=2)
    kc[:, :4], vc[:, :4] = rnd(1, 4, Hkv, D, seed=3), rnd(1, 4, Hkv, D, seed=4)
    qkv = rnd(1, 24 * D)
    out = hip.attn_window_step(qkv, torch.tensor([cap - 1], dtype=torch.int32, device=DEV), kc, vc, 8, left=299, sinks=4)
    ks, vs = torch.cat([kc[:, :4], kc[:, -300:]], 1).contiguous(), torch.cat([vc[:, :4], vc[:, -300:]], 1).contiguous()
    ref = hip.attn_window_step(qkv, torch.tensor([303], dtype=torch.int32, device=DEV), ks, vs, 8, left=299, sinks=4)
    u = half_step(BF)
    within(out, ref.double(), 4 * u * ref.double().abs() + 4 * u * vs.double().abs().max().item(), "far")


def test_empty_batches_are_no_work():
    hip = _hip()
    from OATrans.model import window_attention as wa
    none = hip.seq_table([])
    q = rnd(5, 192)
    out = wa.window_attention(q, none, 1, 1, 64, longest=0)
    assert (out == 0).all() and out.shape == (5, 64)
    empty = rnd(0, 192)
    assert wa.window_attention(empty, none, 1, 1, 64, longest=0).shape == (0, 64)
    assert wa.window_attention(empty, hip.seq_table([0, 0]), 1, 1, 64, longest=0).shape == (0, 64)
    caches = torch.zeros(0, 9, 1, 64, dtype=BF, device=DEV)
    past = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert hip.attn_window_step(empty, past, caches, caches.clone(), 1).shape == (0, 64)
    hip.window_cache_fill(rnd(0, 64), rnd(0, 64), none, caches, caches.clone(), 0)
    rope = hip.RopeAxes((64,))
    assert hip.rope_axes(rnd(0, 64), torch.zeros(1, 1, dtype=torch.int32, device=DEV), rope, 1, 64).shape == (0, 64)


def test_step_pieces_are_read_fresh():
    """The pieces' sums pass between workgroups through memory that earlier calls used: every one of many calls with other data gives
    what a new workspace gives."""
    hip = _hip()
    B, cap, Hq, Hkv, D = 2, 6000, 8, 2, 128
    kc, vc = rnd(B, cap, Hkv, D, seed=1), rnd(B, cap, Hkv, D, seed=2)
    pieces = hip.window_step_workspace(B, Hq, Hkv, D)
    for k in range(12):
        past = torch.tensor([5999 - 311 * k, 400 * k], dtype=torch.int32, device=DEV)
        x = rnd(B, (Hq + 2 * Hkv) * D, seed=50 + k)
        assert torch.equal(hip.attn_window_step(x, past, kc, vc, Hq, pieces=pieces), hip.attn_window_step(x, past, kc, vc, Hq)), k


@pytest.mark.parametrize("cap,sinks,lens", [(40, 0, [40, 1]), (20, 4, [19, 20, 21, 100]), (16, 15, [3, 200]), (5, 9, [4, 5])])
def test_window_cache_fill(cap, sinks, lens):
    hip = _hip()
    Hkv, D = 3, 64
    M = sum(lens)
    k, v = rnd(M, Hkv * D, seed=1), rnd(M, Hkv * D + 8, seed=2)[:, :Hkv * D]
    kc, vc = torch.full((len(lens), cap, Hkv, D), 7.0, dtype=BF, device=DEV), torch.full((len(lens), Hkv, cap, D), 7.0, dtype=BF, device=DEV).transpose(1, 2)
    hip.window_cache_fill(k, v, hip.seq_table(lens), kc, vc, max(lens), sinks=sinks)
    at = 0
    for b, n in enumerate(lens):
        kr, vr = torch.full((cap, Hkv, D), 7.0, dtype=BF), torch.full((cap, Hkv, D), 7.0, dtype=BF)
        for t in range(n):
            s = t if t < min(sinks, cap) or cap <= sinks else sinks + (t - sinks) % (cap - sinks)
            if s < cap:
                kr[s], vr[s] = k[at + t].cpu().view(Hkv, D), v[at + t].cpu().view(Hkv, D)
        assert torch.equal(kc[b].cpu(), kr) and torch.equal(vc[b].cpu(), vr)
        at += n


# ---------------------------------------------------------------------------------------------- as they are used together
@pytest.mark.parametrize("window,slots,sinks,axes", [(None, 60, 0, 1), (12, None, 3, 1), (7, None, 0, 3)])
def test_prompt_then_steps_is_one_long_attention(window, slots, sinks, axes):
    """Prompts into a cache, then token by token: every step's output is the row that attention over the whole sequence has there."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    Hq, Hkv, D, lens, new = 4, 2, 64, [33, 5], 25
    rope = hip.RopeAxes((64,) if axes == 1 else (16, 24, 24))
    W = (Hq + 2 * Hkv) * D
    rows = [rnd(n + new, W, seed=n) for n in lens]
    spots = [torch.stack([torch.arange(n + new) // (1 if axes == 1 else 16), torch.arange(n + new) // 4 % 4, torch.arange(n + new) % 4], 1)[:, :axes].int() for n in lens]
    cache = wa.WindowCache(2, Hq, Hkv, D, window=window, sinks=sinks, slots=slots, rope=rope)
    left = -1 if window is None else window - 1
    out = cache.prompt(torch.cat([r[:n] for r, n in zip(rows, lens)]), hip.seq_table(lens), max(lens),
                       pos=torch.cat([s[:n] for s, n in zip(spots, lens)]).to(DEV).contiguous())
    got = [[out[:33]], [out[33:]]]
    for t in range(new):
        o = cache.step(torch.stack([r[n + t] for r, n in zip(rows, lens)]), pos=None if axes == 1 else torch.stack([s[n + t] for s, n in zip(spots, lens)]).to(DEV).contiguous())
        for b in range(2):
            got[b].append(o[b:b + 1])
    assert cache.past.tolist() == [n + new for n in lens]
    u = half_step(BF)
    for b, n in enumerate(lens):
        qk = hip.rope_axes(rows[b][:, :(Hq + Hkv) * D], spots[b].to(DEV).contiguous(), rope, Hq + Hkv, D)
        r = wo.attention(qk[:, :Hq * D], qk[:, Hq * D:], rows[b][:, (Hq + Hkv) * D:], [(0, n + new, 0, n + new)], Hq, Hkv, D, left, 0, sinks, D ** -0.5)
        within(torch.cat(got[b]), r["out"], u * r["out"].abs() + terms(r, "out", u), "together")


def test_captured_training_and_steps_replay():
    """Forward and backward, and a step, in HIP graphs: replayed with new inputs, other work between, against eager calls."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    Hq, Hkv, D, lens = 4, 2, 64, [100, 61]
    table, rope = hip.seq_table(lens), hip.RopeAxes((64,))
    pos = torch.cat([torch.arange(n) for n in lens])[:, None].int().to(DEV)
    M, W = sum(lens), (Hq + 2 * Hkv) * D
    qkv, dout = torch.zeros(M, W, dtype=BF, device=DEV, requires_grad=True), torch.zeros(M, Hq * D, dtype=BF, device=DEV)

    def train(x, d):
        out = wa.window_attention(x, table, Hq, Hkv, D, left=20, right=0, sinks=2, longest=100, rope=rope, pos=pos)
        return out.detach(), torch.autograd.grad(out, x, d)[0]
    x1 = torch.zeros(2, W, dtype=BF, device=DEV)
    kc, vc = rnd(2, 900, Hkv, D, seed=1), rnd(2, 900, Hkv, D, seed=2)
    past, pieces = torch.zeros(2, dtype=torch.int32, device=DEV), hip.window_step_workspace(2, Hq, Hkv, D)
    step = lambda x, p, ws: hip.attn_window_step(x, p, kc, vc, Hq, left=700, sinks=3, rope=rope, pos=p[:, None].contiguous(), pieces=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train(qkv, dout), step(x1, past, pieces)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = train(qkv, dout)
        one = step(x1, past, pieces)
    for k in range(4):
        with torch.no_grad():
            qkv.copy_(rnd(M, W, seed=20 + k))
            dout.copy_(rnd(M, Hq * D, seed=30 + k))
            x1.copy_(rnd(2, W, seed=40 + k))
            past.copy_(torch.tensor([899 - 200 * k, 10 + k], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = train(qkv.detach().clone().requires_grad_(True), dout)
        assert torch.equal(res[0], eager[0]) and torch.equal(res[1], eager[1])
        assert torch.equal(one, step(x1, past, hip.window_step_workspace(2, Hq, Hkv, D)))


def test_side_stream():
    """Calls go to the current stream."""
    hip = _hip()
    q = rnd(500, 64)
    table = hip.seq_table([500])
    ref = hip.attn_window_fwd(q, q, q, table, 1, 1, 64, 500, 500)
    side = torch.cuda.Stream()
    x = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x.copy_(q)
        out = hip.attn_window_fwd(x, x, x, table, 1, 1, 64, 500, 500)
    side.synchronize()
    assert torch.equal(out, ref)


def test_launch_tape_replays_the_operators():
    hip = _hip()
    q = rnd(300, 192)
    table, rope = hip.seq_table([300]), hip.RopeAxes((64,))
    pos = torch.arange(300, dtype=torch.int32, device=DEV)[:, None].contiguous()
    turned, out = torch.empty(300, 128, dtype=BF, device=DEV), torch.empty(300, 64, dtype=BF, device=DEV)

    def go():
        hip.rope_axes(q[:, :128], pos, rope, 2, 64, out=turned)
        hip.attn_window_fwd(turned[:, :64], turned[:, 64:], q[:, 128:], table, 1, 1, 64, 300, 300, 50, 0, 1, out=out)
    hip.tape_begin()
    go()
    tape = hip.tape_end()
    q.copy_(rnd(300, 192, seed=9))
    go()
    ref = out.clone()
    out.zero_()
    turned.zero_()
    hip.tape_replay(tape)
    assert torch.equal(out, ref)
    hip.tape_free(tape)


def test_reaches_beyond_32_bits_and_counts_beyond_the_rows():
    """A window, sinks or `longest` larger than anything there is the same as one that just covers it."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    M = 150
    qkv, seqs = rnd(M, 192), hip.seq_table([M])
    full = wa.window_attention(qkv, seqs, 1, 1, 64, left=-1, right=-1, longest=M)
    causal = wa.window_attention(qkv, seqs, 1, 1, 64, left=-1, right=0, longest=M)
    for far in (M, 2 ** 29 + 7, 2 ** 32, 2 ** 33 + 5):
        assert torch.equal(wa.window_attention(qkv, seqs, 1, 1, 64, left=far, right=far, longest=far), full)
        assert torch.equal(hip.attn_window_fwd(qkv[:, :64], qkv[:, 64:128], qkv[:, 128:], seqs, 1, 1, 64, M, M, left=far, right=0), causal)
        # (other tiles, another reference: each side rounds its weights and its output, u sum P |v| + u |out|)
        sunk = wa.window_attention(qkv, seqs, 1, 1, 64, left=3, right=0, sinks=far)
        within(sunk, causal.double(), 4 * half_step(BF) * (causal.double().abs() + qkv[:, 128:].double().abs().max()), "sinks")
    rope, none = hip.RopeAxes((64,)), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    empty = rnd(0, 192).requires_grad_()
    out = wa.window_attention(empty, hip.seq_table([0]), 1, 1, 64, rope=rope, pos=none)
    out.sum().backward()
    assert out.shape == (0, 64) and empty.grad.shape == (0, 192)
