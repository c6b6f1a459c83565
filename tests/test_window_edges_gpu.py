"""Calls of the windowed attention, its caches and rotary positions at the edges of what their documentation allows, on a real MI355X
against their definitions in 64 bits (oracle/window_oracle.py)."""
import math

import pytest
import torch

from oracle import window_oracle as wo
from tests.test_window_gpu import BF, DEV, HF, _hip, half_step, rnd, within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- a table that understates its longest count
@pytest.mark.parametrize("window,slots,sinks", [(None, 20, 0), (9, None, 2)])
def test_cache_and_attention_leave_out_the_same_sequences(window, slots, sinks):
    """A sequence with more tokens than `longest` is taken as empty: by the attention, the cache and the cache's counts alike."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    lens, D = [7, 13, 5], 64
    qkv, table = rnd(sum(lens), 3 * D, seed=2), hip.seq_table(lens)
    cache = wa.WindowCache(3, 1, 1, D, window=window, sinks=sinks, slots=slots)
    cache.k.fill_(7.0), cache.v.fill_(7.0)
    out = cache.prompt(qkv, table, 10)
    ok = wa.WindowCache(3, 1, 1, D, window=window, sinks=sinks, slots=slots)
    ok.k.fill_(7.0), ok.v.fill_(7.0)
    ref = ok.prompt(qkv, hip.seq_table([7, 0, 5], q_rows=(0, 7, 20)), 10)
    assert (out[7:20] == 0).all() and torch.equal(out, ref)
    assert torch.equal(cache.k, ok.k) and torch.equal(cache.v, ok.v) and (cache.k[1] == 7.0).all()
    assert cache.past.tolist() == ok.past.tolist() == [7, 0, 5]
    # the next token of the sequence that was left out is its first
    x = rnd(3, 3 * D, seed=3)
    assert torch.equal(cache.step(x)[1], x[1, 2 * D:]) and cache.past.tolist() == [8, 1, 6]


def test_counts_of_tables_that_do_not_fit_are_zero():
    hip = _hip()
    from OATrans.model import window_attention as wa
    qkv = rnd(30, 192)
    for bad in ((-1, 5, 0, 5), (28, 5, 28, 5), (0, 5, 26, 5), (0, 11, 0, 11), (0, -1, 0, 5), (2 ** 31 - 4, 5, 0, 5), (0, 5, 2 ** 31 - 4, 5)):
        cache = wa.WindowCache(2, 1, 1, 64, slots=12)
        table = torch.tensor([bad, (20, 6, 20, 6)], dtype=torch.int32, device=DEV)
        out = cache.prompt(qkv, table, 10)
        assert cache.past.tolist() == [0, 6] and (cache.k[0] == 0).all() and (cache.v[0] == 0).all() and (out[:20] == 0).all()
        assert torch.equal(cache.v[1, :6, 0], qkv[20:26, 128:]) and (cache.v[1, 6:] == 0).all()


# ---------------------------------------------------------------------------------------------- counts
def test_a_full_cache_stops_counting():
    """A plain cache without a slot left: its row is zero, the cache and the count stay; the others go on, and so does one that
    takes no part."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    cache = wa.WindowCache(4, 2, 1, 64, slots=6)
    cache.past.copy_(torch.tensor([4, 0, -1, 6], dtype=torch.int32))
    for t in range(4):
        held = cache.k.clone(), cache.v.clone()
        x = rnd(4, 4 * 64, seed=t)
        out = cache.step(x)
        assert cache.past.tolist() == [min(5 + t, 6), 1 + t, -1, 6]
        assert (out[2:] == 0).all() and (out[1] != 0).any() and (out[0] == 0).all() == (t >= 2)
        for c, h in zip((cache.k, cache.v), held):
            assert torch.equal(c[2:], h[2:]) and torch.equal(c[0], h[0]) == (t >= 2)
    rolling = wa.WindowCache(3, 1, 1, 64, window=4, sinks=1)
    rolling.past.copy_(torch.tensor([2 ** 31 - 1, 9, -5], dtype=torch.int32))
    rolling.step(rnd(3, 192))
    assert rolling.past.tolist() == [2 ** 31 - 1, 10, -5]              # (the largest count is not passed)


# ---------------------------------------------------------------------------------------------- rows without a result
@pytest.mark.parametrize("D,Hq,Hkv,longest,lens", [(64, 2, 1, 10, [7, 13, 5]), (128, 4, 2, 200, [200, 901, 1]), (64, 3, 3, 0, [4, 9]), (128, 1, 1, 3, [])])
@pytest.mark.parametrize("packed", [True, False])
def test_rows_of_a_sequence_that_is_left_out_are_zeros(D, Hq, Hkv, longest, lens, packed):
    """With packed=True the results are new memory that the kernels fill: also for a sequence that has more tokens than `longest`."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    M, W = max(30, sum(lens)) if not lens else sum(lens), (Hq + 2 * Hkv) * D
    qkv, dout, table = rnd(M, W, seed=5).requires_grad_(), rnd(M, Hq * D, seed=6), hip.seq_table(lens)

    def dirty():
        for width in (Hq * D, W):                                        # what the allocator hands out next
            for t in [torch.full((M, width), 7.0, dtype=BF, device=DEV) for _ in range(3)]:
                del t
    dirty()
    out = wa.window_attention(qkv, table, Hq, Hkv, D, 50, 0, 1, longest=longest, packed=packed)
    dirty()
    (g,) = torch.autograd.grad(out, qkv, dout)
    kept = [n if n <= longest else 0 for n in lens]
    starts = [sum(lens[:b]) for b in range(len(lens))]
    ref = wa.window_attention(qkv, hip.seq_table(kept, q_rows=starts), Hq, Hkv, D, 50, 0, 1, longest=longest)
    (gr,) = torch.autograd.grad(ref, qkv, dout)
    assert torch.equal(out, ref) and torch.equal(g, gr)
    own = torch.zeros(M, dtype=torch.bool, device=DEV)
    for at, n in zip(starts, kept):
        own[at:at + n] = True
    assert (out[~own] == 0).all() and (g[~own] == 0).all() and (out[own] != 0).any(1).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_what_is_not_a_number_shows(D, dtype):
    """A query or key that is not a number: the rows it belongs to say so, in out, in lse and in their gradient; lse = -inf is said by rows
    that see nothing only, and rows of other sequences are untouched."""
    hip = _hip()
    n, scale = 150, D ** -0.5
    table = hip.seq_table([n, 40])
    q, k, v, do = (rnd(n + 40, D, dtype=dtype, seed=s) for s in range(4))
    call = lambda q, k, v: (hip.attn_window_fwd(q, k, v, table, 1, 1, D, n, n, left=20, right=-3, sinks=2, lse=lse), lse)
    lse = torch.zeros(n + 40, 1, device=DEV)
    ok, ok_lse = (t.clone() for t in call(q, k, v))
    i = torch.arange(n, device=DEV)
    for name, at in (("q", 77), ("k", 90), ("k", 0)):
        bad = {"q": q.clone(), "k": k.clone()}
        bad[name][at, 5] = float("nan")
        out, l = call(bad["q"], bad["k"], v)
        sees = (i == at) if name == "q" else ((at >= i - 20) | (at < 2))       # no right edge
        assert out[:n][sees].isnan().all() and l[:n, 0][sees].isnan().all()
        assert torch.equal(out[n:], ok[n:]) and torch.equal(l[n:], ok_lse[n:])
        assert torch.equal(out[:n][~sees], ok[:n][~sees]) and torch.equal(l[:n][~sees], ok_lse[:n][~sees])
        g = hip.attn_window_bwd(bad["q"], bad["k"], v, out, l, do, table, 1, 1, D, n, n, left=20, right=-3, sinks=2)
        assert g[0][:n][sees].isnan().all() and not any(t[n:].isnan().any() for t in g)


# ---------------------------------------------------------------------------------------------- bounds that count every rounding once
def tight(r, name, dtype, other):
    """u |value| for its one rounding, u |term| for the 16-bit terms (worst case, or 6 deviations of independent ones; see
    tests/test_window_gpu.py), 2^-14 of the terms for 32-bit sums, exponentials and the log-sum-exp.  What is below the type's normal
    numbers is rounded to a multiple of its least one: off by half of that, s, for the result, and for every 16-bit probability or its
    gradient s times what it multiplies - `other` is the sum of their sizes."""
    u, s = half_step(dtype), torch.finfo(dtype).smallest_normal * half_step(dtype)
    return u * r[name].abs() + torch.minimum(u * r[name + "_abs"], 6 * u * r[name + "_sq"]) + 2.0 ** -14 * r[name + "_abs"] + s + s * other


def _check_attention(q, k, v, do, seqs, Hq, Hkv, D, left, right, sinks, scale):
    """out, lse and the gradients of rows that all belong to a sequence, within `tight`"""
    hip = _hip()
    dtype = q.dtype
    table = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    mq, mk, G = max(s[1] for s in seqs), max(s[3] for s in seqs), Hq // Hkv
    lse = torch.empty(q.shape[0], Hq, device=DEV)
    out = hip.attn_window_fwd(q, k, v, table, Hq, Hkv, D, mq, mk, left, right, sinks, scale, lse=lse)
    dq, dk, dv = hip.attn_window_bwd(q, k, v, out, lse, do, table, Hq, Hkv, D, mq, mk, left, right, sinks, scale)
    r = wo.attention(q, k, v, seqs, Hq, Hkv, D, left, right, sinks, scale, dout=do, out=out)
    Q, K, V, dO = (t.double().abs() for t in (q, k, v, do))
    seen_K, seen_V, seen_Q, seen_dO = torch.zeros_like(Q), torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(K)
    for q0, nq, k0, nk in seqs:
        see = wo.visible(nq, nk, left, right, sinks, DEV).double()
        for h in range(Hq):
            a, b = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            seen_K[q0:q0 + nq, a] = see @ K[k0:k0 + nk, b]
            seen_V[q0:q0 + nq, a] = see @ V[k0:k0 + nk, b]
            seen_Q[k0:k0 + nk, b] += see.t() @ Q[q0:q0 + nq, a]
            seen_dO[k0:k0 + nk, b] += see.t() @ dO[q0:q0 + nq, a]
    some = r["lse"] > -math.inf
    within(lse[some], r["lse"][some], 2.0 ** -17 * (4 + r["lse"][some].abs()), "lse")
    assert (lse[~some] == -math.inf).all()
    # (what is beyond the type's largest number by more than its tolerance is inf of its sign)
    top = torch.finfo(dtype).max

    def within_type(got, ref, tol, what):
        inf = ref.abs() - tol > top
        assert (got[inf].double() == ref[inf].sign() * math.inf).all(), what
        near = ~inf & (ref.abs() + tol >= top)
        within(got[~inf & ~near], ref[~inf & ~near], tol[~inf & ~near], what)
    # 1.01 *_off: delta from the rounded out, and 32-bit rounding of the terms that cancel in the probabilities' gradient
    within_type(out, r["out"], tight(r, "out", dtype, seen_V), "out")
    within_type(dq, r["dq"], tight(r, "dq", dtype, scale * seen_K) + 1.01 * r["dq_off"], "dq")
    within_type(dk, r["dk"], tight(r, "dk", dtype, scale * seen_Q) + 1.01 * r["dk_off"], "dk")
    within_type(dv, r["dv"], tight(r, "dv", dtype, seen_dO), "dv")
    return r


@pytest.mark.parametrize("size", [1.0, 1e-3])
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("lens,Hq,Hkv,D,left,right,sinks", [
    ([2300], 1, 1, 64, 90, 0, 130), ([1100], 1, 1, 64, -1, -1, 0), ([1500], 1, 1, 64, 100, 0, 600), ([520, 130, 90], 2, 1, 128, 100, 30, 33),
    ([700], 8, 1, 64, 64, 0, 2), ([1300, 700], 4, 1, 128, 100, 0, 40), ([1, 40, 1500], 2, 2, 128, -1, 0, 0)])
def test_gradients_of_small_terms(lens, Hq, Hkv, D, left, right, sinks, dtype, size):
    """Probabilities of a thousandth and less, and their gradients for a dout of 1 and 1 / 1000: in fp16 most of the terms are below its
    normal numbers."""
    M, starts = sum(lens), [sum(lens[:b]) for b in range(len(lens))]
    seqs = [(a, n, a, n) for a, n in zip(starts, lens)]
    q, k, v, do = rnd(M, Hq * D, dtype=dtype, seed=1), rnd(M, Hkv * D, dtype=dtype, seed=2), rnd(M, Hkv * D, dtype=dtype, seed=3), rnd(M, Hq * D, dtype=dtype, seed=4, scale=size)
    _check_attention(q, k, v, do, seqs, Hq, Hkv, D, left, right, sinks, 0.9 / math.sqrt(D))


# ---------------------------------------------------------------------------------------------- scores that grow along the keys
def _moves(s, left, right, sinks):
    """How often the forward kernel's reference score moves by a factor between 2^-40 and 1/2, by its rule on 64-bit scores of one head: the
    maximum of the first 32 keys that a row sees, until 16 terms of a step (keys 8 (r >> 2) + 4 half + (r & 3) of it) sum to over 2^10 for
    some row of 32."""
    n = s.shape[0]
    see = wo.visible(n, n, left, right, sinks)
    keys = torch.tensor([[8 * (r >> 2) + 4 * half + (r & 3) for r in range(16)] for half in range(2)])
    ref = torch.full((n,), -math.inf, dtype=torch.float64)
    count = 0
    for j in range(0, n, 32):
        part = torch.full((n, 32), -math.inf, dtype=torch.float64)
        part[:, :min(32, n - j)] = s[:, j:j + 32].masked_fill(~see[:, j:j + 32], -math.inf)
        top = part.amax(1)
        ref = torch.where((ref == -math.inf) & (top > -math.inf), top, ref)
        term = torch.where(part > -math.inf, ((part - ref.clamp_min(-1e300)[:, None]) * math.log2(math.e)).clamp(max=1000).exp2(), torch.zeros_like(part))
        over = (term[:, keys].sum(-1) > 1024).any(1)
        for w in range(0, n, 32):
            if over[w:w + 32].any():
                new = torch.maximum(ref[w:w + 32], top[w:w + 32])
                f = ((ref[w:w + 32] - new) * math.log2(math.e))
                count += int(((f < -1) & (f > -40)).sum())
                ref[w:w + 32] = new
    return count


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,Hq,Hkv,D,left,right,sinks,slope,period,least", [
    (300, 1, 1, 64, -1, 0, 0, 9.0, 300, 400), (300, 2, 1, 128, -1, -1, 0, 7.0, 300, 400), (700, 2, 2, 64, 120, 0, 0, 11.0, 170, 400),
    (640, 4, 1, 128, 150, 0, 3, 10.0, 190, 400), (600, 2, 1, 64, 100, 20, 130, 8.0, 150, 400), (520, 1, 1, 128, 200, 60, 70, 6.0, 240, 300),
    (450, 1, 1, 64, -1, 0, 200, 8.0, 200, 300)])
def test_scores_that_grow_along_the_keys(n, Hq, Hkv, D, left, right, sinks, slope, period, least, dtype):
    """Scores that rise by 6 to 11 (natural units) per 64 keys, in a saw: the reference of a row moves, by factors that leave weight to what
    came before, more than once in many rows - behind sinks, at masked edges, in rows that begin later than their neighbours."""
    scale = D ** -0.5
    j = torch.arange(n, dtype=torch.float64)
    rise = slope * (j % period) / 64
    # q and k share a direction of sixteen values: 2 * rise / 2 / (16 * scale) * 16 * scale = rise, on top of noise
    q, k, v, do = (rnd(n, h * D, dtype=dtype, seed=s, scale=0.5) for s, h in ((1, Hq), (2, Hkv), (3, Hkv), (4, Hq)))
    q.view(n, Hq, D)[..., :16] = 1.0
    k.view(n, Hkv, D)[..., :16] = (rise / (16 * scale)).to(dtype).to(DEV)[:, None, None]
    moved = sum(_moves((q.view(n, Hq, D)[:, h].double() @ k.view(n, Hkv, D)[:, h // (Hq // Hkv)].double().t() * scale).cpu(), left, right, sinks)
                for h in range(Hq))
    assert moved >= least, moved
    r = _check_attention(q, k, v, do, [(0, n, 0, n)], Hq, Hkv, D, left, right, sinks, scale)
    assert r["lse"].max() > 15


def test_step_shows_what_is_not_a_number():
    """A query, or a key in the cache, that is not a number: in one piece and in many."""
    hip = _hip()
    for cap, at in ((300, 17), (5000, 4100), (5000, 3)):
        kc, vc, x = rnd(2, cap, 1, 64, seed=1), rnd(2, cap, 1, 64, seed=2), rnd(2, 192, seed=3)
        past = torch.full((2,), cap - 1, dtype=torch.int32, device=DEV)
        ok = hip.attn_window_step(x, past, kc, vc, 1)
        bad = kc.clone()
        bad[0, at, 0, 9] = float("nan")
        out = hip.attn_window_step(x, past, bad, vc, 1)
        assert out[0].isnan().all() and torch.equal(out[1], ok[1])
        y = x.clone()
        y[1, 3] = float("nan")
        out = hip.attn_window_step(y, past, kc, vc, 1)
        assert out[1].isnan().all() and torch.equal(out[0], ok[0])


# ---------------------------------------------------------------------------------------------- the upper end of fp16
@pytest.mark.parametrize("D,Hq,Hkv,n,sinks", [(64, 2, 1, 300, 0), (128, 2, 2, 300, 0), (64, 1, 1, 1500, 2), (128, 4, 2, 1500, 2)])
def test_fp16_gradients_up_to_the_limit_and_beyond(D, Hq, Hkv, n, sinks):
    """Up to |dS| = 6e4 the gradients are right; beyond 65520 the query's dq and the key's dk are inf or nan, everything else is what it is
    without that term's row."""
    hip = _hip()
    scale = D ** -0.5
    q, k, v = rnd(n, Hq * D, dtype=HF, seed=1, scale=0.25), rnd(n, Hkv * D, dtype=HF, seed=2, scale=0.25), rnd(n, Hkv * D, dtype=HF, seed=3, scale=2.0)
    do = rnd(n, Hq * D, dtype=HF, seed=4)
    seqs = [(0, n, 0, n)]

    def terms_of_scores():
        Q, K, V, O = (t.double().view(n, -1, D).transpose(0, 1) for t in (q, k.repeat(1, 1), v, do))
        K, V = (t.repeat_interleave(Hq // Hkv, 0) for t in (K, V))
        see = wo.visible(n, n, 2, 0, sinks, DEV)
        P = torch.softmax((Q @ K.transpose(1, 2).contiguous() * scale).masked_fill(~see, -math.inf), 2)
        dP = O @ V.transpose(1, 2).contiguous()
        return P * (dP - (P * dP).sum(2, keepdim=True))
    top = terms_of_scores().abs().max().item()
    do = (do.double() * (6.0e4 / top)).to(HF)
    assert do.isfinite().all() and 5.5e4 < terms_of_scores().abs().max().item() < 6.4e4
    _check_attention(q, k, v, do, seqs, Hq, Hkv, D, 2, 0, sinks, scale)
    # one query's gradient times four
    table, at = hip.seq_table([n]), int(terms_of_scores().abs().amax(2)[0].argmax())
    lse = torch.empty(n, Hq, device=DEV)
    out = hip.attn_window_fwd(q, k, v, table, Hq, Hkv, D, n, n, 2, 0, sinks, scale, lse=lse)
    ok = hip.attn_window_bwd(q, k, v, out, lse, do, table, Hq, Hkv, D, n, n, 2, 0, sinks, scale)
    do[at, :D] = (do[at, :D].double() * 4).clamp(-6.5e4, 6.5e4).to(HF)
    over = terms_of_scores().abs() > 65520                              # [Hq, n, n]
    got = hip.attn_window_bwd(q, k, v, out, lse, do, table, Hq, Hkv, D, n, n, 2, 0, sinks, scale)
    rows = over.any(2).t().repeat_interleave(D, 1)
    keys = over.view(Hkv, -1, n, n).any(1).any(1).t().repeat_interleave(D, 1)
    assert over.any() and not got[0][rows].isfinite().any() and not got[1][keys].isfinite().any()
    far = torch.ones(n, dtype=torch.bool, device=DEV)                    # keys that the query does not see
    far[:sinks], far[at - 2:at + 1] = False, False
    assert torch.equal(got[2][far], ok[2][far]) and got[0][~rows].isfinite().all() and got[1][~keys & far[:, None]].isfinite().all()
    other = torch.ones(n, dtype=torch.bool, device=DEV)
    other[at] = False
    assert torch.equal(got[0][other], ok[0][other])


# ---------------------------------------------------------------------------------------------- a cache as a program uses it
@pytest.mark.parametrize("window,slots,sinks", [(None, 40, 0), (6, None, 2)])
def test_captured_prompts_and_steps_replay(window, slots, sinks):
    """A prompt, and a step with its count, in HIP graphs of their own: replayed with new inputs, eager work between, against eager calls."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    Hq, Hkv, D, lens = 4, 2, 64, [9, 17, 1]
    W, M, rope = (Hq + 2 * Hkv) * D, sum(lens), hip.RopeAxes((64,))
    pos, table = torch.cat([torch.arange(n) for n in lens])[:, None].int().to(DEV), hip.seq_table(lens)
    ours, other = (wa.WindowCache(3, Hq, Hkv, D, window=window, sinks=sinks, slots=slots, rope=rope) for _ in range(2))
    qkv, x = torch.zeros(M, W, dtype=BF, device=DEV), torch.zeros(3, W, dtype=BF, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            ours.prompt(qkv, table, max(lens), pos=pos), ours.step(x)
    torch.cuda.current_stream().wait_stream(side)
    first, then = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        read = ours.prompt(qkv, table, max(lens), pos=pos)
    with torch.cuda.graph(then):
        said = ours.step(x)
    for k in range(3):
        qkv.copy_(rnd(M, W, seed=60 + k))
        first.replay()
        assert torch.equal(read, other.prompt(qkv, table, max(lens), pos=pos)) and ours.past.tolist() == lens
        for t in range(30):
            x.copy_(rnd(3, W, seed=100 * k + t))
            then.replay()
            assert torch.equal(said, other.step(x)), (k, t)
        assert torch.equal(ours.past, other.past) and torch.equal(ours.k, other.k) and torch.equal(ours.v, other.v)
        full = [min(n + 30, slots) if slots else n + 30 for n in lens]
        assert ours.past.tolist() == full


def test_a_prompt_without_its_longest_count():
    hip = _hip()
    from OATrans.model import window_attention as wa
    lens, qkv = [5, 12, 3], rnd(20, 192, seed=1)
    a, b = wa.WindowCache(3, 1, 1, 64, slots=20), wa.WindowCache(3, 1, 1, 64, slots=20)
    assert torch.equal(a.prompt(qkv, hip.seq_table(lens)), b.prompt(qkv, hip.seq_table(lens), 12))
    assert a.past.tolist() == b.past.tolist() == lens and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_a_sequence_that_is_left_out_does_not_touch_its_neighbours():
    """A padded batch whose table claims a row too many: that sequence is left out, the next one, whose first row it claims, is not harmed."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    L, D = 300, 64
    qkv, dout = rnd(4 * L, 3 * D, seed=1).requires_grad_(), rnd(4 * L, D, seed=2)
    lens = [L, L + 1, L, 40]
    table, ok = hip.seq_table(lens, q_rows=range(0, 4 * L, L)), hip.seq_table([L, 0, L, 40], q_rows=range(0, 4 * L, L))
    for _ in range(20):
        out = wa.window_attention(qkv, table, 1, 1, D, longest=L)
        ref = wa.window_attention(qkv, ok, 1, 1, D, longest=L)
        assert torch.equal(out, ref)
        assert torch.equal(torch.autograd.grad(out, qkv, dout)[0], torch.autograd.grad(ref, qkv, dout)[0])
