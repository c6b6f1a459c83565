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
