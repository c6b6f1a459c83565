"""Refusals of the windowed attention's entry points, each by its own message, and the caches' checks: no GPU is needed."""
import ctypes

import pytest
import torch

LL = ctypes.c_longlong


def _hip():
    from OATrans.ops import hip
    hip.lib()
    return hip


def _refused(hip, rc, text):
    assert rc < 0 and text in hip.lib().oat_last_error(), hip.lib().oat_last_error()


def test_counts_refusals():
    hip = _hip()
    counts = lambda past=4096, seqs=4096, B=1, rows=10, longest=10: hip.lib().oat_window_cache_counts(past, seqs, B, rows, longest, None)
    for change in (dict(B=-1), dict(rows=-1), dict(longest=-1)):
        _refused(hip, counts(**change), b"negative")
    for change in (dict(past=None), dict(seqs=None), dict(seqs=4100)):
        _refused(hip, counts(**change), b"missing")
    assert counts(B=0) == 0
    past, seqs = torch.zeros(2, dtype=torch.int32), hip.seq_table([1, 2], device="cpu")
    for p, s, rows, longest, text in ((past.long(), seqs, 3, 2, "past must"), (past[:1], seqs, 3, 2, "seqs must"), (past, seqs.long(), 3, 2, "seqs must"),
                                      (past, seqs, -1, 2, "rows"), (past, seqs, 3, 2 ** 30, "largest"), (past, seqs, 3, 2, "no CPU path")):
        with pytest.raises(hip.OatError, match=text):
            hip.window_cache_counts(p, s, rows, longest)


def test_advance_refusals():
    hip = _hip()
    _refused(hip, hip.lib().oat_window_cache_advance(4096, -1, 8, None), b"negative")
    _refused(hip, hip.lib().oat_window_cache_advance(None, 1, 8, None), b"missing")
    assert hip.lib().oat_window_cache_advance(None, 0, 8, None) == 0
    past = torch.zeros(2, dtype=torch.int32)
    for p, slots, text in ((past.long(), 8, "past must"), (past[:, None], 8, "past must"), (past, 0, "slots"), (past, 2 ** 31, "slots"), (past, 8, "no CPU path")):
        with pytest.raises(hip.OatError, match=text):
            hip.window_cache_advance(p, slots)


def test_forward_mode_gradients_are_refused():
    """The operators have gradients in reverse mode only: a tangent is refused, with and without a reverse-mode gradient beside it."""
    from torch.autograd import forward_ad
    hip = _hip()
    from OATrans.model import window_attention as wa
    seqs, rope, pos = hip.seq_table([4], device="cpu"), hip.RopeAxes((64,)), torch.zeros(4, 1, dtype=torch.int32)
    cache = object.__new__(wa.WindowCache)                             # (the refusal comes before anything that needs a GPU)
    cache.heads = cache.kv_heads = 1
    cache.head_dim, cache.left, cache.sinks, cache.rope, cache.rolling = 64, 9, 0, None, True
    cache.past = torch.zeros(4, dtype=torch.int32)
    cache.k = cache.v = torch.zeros(4, 10, 1, 64, dtype=torch.bfloat16)
    cache.pieces = torch.zeros(4)
    for leaf in (torch.zeros(4, 192, dtype=torch.bfloat16), torch.zeros(4, 192, dtype=torch.bfloat16, requires_grad=True)):
        calls = [lambda x: wa.window_attention(x, seqs, 1, 1, 64), lambda x: wa.window_attention(x, seqs, 1, 1, 64, rope=rope, pos=pos),
                 lambda x: wa.rope_axes(x, pos, rope, 3, 64), lambda x: cache.step(x), lambda x: cache.prompt(x, seqs, 4)]
        for call in calls:
            with forward_ad.dual_level():
                with pytest.raises(hip.OatError, match="forward mode"):
                    call(forward_ad.make_dual(leaf, torch.ones_like(leaf)))
                with pytest.raises(hip.OatError) as refused:           # no tangent: what is refused here is the missing GPU (or its buffers)
                    call(leaf)
                assert "forward mode" not in str(refused.value)


# ---------------------------------------------------------------------------------------------- caches whose slots share memory
@pytest.mark.parametrize("k,v,ok", [
    ((1024, 64, 64), (1024, 64, 64), False),                           # two heads in one place
    ((0, 128, 64), (4096, 128, 64), False), ((4096, 128, 64), (0, 128, 64), False),     # one cache for all sequences (expand)
    ((4096, 0, 64), (4096, 128, 64), False), ((1920, 128, 64), (2048, 128, 64), False), ((4096, 64, 128), (4096, 128, 64), False),
    ((4096, 120, 64), (4096, 128, 64), False), ((4096, 128, 56), (4096, 128, 64), False),
    ((2048, 128, 64), (2048, 128, 64), True), ((2048, 64, 1024), (2048, 128, 64), True), ((64, 256, 128), (128, 256, 64), True),
    ((8192, 136, 72), (2048, 64, 1024), True)])
def test_caches_whose_slots_share_memory_are_refused(k, v, ok):
    """The step and the fill write the caches: no two slots (2 sequences, 16 slots, 2 heads of 64) may lie in one place."""
    hip = _hip()
    lib, st = hip.lib(), (LL * 6)(*k, *v)
    # taken as far as the next refusal: the missing counts of the step, the misaligned rows of the fill
    rc = lib.oat_attn_window_step(4096, 384, None, 4096, 4096, st, 16, 4096, 128, 2, 2, 2, 64, 0, -1, 0, 0, 0.125, None, None, 4096, 16, None)
    _refused(hip, rc, b"needed" if ok else b"share")
    _refused(hip, lib.oat_window_cache_fill(4097, 128, 4096, 128, 4096, 2, 10, 10, 4096, 4096, st, 16, 2, 64, 0, None), b"16-byte" if ok else b"share")


def test_strides_of_a_single_sequence_slot_or_head_do_not_matter():
    """torch gives a dimension of one any stride."""
    hip = _hip()
    for B, cap, Hkv, st in ((1, 16, 2, (0, 128, 64)), (2, 1, 2, (128, 0, 64)), (2, 16, 1, (1024, 64, 0)), (1, 1, 1, (0, 0, 0))):
        rc = hip.lib().oat_attn_window_step(4096, 64 * 3 * Hkv, None, 4096, 4096, (LL * 6)(*st, *st), cap, 4096, 128, B, Hkv, Hkv, 64, 0, -1, 0, 0, 0.125,
                                            None, None, 4096, 16, None)
        _refused(hip, rc, b"needed")


# ---------------------------------------------------------------------------------------------- what the binding checks, by message
def _calls():
    """(what it is, call, message): CPU tensors throughout, so a check that is not made ends in 'no CPU path' instead of its own message"""
    hip = _hip()
    from OATrans.model import window_attention as wa
    BF, i32 = torch.bfloat16, torch.int32
    rope = hip.RopeAxes((16, 24, 24))
    x, pos = torch.zeros(4, 64), torch.zeros(4, 3, dtype=i32)
    R = lambda **c: (lambda a: hip.rope_axes(a["x"], a["pos"], rope, a["heads"], a["dim"], out=a["out"]))({**dict(x=x, pos=pos, heads=1, dim=64, out=None), **c})
    yield "rope", lambda: R(), "no CPU path"
    yield "rope: 64-bit x", lambda: R(x=x.double()), "must be bf16, fp16 or fp32"
    yield "rope: x of one dimension", lambda: R(x=x[0]), "rope_axes: x: need"
    yield "rope: narrow x", lambda: R(heads=2), "rope_axes: x: need"
    yield "rope: stepped columns", lambda: R(x=x[:, ::2], dim=32), "rope_axes: x: need"
    yield "rope: 64-bit pos", lambda: R(pos=pos.long()), "pos must be"
    yield "rope: two axes", lambda: R(pos=pos[:, :2]), "pos must be"
    yield "rope: pos not contiguous", lambda: R(pos=torch.zeros(4, 6, dtype=i32)[:, ::2]), "pos must be"
    yield "rope: pos elsewhere", lambda: R(pos=pos.to("meta")), "pos must be"
    yield "rope: short out", lambda: R(out=torch.zeros(3, 64)), "number of rows"
    yield "rope: out of another type", lambda: R(out=torch.zeros(4, 64, dtype=BF)), "rope_axes: out: need"
    yield "rope layer: width", lambda: wa.rope_axes(x, pos, rope, 2, 64), r"\[M, heads \* head_dim\]"
    b, seqs = torch.zeros(4, 64, dtype=BF), hip.seq_table([4], device="cpu")
    lse = torch.zeros(4, 1)
    base = dict(q=b, k=b, v=b, seqs=seqs, heads=1, kv=1, D=64, mq=4, mk=4)
    F = lambda out=None, lse=None, **c: (lambda a: hip.attn_window_fwd(*a.values(), out=out, lse=lse))({**base, **c})
    yield "forward", lambda: F(), "no CPU path"
    for name, change, text in (("32 bits", dict(q=x, k=x, v=x), "bf16 or fp16"), ("narrow q", dict(heads=2), "attn_window_fwd: q: need"), ("narrow k", dict(kv=2), "attn_window_fwd: k: need"),
                               ("k of another type", dict(k=b.half()), "attn_window_fwd: k: need"), ("v of another type", dict(v=b.half()), "attn_window_fwd: v: need"),
                               ("v elsewhere", dict(v=b.to("meta")), "attn_window_fwd: v: need"), ("stepped q", dict(q=torch.zeros(4, 128, dtype=BF)[:, ::2]), "attn_window_fwd: q: need"),
                               ("rows of k", dict(k=b[:3]), "different numbers of rows"), ("rows of v", dict(v=b[:3]), "different numbers of rows"), ("64-bit seqs", dict(seqs=seqs.long()), "seqs must be"),
                               ("seqs of three", dict(seqs=seqs[:, :3].contiguous()), "seqs must be"), ("seqs not contiguous", dict(seqs=torch.zeros(1, 8, dtype=i32)[:, ::2]), "seqs must be"),
                               ("seqs elsewhere", dict(seqs=seqs.to("meta")), "seqs must be"), ("negative count", dict(mq=-1), "largest counts"), ("large count", dict(mk=2 ** 29 + 1), "largest counts")):
        yield "forward: " + name, lambda change=change: F(**change), text
    yield "forward: lse's shape", lambda: F(lse=torch.zeros(4, 2)), "lse must be"
    yield "forward: lse's type", lambda: F(lse=lse.double()), "lse must be"
    yield "forward: lse's order", lambda: hip.attn_window_fwd(torch.zeros(4, 128, dtype=BF), b, b, seqs, 2, 1, 64, 4, 4, lse=torch.zeros(2, 4).t()), "lse must be"
    yield "forward: short out", lambda: F(out=b[:3]), "number of rows than q"
    yield "forward: out's type", lambda: F(out=x), "attn_window_fwd: out: need"
    G = lambda **c: (lambda a: hip.attn_window_bwd(a["q"], a["k"], a["v"], a["out"], a["lse"], a["dout"], seqs, 1, 1, 64, 4, 4, dq=a["dq"], dk=a["dk"], dv=a["dv"], workspace=a["ws"]))(
        {**base, **dict(out=b, lse=lse, dout=b, dq=None, dk=None, dv=None, ws=None), **c})
    yield "backward", lambda: G(), "no CPU path"
    for name, change, text in (("out's type", dict(out=x), "attn_window_bwd: out: need"), ("dout's type", dict(dout=x), "attn_window_bwd: dout: need"), ("short dout", dict(dout=b[:3]), "as many rows as q"),
                               ("short out", dict(out=b[:3]), "as many rows as q"), ("lse's shape", dict(lse=torch.zeros(4, 2)), "lse must be"), ("dq's type", dict(dq=x), "attn_window_bwd: dq: need"),
                               ("narrow dk", dict(dk=b[:, :32]), "attn_window_bwd: dk: need"), ("dv elsewhere", dict(dv=b.to("meta")), "attn_window_bwd: dv: need"), ("short dq", dict(dq=b[:3]), "as many rows as q, k, v"),
                               ("short dv", dict(dv=b[:3]), "as many rows as q, k, v"), ("workspace elsewhere", dict(ws=lse.to("meta")), "workspace must be"),
                               ("stepped workspace", dict(ws=torch.zeros(64)[::2]), "workspace must be")):
        yield "backward: " + name, lambda change=change: G(**change), text
    c, past, row, ws = torch.zeros(4, 8, 1, 64, dtype=BF), torch.zeros(4, dtype=i32), torch.zeros(4, 192, dtype=BF), torch.zeros(4)
    S = lambda **o: (lambda a: hip.attn_window_step(a["qkv"], a["past"], a["k"], a["v"], a["heads"], rope=a["rope"], pos=a["pos"], pieces=a["ws"], out=a["out"]))(
        {**dict(qkv=row, past=past, k=c, v=c, heads=1, rope=None, pos=None, ws=ws, out=None), **o})
    yield "step", lambda: S(), "no CPU path"
    for name, change, text in (("64-bit past", dict(past=past.long()), "past must be"), ("short past", dict(past=past[:3]), "past must be"), ("past elsewhere", dict(past=past.to("meta")), "past must be"),
                               ("stepped past", dict(past=torch.zeros(8, dtype=i32)[::2]), "past must be"), ("short qkv", dict(qkv=row[:3]), "one row of qkv"), ("narrow qkv", dict(heads=2), "attn_window_step: qkv: need"),
                               ("qkv's type", dict(qkv=row.half()), "differ in type or device"), ("qkv elsewhere", dict(qkv=row.to("meta")), "differ in type or device"), ("caches that differ", dict(v=c[:, :4]), "both alike"),
                               ("32-bit caches", dict(k=c.float(), v=c.float()), "both alike"), ("caches of three dimensions", dict(k=c[0], v=c[0]), "both alike"), ("stepped caches", dict(k=c[..., ::2], v=c[..., ::2]), "both alike"),
                               ("no pos", dict(rope=rope), "pos must be"), ("short pos", dict(rope=rope, pos=pos[:3]), "pos must be"), ("64-bit pos", dict(rope=rope, pos=pos.long()), "pos must be"),
                               ("stepped workspace", dict(ws=torch.zeros(64)[::2]), "pieces must be"), ("short out", dict(out=b[:3]), "one row of out"), ("out's type", dict(out=x), "attn_window_step: out: need")):
        yield "step: " + name, lambda change=change: S(**change), text
    seqs4 = hip.seq_table([1, 1, 1, 1], device="cpu")
    L = lambda **o: (lambda a: hip.window_cache_fill(a["k"], a["v"], a["seqs"], a["kc"], a["vc"], a["most"]))({**dict(k=b, v=b, seqs=seqs4, kc=c, vc=c, most=4), **o})
    yield "fill", lambda: L(), "no CPU path"
    for name, change, text in (("B", dict(seqs=seqs), "seqs must be"), ("64-bit seqs", dict(seqs=seqs4.long()), "seqs must be"), ("k's type", dict(k=b.half()), "window_cache_fill: k: need"),
                               ("narrow v", dict(v=b[:, :32]), "window_cache_fill: v: need"), ("rows", dict(v=b[:3]), "different numbers"), ("count", dict(most=-1), "largest count"), ("large count", dict(most=2 ** 30), "largest count")):
        yield "fill: " + name, lambda change=change: L(**change), text
    W = lambda **o: (lambda a: wa.window_attention(a.pop("qkv"), a.pop("seqs"), a.pop("heads"), a.pop("kv"), a.pop("D"), **a))({**dict(qkv=row, seqs=seqs, heads=1, kv=1, D=64), **o})
    yield "layer", lambda: W(), "no CPU path"
    yield "layer: gradient", lambda: W(qkv=row.clone().requires_grad_()), "no CPU path"
    for name, change, text in (("width", dict(D=128), r"qkv must be \[M, 384\]"), ("32 bits", dict(qkv=row.float()), "bf16 or fp16"), ("stepped columns", dict(qkv=torch.zeros(4, 384, dtype=BF)[:, ::2]), "unit column stride"),
                               ("rope alone", dict(rope=rope), "belong together"), ("pos alone", dict(pos=pos), "belong together"), ("64-bit pos", dict(rope=rope, pos=pos.long()), "pos must be"),
                               ("64-bit seqs", dict(seqs=seqs.long()), "seqs must be"), ("right with a cache", dict(right=1, cache=(c[:1], c[:1])), "causal attention"),
                               ("few slots", dict(longest=9, qkv=torch.zeros(9, 192, dtype=BF), cache=(c[:1], c[:1])), "slot for every token"),
                               ("gradient with a cache", dict(qkv=row.clone().requires_grad_(), cache=(c[:1], c[:1])), "without a gradient"), ("cache of another batch", dict(cache=(c, c)), r"caches must be \[1, slots"),
                               ("cache's type", dict(cache=(c[:1].half(), c[:1].half())), "caches must be"), ("caches that differ", dict(cache=(c[:1], c[:1, :4])), "both alike")):
        yield "layer: " + name, lambda change=change: W(**change), text
    yield "cache: window and slots", lambda: wa.WindowCache(1, 1, 1, 64, window=4, slots=4, device="cpu"), "either a window"
    yield "cache: neither", lambda: wa.WindowCache(1, 1, 1, 64, device="cpu"), "either a window"
    yield "cache: no window", lambda: wa.WindowCache(1, 1, 1, 64, window=0, device="cpu"), "either a window"
    yield "cache: no slots", lambda: wa.WindowCache(1, 1, 1, 64, slots=0, device="cpu"), "either a window"
    yield "cache: sinks", lambda: wa.WindowCache(1, 1, 1, 64, window=4, sinks=-1, device="cpu"), "sinks"
    yield "cache: heads", lambda: wa.WindowCache(1, 3, 2, 64, window=4, device="cpu"), "multiple"
    yield "cache: head_dim", lambda: wa.WindowCache(1, 2, 2, 32, window=4, device="cpu"), "64 or 128"
    yield "cache: type", lambda: wa.WindowCache(1, 2, 2, 64, window=4, dtype=torch.float32, device="cpu"), "bf16 or fp16"
    yield "table: lengths", lambda: hip.seq_table([1, 2], [1]), "one count"
    yield "table: negative", lambda: hip.seq_table([1, -1]), "one count"
    yield "table: rows", lambda: hip.seq_table([1, 2], q_rows=(0,)), "first row"


def test_every_check_of_the_binding_says_what_is_wrong():
    hip = _hip()
    count = 0
    for name, call, text in _calls():
        with pytest.raises(hip.OatError, match=text):
            call()
            pytest.fail(f"{name}: taken")
        count += 1
    assert count > 90


def test_rows_beyond_32_bits_are_not_cut():
    """2^32 + 8 rows of two values fit the card: they are refused, not taken for 8."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    x, rope, pos = torch.zeros(1, 2, dtype=torch.bfloat16).expand(2 ** 32 + 8, 2), hip.RopeAxes((2,)), torch.zeros(8, 1, dtype=torch.int32)
    for call in (hip.rope_axes, wa.rope_axes):
        with pytest.raises(hip.OatError, match="2.31 rows"):
            call(x, pos, rope, 1, 2)


@pytest.mark.parametrize("change,text", [(dict(D=96), b"64 or 128"), (dict(Hkv=0), b"no heads"), (dict(longest=-1), b"lengths"), (dict(scale=0.0), b"scale"), (dict(seqs=None), b"table")])
def test_packed_layer_refusals(change, text):
    from tests.test_window_cpu import LAYER
    hip = _hip()
    a = {**LAYER, **change}
    _refused(hip, hip.lib().oat_window_attention_packed_fwd(*a.values(), None), text)
    head = [a[n] for n in ("qkv", "ld", "turned", "table", "rope", "pos", "period", "out")] + [4096, 4096, 4096]
    tail = [a[n] for n in ("seqs", "B", "longest", "M", "Hq", "Hkv", "D", "dtype", "left", "right", "sinks", "scale")]
    _refused(hip, hip.lib().oat_window_attention_packed_bwd(*head, *tail, 4096, 1 << 40, None), text)
