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
