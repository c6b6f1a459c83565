"""Refusals of the rotary and windowed-attention operators: they run before any launch, so no GPU is needed."""
import ctypes

import pytest
import torch


def _hip():
    from OATrans.ops import hip
    hip.lib()
    return hip


ONE, LL = ctypes.c_void_p(4096), ctypes.c_longlong


def _refused(hip, rc, text):
    assert rc < 0 and text in hip.lib().oat_last_error(), hip.lib().oat_last_error()


def test_rope_refusals():
    hip = _hip()
    rope = hip.RopeAxes((16, 24, 24))
    call = lambda x=4096, ldx=64, out=8192, ldo=64, dtype=0, pos=4096, period=1, M=4, heads=1, dim=64, r=rope.struct, inverse=0: \
        hip.lib().oat_rope_axes(x, ldx, out, ldo, dtype, pos, period, M, heads, dim, r, inverse, None)
    _refused(hip, call(dtype=3), b"element type")
    _refused(hip, call(period=3), b"whole number")
    _refused(hip, call(period=0), b"whole number")
    _refused(hip, call(ldx=63), b"shorter")
    _refused(hip, call(heads=0), b"no heads")
    _refused(hip, call(dim=62, ldx=62), b"more than the head")
    _refused(hip, call(x=None), b"needed")
    _refused(hip, call(pos=None), b"needed")
    _refused(hip, call(M=-1), b"no heads")
    _refused(hip, call(out=4096, ldo=128), b"one row pitch")
    _refused(hip, call(dim=1 << 15, heads=64, ldx=1 << 21, ldo=1 << 21), b"2^20")
    for field, value in (("n_pairs", 0), ("n_pairs", 65), ("n_axes", 0), ("n_axes", 5), ("n_axes", 2)):
        bad = hip.RopeAxes((16, 24, 24)).struct
        setattr(bad, field, value)
        assert call(r=bad) < 0
    bad = hip.RopeAxes((16, 24, 24)).struct
    bad.turns[3] = float("nan")
    _refused(hip, call(r=bad), b"not a number")
    assert call(M=0) == 0                                          # nothing to do
    for sections, theta in (((), 1e4), ((3,), 1e4), ((0,), 1e4), ((64, 66), 1e4), ((2, 2, 2, 2, 2), 1e4), ((64,), 0.0), ((64,), float("inf"))):
        with pytest.raises(hip.OatError):
            hip.RopeAxes(sections, theta)


def test_rope_ladders():
    hip = _hip()
    f, a = hip.RopeAxes((4, 6), theta=100.0).frequencies()
    assert a.tolist() == [0, 0, 1, 1, 1]
    assert torch.allclose(f, torch.tensor([1.0, 100.0 ** -0.5, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64), rtol=1e-15)
    f, _ = hip.RopeAxes((4, 6), theta=100.0, shared=True).frequencies()
    assert torch.allclose(f, 100.0 ** (-torch.arange(5, dtype=torch.float64) / 5), rtol=1e-15)


FWD = dict(q=4096, ldq=128, k=4096, ldk=64, v=4096, ldv=64, out=8192, ldo=128, lse=None, seqs=4096, B=1, max_q=10, max_k=10, rows_q=10, rows_k=10,
           Hq=2, Hkv=1, D=64, dtype=0, left=-1, right=0, sinks=0, scale=0.125)


@pytest.mark.parametrize("change,text", [
    (dict(D=96), b"64 or 128"), (dict(dtype=2), b"element type"), (dict(Hq=3, Hkv=2), b"multiple"), (dict(Hkv=0), b"multiple"),
    (dict(B=-1), b"lengths"), (dict(max_q=2 ** 30), b"lengths"), (dict(rows_k=-1), b"lengths"), (dict(seqs=None), b"table"), (dict(seqs=4100), b"table"),
    (dict(sinks=-1), b"sinks"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(q=4098), b"16-byte"), (dict(ldq=127), b"16-byte"), (dict(ldk=56), b"16-byte"), (dict(v=None), b"16-byte"), (dict(out=None), b"16-byte"),
    (dict(ldv=2 ** 23), b"16-byte"), (dict(B=2 ** 22, Hq=256, max_q=2 ** 15), b"tiles")])
def test_attention_refusals(change, text):
    hip = _hip()
    a = {**FWD, **change}
    _refused(hip, hip.lib().oat_attn_window_fwd(*a.values(), None), text)
    b = [a[n] for n in ("q", "ldq", "k", "ldk", "v", "ldv", "out", "ldo")] + [4096, 4096, 128, 4096, 128, 4096, 64, 4096, 64]
    b += [a[n] for n in ("seqs", "B", "max_q", "max_k", "rows_q", "rows_k", "Hq", "Hkv", "D", "dtype", "left", "right", "sinks", "scale")]
    _refused(hip, hip.lib().oat_attn_window_bwd(*b, 4096, 1 << 40, None), text)


def test_attention_backward_needs_its_workspace_and_gradients():
    hip = _hip()
    bwd = lambda lse=4096, dout=4096, dq=4096, ws=4096, n=160: hip.lib().oat_attn_window_bwd(
        4096, 128, 4096, 64, 4096, 64, 4096, 128, lse, dout, 128, dq, 128, 4096, 64, 4096, 64, 4096, 1, 10, 10, 10, 10, 2, 1, 64, 0, -1, 0, 0, 0.125, ws, n, None)
    need = hip.lib().oat_attn_window_bwd_workspace_bytes(10, 1, 10, 10, 2, 1, 64, -1, 0)
    assert need == 160
    _refused(hip, bwd(n=need - 1), b"workspace")
    _refused(hip, bwd(ws=None), b"workspace")
    _refused(hip, bwd(lse=None), b"lse")
    _refused(hip, bwd(dq=4097), b"16-byte")


STEP = dict(qkv=4096, ldqkv=256, past=4096, kc=4096, vc=4096, strides=(64 * 16, 64, 64) * 2, cap=16, out=4096, ldo=128, B=1, Hq=2, Hkv=1, D=64,
            dtype=0, left=-1, sinks=0, rolling=0, scale=0.125, rope=None, pos=None, ws=4096, n=1 << 30)


@pytest.mark.parametrize("change,text", [
    (dict(D=32), b"64 or 128"), (dict(dtype=2), b"element type"), (dict(Hq=3, Hkv=2), b"multiple"), (dict(cap=0), b"no slots"), (dict(kc=None), b"missing"),
    (dict(kc=4104), b"aligned"), (dict(strides=(1024, 63, 64, 1024, 64, 64)), b"strides"), (dict(scale=0.0), b"scale"), (dict(qkv=None), b"needed"),
    (dict(past=None), b"needed"), (dict(ldqkv=248), b"16-byte"), (dict(out=4097), b"16-byte"), (dict(rolling=1, sinks=16), b"rolling"),
    (dict(rolling=1, left=3), b"rolling"), (dict(rope=True), b"positions"), (dict(n=16), b"workspace"), (dict(ws=None), b"workspace"), (dict(sinks=-1), b"slots")])
def test_step_refusals(change, text):
    hip = _hip()
    a = {**STEP, **change}
    a["strides"] = (LL * 6)(*a["strides"])
    if a["rope"]:
        a["rope"] = hip.RopeAxes((64,)).struct
    _refused(hip, hip.lib().oat_attn_window_step(*a.values(), None), text)
    if not set(change) & {"D", "cap", "kc", "strides", "sinks"} or "rolling" in change:
        return
    _refused(hip, hip.lib().oat_window_cache_fill(4096, 64, 4096, 64, 4096, 1, 10, 10, a["kc"], a["vc"], a["strides"], a["cap"], 1, a["D"], a["sinks"], None), text)


def test_fill_refusals():
    hip = _hip()
    st = (LL * 6)(1024, 64, 64, 1024, 64, 64)
    fill = lambda k=4096, ldk=64, seqs=4096, B=1, rows=10: hip.lib().oat_window_cache_fill(k, ldk, 4096, 64, seqs, B, rows, 10, 4096, 4096, st, 16, 1, 64, 0, None)
    _refused(hip, fill(k=4097), b"16-byte")
    _refused(hip, fill(ldk=56), b"16-byte")
    _refused(hip, fill(seqs=None), b"16-byte")
    _refused(hip, fill(rows=-1), b"no rows")
    _refused(hip, fill(B=65536), b"65535")


def test_python_refuses_what_the_library_cannot_see():
    """Types, shapes and devices are the binding's to check; nothing here reaches a launch."""
    hip = _hip()
    from OATrans.model import window_attention as wa
    x, pos, rope = torch.zeros(4, 64), torch.zeros(4, 3, dtype=torch.int32), hip.RopeAxes((16, 24, 24))
    bad = [lambda: hip.rope_axes(x, pos, rope, 1, 64),                                        # on the CPU
           lambda: hip.rope_axes(x.double(), pos, rope, 1, 64), lambda: hip.rope_axes(x, pos.long(), rope, 1, 64),
           lambda: hip.rope_axes(x, pos[:, :2], rope, 1, 64), lambda: hip.rope_axes(x, pos, rope, 2, 64),
           lambda: hip.rope_axes(x, pos, rope, 1, 64, out=torch.zeros(3, 64)), lambda: hip.rope_axes(x[:, ::2], pos, rope, 1, 32)]
    b = torch.zeros(4, 64, dtype=torch.bfloat16)
    seqs = hip.seq_table([4], device="cpu")
    bad += [lambda: hip.attn_window_fwd(b, b, b, seqs, 1, 1, 64, 4, 4), lambda: hip.attn_window_fwd(x, x, x, seqs, 1, 1, 64, 4, 4),
            lambda: hip.attn_window_fwd(b, b[:3], b, seqs, 1, 1, 64, 4, 4), lambda: hip.attn_window_fwd(b, b, b, seqs.long(), 1, 1, 64, 4, 4),
            lambda: hip.attn_window_fwd(b, b, b, seqs, 1, 1, 64, 4, 4, lse=torch.zeros(4, 2)), lambda: hip.seq_table([1, -1]), lambda: hip.seq_table([1, 2], [1])]
    c = torch.zeros(4, 8, 1, 64, dtype=torch.bfloat16)
    past = torch.zeros(4, dtype=torch.int32)
    row = torch.zeros(4, 192, dtype=torch.bfloat16)
    ws = torch.zeros(4)
    bad += [lambda: hip.attn_window_step(row, past, c, c, 1, pieces=ws), lambda: hip.attn_window_step(row, past.long(), c, c, 1, pieces=ws),
            lambda: hip.attn_window_step(row[:3], past, c, c, 1, pieces=ws), lambda: hip.attn_window_step(row, past, c, c[:, :4], 1, pieces=ws),
            lambda: hip.attn_window_step(row, past, c, c, 1, rope=rope, pieces=ws), lambda: hip.window_cache_fill(b, b, seqs, c, c, 4)]
    qkv = torch.zeros(4, 192, dtype=torch.bfloat16)
    bad += [lambda: wa.window_attention(qkv, seqs, 1, 1, 128), lambda: wa.window_attention(qkv, seqs, 1, 1, 64, rope=rope),
            lambda: wa.window_attention(qkv, seqs, 1, 1, 64, right=1, cache=(c, c)), lambda: wa.window_attention(qkv, seqs, 1, 1, 64, longest=9, cache=(c, c)),
            lambda: wa.window_attention(qkv.clone().requires_grad_(), seqs, 1, 1, 64, cache=(c, c)),
            lambda: wa.WindowCache(1, 1, 1, 64, device="cpu"), lambda: wa.WindowCache(1, 1, 1, 64, window=0, device="cpu")]
    for i, call in enumerate(bad):
        with pytest.raises(hip.OatError):
            call()
            pytest.fail(f"call {i} was taken")


def test_seq_table():
    hip = _hip()
    assert hip.seq_table([3, 0, 5], device="cpu").tolist() == [[0, 3, 0, 3], [3, 0, 3, 0], [3, 5, 3, 5]]
    assert hip.seq_table([1, 1], [7, 9], device="cpu").tolist() == [[0, 1, 0, 7], [1, 1, 7, 9]]
    assert hip.seq_table([2, 3], q_rows=(0, 10), device="cpu").tolist() == [[0, 2, 0, 2], [10, 3, 10, 3]]
    assert hip.seq_table([], device="cpu").shape == (0, 4)


def test_oracle_of_the_window_against_dense_attention():
    """The 64-bit definition itself: no window = dense softmax attention; a rolling cache's slots are the window and its sinks."""
    from oracle import window_oracle as wo
    q, k, v = (torch.randn(9, 64, dtype=torch.float64) for _ in range(3))
    ref = torch.softmax(q @ k.t() / 8, 1) @ v
    assert torch.allclose(wo.attention(q, k, v, [(0, 9, 0, 9)], 1, 1, 64, -1, -1, 0, 0.125)["out"], ref)
    see = wo.visible(4, 6, 1, 0, 1)
    assert see.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    slots = {t: wo.slot(t, 7, 2, True) for t in range(40)}
    assert sorted(slots[t] for t in [0, 1] + list(range(35, 40))) == list(range(7))
    x = torch.randn(3, 2, 8, dtype=torch.float64)
    pos = torch.tensor([[1, 5], [0, 0], [7, 2]])
    y = wo.rope(x, pos, (4, 4), 50.0)
    assert torch.allclose(wo.rope(y, pos, (4, 4), 50.0, inverse=True), x) and torch.allclose(y[1], x[1]) and torch.allclose(y.norm(dim=-1), x.norm(dim=-1))


LAYER = dict(qkv=4096, ld=256, turned=None, table=None, rope=None, pos=None, period=0, out=4096, lse=None, seqs=4096, B=1, longest=10, M=10, Hq=2, Hkv=1, D=64,
             dtype=0, left=-1, right=0, sinks=0, scale=0.125, kc=None, vc=None, strides=None, cap=0)


@pytest.mark.parametrize("change,text", [
    (dict(D=96), b"64 or 128"), (dict(dtype=2), b"element type"), (dict(Hq=3, Hkv=2), b"multiple"), (dict(Hkv=0), b"no heads"), (dict(M=-1), b"no heads"),
    (dict(longest=2 ** 30), b"lengths"), (dict(seqs=None), b"table"), (dict(sinks=-1), b"sinks"), (dict(scale=0.0), b"scale"), (dict(qkv=4098), b"16-byte"),
    (dict(ld=248, D=128), b"16-byte"), (dict(rope=True, pos=4096, period=10), b"turned"), (dict(rope=True, turned=4096, period=10), b"needed"),
    (dict(rope=True, turned=4096, pos=4096, period=3), b"whole number")])
def test_layer_refusals(change, text):
    hip = _hip()
    a = {**LAYER, **change}
    if a["rope"]:
        a["rope"] = hip.RopeAxes((64,)).struct
    _refused(hip, hip.lib().oat_window_attention_fwd(*a.values(), None), text)
    if "period" in change and text != b"turned":                   # (the way back turns last: its rotary arguments are the forward's)
        return
    head = [a[n] for n in ("qkv", "ld", "turned", "table", "rope", "pos", "period", "out")] + [4096, 4096, 4096]
    tail = [a[n] for n in ("seqs", "B", "longest", "M", "Hq", "Hkv", "D", "dtype", "left", "right", "sinks", "scale")]
    _refused(hip, hip.lib().oat_window_attention_bwd(*head, *tail, 4096, 1 << 40, None), text)


def test_workspaces_belong_to_their_sizes():
    hip = _hip()
    a = {**STEP, "strides": (LL * 6)(*STEP["strides"])}
    need = hip.lib().oat_attn_window_step_workspace_bytes(1, 2, 1, 64)
    for n in (need - 4, need + 4, hip.lib().oat_attn_window_step_workspace_bytes(2, 2, 1, 64)):
        _refused(hip, hip.lib().oat_attn_window_step(*{**a, "n": n}.values(), None), b"workspace")
    _refused(hip, hip.lib().oat_attn_window_step(*{**a, "n": need, "ws": 4100}.values(), None), b"workspace")
    q = torch.zeros(4, 64, dtype=torch.bfloat16)
    for most in (-1, 2 ** 29 + 1, 2 ** 32 + 4):                    # a count is not cut to its low 32 bits
        with pytest.raises(hip.OatError, match="largest counts"):
            hip.attn_window_fwd(q, q, q, hip.seq_table([4], device="cpu"), 1, 1, 64, most, 4)
    assert [hip._reach(n) for n in (-7, -1, 0, 9, 2 ** 29, 2 ** 29 + 1, 2 ** 32, 2 ** 63)] == [-1, -1, 0, 9] + [2 ** 29] * 4


def test_layer_backward_refuses_a_misaligned_table():
    hip = _hip()
    rope = hip.RopeAxes((64,)).struct
    args = [4096, 256, 4096, 4100, rope, 4096, 10, 4096, 4096, 4096, 4096] + [LAYER[n] for n in (
        "seqs", "B", "longest", "M", "Hq", "Hkv", "D", "dtype", "left", "right", "sinks", "scale")]
    _refused(hip, hip.lib().oat_window_attention_bwd(*args, 4096, 1 << 40, None), b"not aligned")
