"""Windowed attention for token sequences that the divided space / time attention does not cover: a clip as ONE sequence of
(time, height, width) tokens behind its class token, captions of any length, text written token by token.

    rope = hip.RopeAxes((16, 24, 24))                     # rotary positions over time, height and width, head_dim 64
    out = window_attention(qkv, seqs, 12, 12, 64, left=392, right=392, sinks=1, longest=1569, rope=rope, pos=pos)

Forward and backward run on liboatrans_hip; there is no CPU path."""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..ops import hip


def _no_tangent(x, what):
    # (the level first: outside of forward mode unpack_dual alone takes 0.9 us)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise hip.OatError(f"{what}: no gradients in forward mode (the tangent would be lost)")


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, rope, heads, head_dim):
        ctx.save_for_backward(pos)
        ctx.args = rope, heads, head_dim
        return hip.rope_axes(x, pos, rope, heads, head_dim)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (pos,) = ctx.saved_tensors
        rope, heads, head_dim = ctx.args
        return hip.rope_axes(g.contiguous(), pos, rope, heads, head_dim, inverse=True), None, None, None, None


def rope_axes(x, pos, rope, heads, head_dim):
    """Rotary positions (hip.rope_axes, which has none) with a gradient: x [M, heads * head_dim] -> a new tensor."""
    _no_tangent(x, "rope_axes")
    if x.shape[1] != heads * head_dim:
        raise hip.OatError("rope_axes: x must be [M, heads * head_dim]")
    return _RopeFn.apply(x, pos, rope, heads, head_dim)


def _new(packed, longest, seqs):
    """how a result starts: where every row belongs to a sequence the library writes them all, if there is any work"""
    return torch.empty if packed and longest > 0 and seqs.shape[0] else torch.zeros


def _forward(qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed, lse, cache):
    """-> (out, turned q | k or None, the turns or None): rotary positions into a new buffer (the values stay where they are), attention
    over it, and the prompt's rows into the cache, in one call.  The turns - every row's cos and sin - are kept for a backward pass
    that can use them (pairs that are a head's two halves)."""
    M, dev, dt = qkv.shape[0], qkv.device, qkv.dtype
    what = "window_attention"
    if qkv.stride(1) != 1 or (dt is not torch.bfloat16 and dt is not torch.float16):
        raise hip.OatError(f"{what}: qkv must be bf16 or fp16 with unit column stride")
    if seqs.dtype is not torch.int32 or seqs.dim() != 2 or seqs.shape[1] != 4 or not seqs.is_contiguous() or seqs.device != dev:
        raise hip.OatError(f"{what}: seqs must be a contiguous int32 [B, 4] on {dev}")
    qk = turned = turns = struct = places = None
    period = 0
    if rope is not None:
        if pos.dtype is not torch.int32 or pos.dim() != 2 or pos.shape[1] != rope.axes or not pos.is_contiguous() or pos.device != dev:
            raise hip.OatError(f"{what}: pos must be a contiguous int32 [P, {rope.axes}] on {dev}")
        qk = torch.empty(M, (heads + kv_heads) * D, dtype=dt, device=dev)
        turned, struct, places, period = qk.data_ptr(), rope.struct, pos.data_ptr(), pos.shape[0]
        if lse is not None and 2 * rope.pairs == D and not rope.interleaved:
            turns = torch.empty(rope.pairs, M, 2, dtype=torch.float32, device=dev)
    out = _new(packed, longest, seqs)(M, heads * D, dtype=dt, device=dev)
    kc = vc = strides = None
    cap = 0
    if cache is not None:
        k, v = cache
        strides, cap = hip._cache_args(k, v, what), k.shape[1]
        if k.dtype is not dt or k.device != dev or k.shape[0] != seqs.shape[0] or k.shape[2] != kv_heads or k.shape[3] != D:
            raise hip.OatError(f"{what}: the caches must be [{seqs.shape[0]}, slots, {kv_heads}, {D}] of {dt} on {dev}")
        kc, vc = k.data_ptr(), v.data_ptr()
    hip._launch(dev, hip.lib().oat_window_attention_packed_fwd if packed else hip.lib().oat_window_attention_fwd, (
        qkv.data_ptr(), hip._ld(qkv), turned, turns.data_ptr() if turns is not None else None, struct, places, period, out.data_ptr(), lse.data_ptr() if lse is not None else None,
        seqs.data_ptr(), seqs.shape[0], longest, M, heads, kv_heads, D, hip._ELEMENTS[dt], *window, D ** -0.5 if scale is None else scale,
        kc, vc, strides, cap), what)
    return out, qk, turns


class _WindowFn(torch.autograd.Function):
    """Rotary positions, attention over the window and its sinks, and the gradient of all of it with respect to qkv.  Saved: qkv, the
    turned q | k, the turns, out and the log-sum-exp; backward forms the probabilities again."""

    @staticmethod
    def forward(ctx, qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed):
        lse = torch.empty(qkv.shape[0], heads, dtype=torch.float32, device=qkv.device)
        out, qk, turns = _forward(qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed, lse, None)
        ctx.save_for_backward(qkv, qk, turns, out, lse, seqs, pos)
        ctx.args = heads, kv_heads, D, longest, window, scale, rope, packed
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, qk, turns, out, lse, seqs, pos = ctx.saved_tensors
        heads, kv_heads, D, longest, window, scale, rope, packed = ctx.args
        dout, dev, lib = dout.contiguous(), qkv.device, hip.lib()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        M, B = qkv.shape[0], seqs.shape[0]
        dqkv = _new(packed, longest, seqs)(qkv.shape, dtype=qkv.dtype, device=dev)
        need = lib.oat_attn_window_bwd_workspace_bytes(M, B, longest, longest, heads, kv_heads, D, window[0], window[2])
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        hip._launch(dev, lib.oat_window_attention_packed_bwd if packed else lib.oat_window_attention_bwd, (
            qkv.data_ptr(), hip._ld(qkv), qk.data_ptr() if qk is not None else None,
            turns.data_ptr() if turns is not None else None, rope.struct if rope is not None else None,
            pos.data_ptr() if pos is not None else None, pos.shape[0] if pos is not None else 0, out.data_ptr(), lse.data_ptr(),
            dout.data_ptr(), dqkv.data_ptr(), seqs.data_ptr(), B, longest, M, heads, kv_heads, D, hip._ELEMENTS[qkv.dtype], *window,
            D ** -0.5 if scale is None else scale, ws.data_ptr(), need), "window_attention backward")
        return dqkv, None, None, None, None, None, None, None, None, None, None


def window_attention(qkv, seqs, heads, kv_heads, head_dim, left=-1, right=0, sinks=0, longest=None, scale=None, rope=None, pos=None,
                     packed=False, cache=None):
    """qkv [M, (heads + 2 * kv_heads) * head_dim] (bf16 / fp16; q | k | v) -> [M, heads * head_dim].

    seqs: int32 [B, 4] on the device (hip.seq_table); longest: the largest count in it (default: M; a sequence with more is taken as
    empty: zeros).  Token i of a sequence sees
    token j if j <= i + right and (j >= i - left or j < sinks); left / right < 0: no such edge, right = 0: causal.
    rope, pos: rotary positions of q and k, pos int32 [P, axes] with M a multiple of P.
    packed: the caller states that every row belongs to a sequence; otherwise rows of none (padding) get zeros, and zero gradients.
    Rows of no sequence may hold anything; rows of a sequence have to be finite (a masked pair's weight is an exact zero, and it is
    multiplied).  fp16 gradients: the probabilities' gradient P (dout . v - delta) has to stay below 65504: beyond, dq and dk are inf or nan,
    which a loss scaler sees; below 2^-14 it loses bits.
    cache: (k, v) of [B, slots, kv_heads, head_dim] that take the prompt's turned keys and its values (no gradient then); fewer slots
    than tokens only where they are the sinks and the window, sinks + left + 1."""
    D = head_dim
    _no_tangent(qkv, "window_attention")
    if qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * kv_heads) * D:
        raise hip.OatError(f"window_attention: qkv must be [M, {(heads + 2 * kv_heads) * D}]")
    if (rope is None) != (pos is None):
        raise hip.OatError("window_attention: rope and pos belong together")
    longest = qkv.shape[0] if longest is None else min(int(longest), qkv.shape[0])
    left, right, sinks = hip._reach(left), hip._reach(right), hip._reach(sinks)
    grad = torch.is_grad_enabled() and qkv.requires_grad
    if cache is None and grad:
        return _WindowFn.apply(qkv, seqs, pos, heads, kv_heads, D, longest, (left, right, sinks), scale, rope, packed)
    if grad:
        raise hip.OatError("window_attention: a cache takes a prompt without a gradient (use torch.no_grad())")
    if cache is not None:
        slots = cache[0].shape[1]
        if right != 0 or (slots < longest and not (left >= 0 and slots == sinks + left + 1)):
            raise hip.OatError("window_attention: a cache belongs to causal attention (right = 0) and needs a slot for every token, or "
                               "sinks + left + 1 slots")
    return _forward(qkv, seqs, pos, heads, kv_heads, D, longest, (left, right, sinks), scale, rope, packed, None, cache)[0]


class WindowCache:
    """Keys and values of B sequences that are written token by token, with the operator's workspace and the counts of tokens.

    window: tokens that stay visible besides the `sinks` first ones; the cache then holds sinks + window slots and rolls.  None: it
    holds `slots` tokens and everything is visible; a sequence without a slot left takes no part any more: step gives it a row of
    zeros, and its cache and its count (past == slots) stay.  past may be set by the caller: a negative count takes no part either."""

    def __init__(self, B, heads, kv_heads, head_dim, window=None, sinks=0, slots=None, rope=None, dtype=torch.bfloat16, device="cuda"):
        if (window is None) == (slots is None) or (window is not None and window < 1) or (slots is not None and slots < 1):
            raise hip.OatError("WindowCache: either a window (it rolls) or a number of slots, at least 1")
        if head_dim not in (64, 128) or kv_heads < 1 or heads < 1 or heads % kv_heads or dtype not in (torch.bfloat16, torch.float16) or B < 0 or sinks < 0:
            raise hip.OatError("WindowCache: heads of 64 or 128 in bf16 or fp16, query heads a multiple of the key heads, no negative sinks")
        self.rolling, self.left = window is not None, -1 if window is None else window - 1
        self.slots = slots if window is None else sinks + window
        self.heads, self.kv_heads, self.head_dim, self.sinks, self.rope = heads, kv_heads, head_dim, sinks, rope
        self.k = torch.zeros(B, self.slots, kv_heads, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.past = torch.zeros(B, dtype=torch.int32, device=self.k.device)
        self.pieces = hip.window_step_workspace(B, heads, kv_heads, head_dim, self.k.device)

    @torch.no_grad()
    def prompt(self, qkv, seqs, longest=None, pos=None, scale=None):
        """Causal attention over the prompts; their keys and values and their counts go into the cache.  longest: the largest count of
        the table (default: all rows); a sequence with more is taken as empty, here and in its counts."""
        longest = qkv.shape[0] if longest is None else min(int(longest), qkv.shape[0])
        out = window_attention(qkv, seqs, self.heads, self.kv_heads, self.head_dim, left=self.left, right=0, sinks=self.sinks,
                               longest=longest, scale=scale, rope=self.rope, pos=pos, cache=(self.k, self.v))
        hip.window_cache_counts(self.past, seqs, qkv.shape[0], longest)
        return out

    @torch.no_grad()
    def step(self, qkv, pos=None, scale=None):
        """One new token of every sequence: qkv [B, (heads + 2 * kv_heads) * head_dim] -> [B, heads * head_dim].  pos: int32 [B, axes]
        (default, one axis: the count of tokens so far)."""
        _no_tangent(qkv, "WindowCache.step")
        if self.rope is not None and pos is None:
            if self.rope.axes != 1:
                raise hip.OatError("WindowCache.step: several axes need pos")
            pos = self.past[:, None]
        out = hip.attn_window_step(qkv, self.past, self.k, self.v, self.heads, left=self.left, sinks=self.sinks, rolling=self.rolling,
                                   scale=scale, rope=self.rope, pos=pos, pieces=self.pieces)
        hip.window_cache_advance(self.past, None if self.rolling else self.slots)
        return out
