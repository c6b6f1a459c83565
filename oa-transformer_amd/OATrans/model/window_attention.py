"""Windowed attention for token sequences that the divided space / time attention does not cover: a clip as ONE sequence of
(time, height, width) tokens behind its class token, captions of any length, text written token by token.

    rope = hip.RopeAxes((16, 24, 24))                     # rotary positions over time, height and width, head_dim 64
    out = window_attention(qkv, seqs, 12, 12, 64, left=392, right=392, sinks=1, longest=1569, rope=rope, pos=pos)

Forward and backward run on liboatrans_hip; there is no CPU path."""
import torch
from torch.autograd.function import once_differentiable

from ..ops import hip


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
    """Rotary positions (hip.rope_axes) with a gradient: x [M, heads * head_dim] -> a new tensor."""
    if x.shape[1] != heads * head_dim:
        raise hip.OatError("rope_axes: x must be [M, heads * head_dim]")
    return _RopeFn.apply(x, pos, rope, heads, head_dim)


def _forward(qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed, lse):
    """-> (out, turned q | k or None): rotary positions into a new buffer (the values stay where they are), attention over it.  The
    arguments of both calls are columns of two buffers, checked here once, so the calls get addresses."""
    M, n = qkv.shape[0], (heads + kv_heads) * D
    what = "window_attention"
    if qkv.stride(1) != 1 or qkv.dtype not in (torch.bfloat16, torch.float16):
        raise hip.OatError(f"{what}: qkv must be bf16 or fp16 with unit column stride")
    if seqs.dtype != torch.int32 or seqs.dim() != 2 or seqs.shape[1] != 4 or not seqs.is_contiguous() or seqs.device != qkv.device:
        raise hip.OatError(f"{what}: seqs must be a contiguous int32 [B, 4] on {qkv.device}")
    lib, dtype, base, ld = hip.lib(), hip._ELEMENTS[qkv.dtype], qkv.data_ptr(), hip._ld(qkv)
    qk, at, ldqk = None, base, ld
    if rope is not None:
        if pos.dtype != torch.int32 or pos.dim() != 2 or pos.shape[1] != rope.axes or not pos.is_contiguous() or pos.device != qkv.device:
            raise hip.OatError(f"{what}: pos must be a contiguous int32 [P, {rope.axes}] on {qkv.device}")
        qk = torch.empty(M, n, dtype=qkv.dtype, device=qkv.device)
        at, ldqk = qk.data_ptr(), n
        hip._launch(qkv.device, lib.oat_rope_axes, (base, ld, at, n, dtype, pos.data_ptr(), pos.shape[0], M, heads + kv_heads, D, rope.struct, 0),
                    "oat_rope_axes")
    out = (torch.empty if packed else torch.zeros)(M, heads * D, dtype=qkv.dtype, device=qkv.device)
    size = qkv.element_size()
    hip._launch(qkv.device, lib.oat_attn_window_fwd, (
        at, ldqk, at + heads * D * size, ldqk, base + n * size, ld, out.data_ptr(), heads * D, lse.data_ptr() if lse is not None else None,
        seqs.data_ptr(), seqs.shape[0], longest, longest, M, M, heads, kv_heads, D, dtype, *window, D ** -0.5 if scale is None else scale),
        "oat_attn_window_fwd")
    return out, qk


class _WindowFn(torch.autograd.Function):
    """Rotary positions, attention over the window and its sinks, and the gradient of all of it with respect to qkv.  Saved: qkv, the
    turned q | k, out and the log-sum-exp; backward forms the probabilities again."""

    @staticmethod
    def forward(ctx, qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed):
        lse = torch.empty(qkv.shape[0], heads, dtype=torch.float32, device=qkv.device)
        out, qk = _forward(qkv, seqs, pos, heads, kv_heads, D, longest, window, scale, rope, packed, lse)
        ctx.save_for_backward(qkv, qk, out, lse, seqs, pos)
        ctx.args = heads, kv_heads, D, longest, window, scale, rope, packed
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, qk, out, lse, seqs, pos = ctx.saved_tensors
        heads, kv_heads, D, longest, window, scale, rope, packed = ctx.args
        n, a = (heads + kv_heads) * D, heads * D
        qk = qkv if qk is None else qk
        dqkv = (torch.empty if packed else torch.zeros)(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        hip.attn_window_bwd(qk[:, :a], qk[:, a:n], qkv[:, n:], out, lse, dout.contiguous(), seqs, heads, kv_heads, D, longest, longest, *window,
                            scale=scale, dq=dqkv[:, :a], dk=dqkv[:, a:n], dv=dqkv[:, n:])
        if rope is not None:
            turned = dqkv[:, :n]
            hip.rope_axes(turned, pos, rope, heads + kv_heads, D, out=turned, inverse=True)
        return dqkv, None, None, None, None, None, None, None, None, None, None


def window_attention(qkv, seqs, heads, kv_heads, head_dim, left=-1, right=0, sinks=0, longest=None, scale=None, rope=None, pos=None,
                     packed=False, cache=None):
    """qkv [M, (heads + 2 * kv_heads) * head_dim] (bf16 / fp16; q | k | v) -> [M, heads * head_dim].

    seqs: int32 [B, 4] on the device (hip.seq_table); longest: the largest count in it (default: M).  Token i of a sequence sees
    token j if j <= i + right and (j >= i - left or j < sinks); left / right < 0: no such edge, right = 0: causal.
    rope, pos: rotary positions of q and k, pos int32 [P, axes] with M a multiple of P.
    packed: the caller states that every row belongs to a sequence; otherwise rows of none (padding) get zeros, and zero gradients.
    cache: (k, v) of [B, slots, kv_heads, head_dim] that take the prompt's turned keys and its values (no gradient then); fewer slots
    than tokens only where they are the sinks and the window, sinks + left + 1."""
    D = head_dim
    if qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * kv_heads) * D:
        raise hip.OatError(f"window_attention: qkv must be [M, {(heads + 2 * kv_heads) * D}]")
    if (rope is None) != (pos is None):
        raise hip.OatError("window_attention: rope and pos belong together")
    longest = qkv.shape[0] if longest is None else int(longest)
    grad = torch.is_grad_enabled() and qkv.requires_grad
    if cache is None and grad:
        return _WindowFn.apply(qkv, seqs, pos, heads, kv_heads, D, longest, (left, right, sinks), scale, rope, packed)
    if grad:
        raise hip.OatError("window_attention: a cache takes a prompt without a gradient (use torch.no_grad())")
    qkv = qkv.detach()
    if cache is not None:
        slots = cache[0].shape[1]
        if right != 0 or (slots < longest and not (left >= 0 and slots == sinks + left + 1)):
            raise hip.OatError("window_attention: a cache belongs to causal attention (right = 0) and needs a slot for every token, or "
                               "sinks + left + 1 slots")
    out, qk = _forward(qkv, seqs, pos, heads, kv_heads, D, longest, (left, right, sinks), scale, rope, packed, None)
    if cache is not None:
        n = (heads + kv_heads) * D
        hip.window_cache_fill((qkv if qk is None else qk)[:, heads * D:n], qkv[:, n:], seqs, cache[0], cache[1], longest, sinks=sinks)
    return out


class WindowCache:
    """Keys and values of B sequences that are written token by token, with the operator's workspace and the counts of tokens.

    window: tokens that stay visible besides the `sinks` first ones; the cache then holds sinks + window slots and rolls.  None: it
    holds `slots` tokens and everything is visible."""

    def __init__(self, B, heads, kv_heads, head_dim, window=None, sinks=0, slots=None, rope=None, dtype=torch.bfloat16, device="cuda"):
        if (window is None) == (slots is None) or (window is not None and window < 1) or (slots is not None and slots < 1):
            raise hip.OatError("WindowCache: either a window (it rolls) or a number of slots, at least 1")
        self.rolling, self.left = window is not None, -1 if window is None else window - 1
        self.slots = slots if window is None else sinks + window
        self.heads, self.kv_heads, self.head_dim, self.sinks, self.rope = heads, kv_heads, head_dim, sinks, rope
        self.k = torch.zeros(B, self.slots, kv_heads, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.past = torch.zeros(B, dtype=torch.int32, device=self.k.device)
        self.pieces = hip.window_step_workspace(B, heads, kv_heads, head_dim, self.k.device)

    @torch.no_grad()
    def prompt(self, qkv, seqs, longest, pos=None, scale=None):
        """Causal attention over the prompts; their keys and values and their counts go into the cache."""
        out = window_attention(qkv, seqs, self.heads, self.kv_heads, self.head_dim, left=self.left, right=0, sinks=self.sinks,
                               longest=longest, scale=scale, rope=self.rope, pos=pos, cache=(self.k, self.v))
        self.past.copy_(seqs[:, 3])
        return out

    @torch.no_grad()
    def step(self, qkv, pos=None, scale=None):
        """One new token of every sequence: qkv [B, (heads + 2 * kv_heads) * head_dim] -> [B, heads * head_dim].  pos: int32 [B, axes]
        (default, one axis: the count of tokens so far)."""
        if self.rope is not None and pos is None:
            if self.rope.axes != 1:
                raise hip.OatError("WindowCache.step: several axes need pos")
            pos = self.past[:, None]
        out = hip.attn_window_step(qkv, self.past, self.k, self.v, self.heads, left=self.left, sinks=self.sinks, rolling=self.rolling,
                                   scale=scale, rope=self.rope, pos=pos, pieces=self.pieces)
        self.past += self.past >= 0
        return out
