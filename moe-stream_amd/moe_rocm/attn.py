"""The attention side of a decoder layer (include/moe_rocm_attn.h): rotary positions with head norms, a
paged cache of keys and values, attention over it and over packed prompts. Re-exported by moe_rocm.

Arguments are device buffers or addresses, as everywhere in this package; rows of heads are described by
Heads. Index arrays (positions, slots, lengths, pages, offsets) are device int32.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import Context, _f32, _lib, _ptr, _register, _u32, _u64, _vp

F32, F16, BF16 = 0, 1, 2
ROPE_HALF, ROPE_INTERLEAVED = 0, 1
ROPE_PLAIN, ROPE_LINEAR, ROPE_YARN, ROPE_YARN_EXACT = 0, 1, 2, 3
KV_F16, KV_MXINT8, KV_MXFP4 = 16, 8, 4


class CHeads(C.Structure):
    _fields_ = [("data", _vp), ("dtype", _u32), ("n_heads", _u32), ("token_stride", _u64), ("head_stride", _u64)]


class RopeDesc(C.Structure):
    _fields_ = [("head_dim", _u32), ("rotary_dim", _u32), ("layout", _u32), ("scaling", _u32), ("base", C.c_double),
                ("factor", C.c_double), ("orig_context", _u32), ("beta_fast", _f32), ("beta_slow", _f32),
                ("attn_factor", _f32)]


class KvDesc(C.Structure):
    _fields_ = [("format", _u32), ("n_pages", _u32), ("page_size", _u32), ("n_heads", _u32), ("head_dim", _u32)]


class AttnOpts(C.Structure):
    _fields_ = [("scale", _f32), ("window", _u32), ("sinks", _vp)]


_H = C.POINTER(CHeads)
_register({
    "mr_rope_create": (C.c_int, [_vp, C.POINTER(RopeDesc), C.POINTER(_vp)]),
    "mr_rope_destroy": (None, [_vp]),
    "mr_rope_frequencies": (C.POINTER(C.c_double), [_vp, C.POINTER(_u32), C.POINTER(_f32)]),
    "mr_qk_norm_rope": (C.c_int, [_vp, _vp, _H, _H, _vp, _vp, _f32, _vp, _u32, _H, _H]),
    "mr_kv_create": (C.c_int, [_vp, C.POINTER(KvDesc), C.POINTER(_vp)]),
    "mr_kv_destroy": (None, [_vp]),
    "mr_kv_bytes": (_u64, [C.POINTER(KvDesc)]),
    "mr_kv_write": (C.c_int, [_vp, _vp, _H, _H, _u32, _vp]),
    "mr_kv_read": (C.c_int, [_vp, _vp, _u32, _vp, _H, _H]),
    "mr_attn_decode": (C.c_int, [_vp, _vp, _H, _u32, _vp, _vp, _u32, C.POINTER(AttnOpts), _H]),
    "mr_attn_prefill": (C.c_int, [_vp, _u32, _H, _u32, _H, _H, _u32, _u32, _vp, _vp, C.POINTER(AttnOpts), _H]),
})


class Heads:
    """Rows [tokens, n_heads, head_dim] of a device buffer or address (mr_heads); strides in elements,
    0 for dense rows."""

    def __init__(self, data, n_heads: int, dtype: int = F32, token_stride: int = 0, head_stride: int = 0):
        self._keep = data
        self.c = CHeads(_ptr(data), dtype, n_heads, token_stride, head_stride)


def _heads(h: Heads | None):
    return None if h is None else C.byref(h.c)


def _opts(scale: float, window: int, sinks) -> AttnOpts:
    return AttnOpts(scale, window, _ptr(sinks))


class Rope:
    """Rotary frequencies of a model (mr_rope)."""

    def __init__(self, ctx: Context, head_dim: int, *, rotary_dim: int = 0, base: float = 10000.0,
                 layout: int = ROPE_HALF, scaling: int = ROPE_PLAIN, factor: float = 1.0, orig_context: int = 0,
                 beta_fast: float = 0.0, beta_slow: float = 0.0, attn_factor: float = 0.0):
        d = RopeDesc(head_dim, rotary_dim, layout, scaling, base, factor, orig_context, beta_fast, beta_slow, attn_factor)
        h = _vp()
        ctx.check(_lib.mr_rope_create(ctx.h, C.byref(d), C.byref(h)))
        self.ctx, self.h, self.head_dim = ctx, h.value, head_dim

    def frequencies(self) -> tuple[np.ndarray, float]:
        """Radians per position of each pair, and the factor on cosine and sine."""
        n, mul = _u32(), _f32()
        p = _lib.mr_rope_frequencies(self.h, C.byref(n), C.byref(mul))
        return np.ctypeslib.as_array(p, (n.value,)).copy(), float(mul.value)

    def close(self) -> None:
        if self.h:
            _lib.mr_rope_destroy(self.h)
            self.h = None


def qk_norm_rope(ctx: Context, rope: Rope, q: Heads, k: Heads | None, n_tokens: int, positions, q_out: Heads,
                 k_out: Heads | None, *, q_norm=None, k_norm=None, eps: float = 0.0) -> None:
    """mr_qk_norm_rope: the heads' RMSNorm (where a weight is given), then the rotation by positions."""
    ctx.check(_lib.mr_qk_norm_rope(ctx.h, rope.h, _heads(q), _heads(k), _ptr(q_norm), _ptr(k_norm), eps,
                                   _ptr(positions), n_tokens, _heads(q_out), _heads(k_out)))


class KvCache:
    """One layer's paged cache of keys and values (mr_kv)."""

    def __init__(self, ctx: Context, fmt: int, n_pages: int, page_size: int, n_heads: int, head_dim: int):
        d = KvDesc(fmt, n_pages, page_size, n_heads, head_dim)
        h = _vp()
        ctx.check(_lib.mr_kv_create(ctx.h, C.byref(d), C.byref(h)))
        self.ctx, self.h, self.desc = ctx, h.value, d

    @staticmethod
    def nbytes(fmt: int, n_pages: int, page_size: int, n_heads: int, head_dim: int) -> int:
        """Device bytes of such a cache, 0 for one that cannot be created."""
        return int(_lib.mr_kv_bytes(C.byref(KvDesc(fmt, n_pages, page_size, n_heads, head_dim))))

    def write(self, k: Heads, v: Heads, n_tokens: int, slots) -> None:
        """mr_kv_write: token t into slot slots[t]; negative slots are left out."""
        self.ctx.check(_lib.mr_kv_write(self.ctx.h, self.h, _heads(k), _heads(v), n_tokens, _ptr(slots)))

    def read(self, n_tokens: int, slots, k: Heads | None, v: Heads | None) -> None:
        """mr_kv_read: the values of slot slots[t] to token t; zeros for negative slots."""
        self.ctx.check(_lib.mr_kv_read(self.ctx.h, self.h, n_tokens, _ptr(slots), _heads(k), _heads(v)))

    def attend(self, q: Heads, n_seqs: int, seq_len, block_table, max_pages: int, out: Heads, *, scale: float = 0.0,
               window: int = 0, sinks=None) -> None:
        """mr_attn_decode: one query token of each sequence over its cached tokens."""
        o = _opts(scale, window, sinks)
        self.ctx.check(_lib.mr_attn_decode(self.ctx.h, self.h, _heads(q), n_seqs, _ptr(seq_len), _ptr(block_table),
                                           max_pages, C.byref(o), _heads(out)))

    def extend(self, q: Heads, n_q: int, n_seqs: int, cu_q, seq_len, block_table, max_pages: int, out: Heads, *,
               scale: float = 0.0, window: int = 0, sinks=None) -> None:
        """mr_attn_extend: the packed new tokens of each sequence over its cached tokens, themselves among them."""
        o = _opts(scale, window, sinks)
        self.ctx.check(_lib.mr_attn_extend(self.ctx.h, self.h, _heads(q), n_q, n_seqs, _ptr(cu_q), _ptr(seq_len),
                                           _ptr(block_table), max_pages, C.byref(o), _heads(out)))

    def close(self) -> None:
        if self.h:
            _lib.mr_kv_destroy(self.h)
            self.h = None


def attn_prefill(ctx: Context, head_dim: int, q: Heads, k: Heads, v: Heads, n_q: int, n_k: int, n_seqs: int, cu_q,
                 cu_k, out: Heads, *, scale: float = 0.0, window: int = 0, sinks=None) -> None:
    """mr_attn_prefill: causal attention over packed prompts."""
    o = _opts(scale, window, sinks)
    ctx.check(_lib.mr_attn_prefill(ctx.h, head_dim, _heads(q), n_q, _heads(k), _heads(v), n_k, n_seqs, _ptr(cu_q),
                                   _ptr(cu_k), C.byref(o), _heads(out)))
