"""New tokens of many sequences over what those sequences keep (include/moe_rocm_state.h): short causal convolutions
and the gated delta rule over states; KvCache.extend (attn.py) is the attention of new tokens over the cache.
Re-exported by moe_rocm.

Arguments are device buffers or addresses. Tokens are packed, `cu` holds the sequences' offsets; `source` and `target`
name the slots that each sequence's state comes from and goes to (negative: zeros, nowhere; None: throughout).
"""
from __future__ import annotations

import ctypes as C

from . import Context, _f32, _lib, _ptr, _register, _u32, _u64, _vp
from .attn import F32, AttnOpts, CHeads, Heads, _heads


class CRows(C.Structure):
    _fields_ = [("data", _vp), ("dtype", _u32), ("width", _u32), ("stride", _u64)]


class DeltaDesc(C.Structure):
    _fields_ = [("n_key_heads", _u32), ("n_value_heads", _u32), ("key_dim", _u32), ("value_dim", _u32), ("scale", _f32),
                ("unit_eps", _f32), ("gate_stride", _u64), ("a_log", _vp), ("dt_bias", _vp)]


_H, _R = C.POINTER(CHeads), C.POINTER(CRows)
_register({
    "mr_attn_extend": (C.c_int, [_vp, _vp, _H, _u32, _u32, _vp, _vp, _vp, _u32, C.POINTER(AttnOpts), _H]),
    "mr_causal_conv": (C.c_int, [_vp, _R, _vp, _u32, _vp, _u32, _u32, _u32, _vp, _vp, _u32, _vp, _vp, _R]),
    "mr_delta_create": (C.c_int, [_vp, C.POINTER(DeltaDesc), C.POINTER(_vp)]),
    "mr_delta_destroy": (None, [_vp]),
    "mr_delta_rule": (C.c_int, [_vp, _vp, _H, _H, _H, _vp, _vp, _u32, _u32, _vp, _vp, _u32, _vp, _vp, _H]),
})


class Rows:
    """Rows [tokens, width] of a device buffer or address (mr_rows); stride in elements, 0 for dense rows."""

    def __init__(self, data, width: int, dtype: int = F32, stride: int = 0):
        self._keep = data
        self.c = CRows(_ptr(data), dtype, width, stride)


def _rows(r: Rows | None):
    return None if r is None else C.byref(r.c)


def causal_conv(ctx: Context, x: Rows, w, taps: int, n_tokens: int, n_seqs: int, cu, out: Rows, *, bias=None,
                silu: bool = False, states=None, n_slots: int = 0, source=None, target=None) -> None:
    """mr_causal_conv: a causal convolution of `taps` tokens for each channel."""
    ctx.check(_lib.mr_causal_conv(ctx.h, _rows(x), _ptr(w), taps, _ptr(bias), int(silu), n_tokens, n_seqs, _ptr(cu),
                                  _ptr(states), n_slots, _ptr(source), _ptr(target), _rows(out)))


class DeltaRule:
    """The gated delta rule of one layer (mr_delta)."""

    def __init__(self, ctx: Context, n_key_heads: int, n_value_heads: int, key_dim: int, value_dim: int, *,
                 scale: float = 0.0, unit_eps: float = 0.0, gate_stride: int = 0, a_log=None, dt_bias=None):
        d = DeltaDesc(n_key_heads, n_value_heads, key_dim, value_dim, scale, unit_eps, gate_stride, _ptr(a_log), _ptr(dt_bias))
        h = _vp()
        ctx.check(_lib.mr_delta_create(ctx.h, C.byref(d), C.byref(h)))
        self.ctx, self.h, self.desc, self._keep = ctx, h.value, d, (a_log, dt_bias)

    def forward(self, q: Heads, k: Heads, v: Heads, decay, beta, n_tokens: int, n_seqs: int, cu, out: Heads, *,
                states=None, n_slots: int = 0, source=None, target=None) -> None:
        """mr_delta_rule over the new tokens of n_seqs sequences."""
        self.ctx.check(_lib.mr_delta_rule(self.ctx.h, self.h, _heads(q), _heads(k), _heads(v), _ptr(decay), _ptr(beta),
                                          n_tokens, n_seqs, _ptr(cu), _ptr(states), n_slots, _ptr(source), _ptr(target),
                                          _heads(out)))

    def close(self) -> None:
        if self.h:
            _lib.mr_delta_destroy(self.h)
            self.h = None
