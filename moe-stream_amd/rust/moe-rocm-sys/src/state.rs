//! Raw declarations of include/moe_rocm_state.h: new tokens of many sequences over what those sequences keep.
//!
//! Attention of packed chunks over the paged cache, and the short causal convolution and gated delta rule of a
//! layer whose attention is linear (deltanet_forward, deltanet.rs:148-543).

use crate::attn::{mr_attn_opts, mr_heads, mr_kv};
use crate::mr_ctx;
use core::ffi::{c_int, c_void};

#[repr(C)]
pub struct mr_delta {
    _p: [u8; 0],
}

/// Rows [tokens, width]; stride in elements, 0 for dense rows.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_rows {
    pub data: *mut c_void,
    pub dtype: u32,
    pub width: u32,
    pub stride: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_delta_desc {
    pub n_key_heads: u32,
    pub n_value_heads: u32,
    pub key_dim: u32,
    pub value_dim: u32,
    pub scale: f32,
    pub unit_eps: f32,
    pub gate_stride: u64,
    pub a_log: *const f32,
    pub dt_bias: *const f32,
}

#[rustfmt::skip]
extern "C" {
    pub fn mr_attn_extend(ctx: *mut mr_ctx, kv: *const mr_kv, q: *const mr_heads, n_q: u32, n_seqs: u32, cu_q: *const i32, seq_len: *const i32, block_table: *const i32, max_pages: u32, opts: *const mr_attn_opts, out: *const mr_heads) -> c_int;
    pub fn mr_causal_conv(ctx: *mut mr_ctx, x: *const mr_rows, w: *const f32, taps: u32, bias: *const f32, silu: u32, n_tokens: u32, n_seqs: u32, cu: *const i32, states: *mut f32, n_slots: u32, source: *const i32, target: *const i32, out: *const mr_rows) -> c_int;
    pub fn mr_delta_create(ctx: *mut mr_ctx, desc: *const mr_delta_desc, out: *mut *mut mr_delta) -> c_int;
    pub fn mr_delta_destroy(delta: *mut mr_delta);
    pub fn mr_delta_rule(ctx: *mut mr_ctx, delta: *const mr_delta, q: *const mr_heads, k: *const mr_heads, v: *const mr_heads, decay: *const f32, beta: *const f32, n_tokens: u32, n_seqs: u32, cu: *const i32, states: *mut f32, n_slots: u32, source: *const i32, target: *const i32, out: *const mr_heads) -> c_int;
}
