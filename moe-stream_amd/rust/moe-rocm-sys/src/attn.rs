//! Raw declarations of include/moe_rocm_attn.h: the attention side of a decoder layer.
//!
//! The steps between the QKV and the output projection (run_attention, layer.rs:511-755): norms and
//! rotary positions of the heads, the paged cache, attention over it and over packed prompts.

use crate::mr_ctx;
use core::ffi::{c_int, c_void};

// ---- element types
pub const MR_F32: u32 = 0;
pub const MR_F16: u32 = 1;
pub const MR_BF16: u32 = 2;

// ---- rotary positions
pub const MR_ROPE_HALF: u32 = 0;
pub const MR_ROPE_INTERLEAVED: u32 = 1;
pub const MR_ROPE_PLAIN: u32 = 0;
pub const MR_ROPE_LINEAR: u32 = 1;
pub const MR_ROPE_YARN: u32 = 2;
pub const MR_ROPE_YARN_EXACT: u32 = 3;

// ---- cache formats
pub const MR_KV_F16: u32 = 16;
pub const MR_KV_MXINT8: u32 = 8;
pub const MR_KV_MXFP4: u32 = 4;

#[repr(C)]
pub struct mr_rope {
    _p: [u8; 0],
}
#[repr(C)]
pub struct mr_kv {
    _p: [u8; 0],
}

/// Rows [tokens, n_heads, head_dim]; strides in elements, 0 for dense rows.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_heads {
    pub data: *mut c_void,
    pub dtype: u32,
    pub n_heads: u32,
    pub token_stride: u64,
    pub head_stride: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_rope_desc {
    pub head_dim: u32,
    pub rotary_dim: u32,
    pub layout: u32,
    pub scaling: u32,
    pub base: f64,
    pub factor: f64,
    pub orig_context: u32,
    pub beta_fast: f32,
    pub beta_slow: f32,
    pub attn_factor: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_kv_desc {
    pub format: u32,
    pub n_pages: u32,
    pub page_size: u32,
    pub n_heads: u32,
    pub head_dim: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mr_attn_opts {
    pub scale: f32,
    pub window: u32,
    pub sinks: *const f32,
}

extern "C" {
    pub fn mr_rope_create(ctx: *mut mr_ctx, desc: *const mr_rope_desc, out: *mut *mut mr_rope) -> c_int;
    pub fn mr_rope_destroy(rope: *mut mr_rope);
    pub fn mr_rope_frequencies(rope: *const mr_rope, n: *mut u32, attn_factor: *mut f32) -> *const f64;
    pub fn mr_qk_norm_rope(
        ctx: *mut mr_ctx,
        rope: *const mr_rope,
        q: *const mr_heads,
        k: *const mr_heads,
        q_norm: *const f32,
        k_norm: *const f32,
        eps: f32,
        positions: *const i32,
        n_tokens: u32,
        q_out: *const mr_heads,
        k_out: *const mr_heads,
    ) -> c_int;
    pub fn mr_kv_create(ctx: *mut mr_ctx, desc: *const mr_kv_desc, out: *mut *mut mr_kv) -> c_int;
    pub fn mr_kv_destroy(kv: *mut mr_kv);
    pub fn mr_kv_bytes(desc: *const mr_kv_desc) -> u64;
    pub fn mr_kv_write(
        ctx: *mut mr_ctx,
        kv: *mut mr_kv,
        k: *const mr_heads,
        v: *const mr_heads,
        n_tokens: u32,
        slots: *const i32,
    ) -> c_int;
    pub fn mr_kv_read(
        ctx: *mut mr_ctx,
        kv: *const mr_kv,
        n_tokens: u32,
        slots: *const i32,
        k: *const mr_heads,
        v: *const mr_heads,
    ) -> c_int;
    pub fn mr_attn_decode(
        ctx: *mut mr_ctx,
        kv: *const mr_kv,
        q: *const mr_heads,
        n_seqs: u32,
        seq_len: *const i32,
        block_table: *const i32,
        max_pages: u32,
        opts: *const mr_attn_opts,
        out: *const mr_heads,
    ) -> c_int;
    pub fn mr_attn_prefill(
        ctx: *mut mr_ctx,
        head_dim: u32,
        q: *const mr_heads,
        n_q: u32,
        k: *const mr_heads,
        v: *const mr_heads,
        n_k: u32,
        n_seqs: u32,
        cu_q: *const i32,
        cu_k: *const i32,
        opts: *const mr_attn_opts,
        out: *const mr_heads,
    ) -> c_int;
}
