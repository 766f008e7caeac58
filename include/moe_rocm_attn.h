/*
 * moe_rocm_attn.h -- C ABI of the attention side of a decoder layer on the MI355X (gfx950):
 * the steps between the QKV projection and the output projection, in front of the MoE block of
 * moe_rocm.h (the reference's run_attention, layer.rs:511-755, with ops/attention.rs:9-271 and
 * kv_cache.rs:37-60). Contexts, status codes, streams, graphs and conventions are those of
 * moe_rocm.h.
 *
 *   mr_qk_norm_rope   RMSNorm of each query and key head, then the rotary position
 *   mr_kv_write/read  keys and values into a paged cache of 4, 8 or 16 bits, and back
 *   mr_attn_decode    one query token per sequence over that cache
 *   mr_attn_prefill   causal attention over packed prompts
 *
 * Further conventions
 *  - All arrays are device memory. Row data and norm weights are 16-byte aligned, index and
 *    sink arrays 4-byte aligned. Outputs overlap no input, except where a call says so.
 *  - Index arrays (slots, lengths, pages, offsets) are read on the device, so that captured
 *    graphs see their present values. An entry out of its range is never followed: the call
 *    leaves out what it names, as stated below, and the next mr_sync of the context returns
 *    MR_E_INVAL and says which kind of entry it was.
 *  - Zero tokens, rows or sequences: MR_OK, nothing is launched. More than a launch can hold
 *    (2^24 tokens or more of mr_qk_norm_rope, more than 2^24 - 8 tiles of 128 rows and a head, one of them
 *    for each sequence's last rows, of mr_attn_prefill): MR_E_INVAL.
 *  - mr_attn_decode keeps partial results in scratch of the context, allocated with its first cache and of
 *    one size for all calls: like all scratch of a context it serves one call at a time.
 *  - Kernel names for mr_profile_read: "qk_norm_rope", "kv_write", "kv_read", "attn_decode", "attn_join",
 *    "attn_prefill".
 */
#ifndef MOE_ROCM_ATTN_H
#define MOE_ROCM_ATTN_H

#include "moe_rocm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rows of heads ---------------------------------------------------------- */
#define MR_F32 0
#define MR_F16 1
#define MR_BF16 2

/* Rows [tokens, n_heads, head_dim]; the head_dim elements of a head are adjacent. Strides
 * count elements and are multiples of 16 bytes; 0 stands for dense rows (head_dim, and
 * n_heads * head_dim). A fused QKV projection's output is three views with one token stride. */
typedef struct mr_heads {
  void* data;
  uint32_t dtype;   /* MR_F32, MR_F16, MR_BF16 */
  uint32_t n_heads; /* 1..1024 */
  uint64_t token_stride;
  uint64_t head_stride;
} mr_heads;

/* ---- rotary positions (RoPE tables and partial RoPE, attention.rs:9-176) ------- */
#define MR_ROPE_HALF 0        /* pairs (i, i + rotary_dim / 2) */
#define MR_ROPE_INTERLEAVED 1 /* pairs (2i, 2i + 1) */

#define MR_ROPE_PLAIN 0      /* f_i = base^(-2i / rotary_dim) radians per position */
#define MR_ROPE_LINEAR 1     /* f_i / factor */
#define MR_ROPE_YARN 2       /* YaRN (Peng et al. 2023): f_i / factor for slow pairs, f_i for fast ones, a
                                ramp between the pairs that turn beta_slow and beta_fast times in
                                orig_context positions; these bounds rounded outwards to whole pairs */
#define MR_ROPE_YARN_EXACT 3 /* the same, bounds not rounded (GPT-OSS) */

typedef struct mr_rope_desc {
  uint32_t head_dim;     /* multiple of 8, up to 512 */
  uint32_t rotary_dim;   /* the first rotary_dim elements of a head turn; multiple of 8; 0: all */
  uint32_t layout;       /* MR_ROPE_HALF, MR_ROPE_INTERLEAVED */
  uint32_t scaling;      /* MR_ROPE_PLAIN .. MR_ROPE_YARN_EXACT */
  double base;           /* > 1 */
  double factor;         /* >= 1 (linear, YaRN; 0 with MR_ROPE_PLAIN) */
  uint32_t orig_context; /* YaRN: positions of the original training */
  float beta_fast;       /* YaRN: 0 stands for 32 */
  float beta_slow;       /* YaRN: 0 stands for 1 */
  float attn_factor;     /* factor on cosine and sine; 0: 0.1 ln(factor) + 1 with YaRN, else 1 */
} mr_rope_desc;

typedef struct mr_rope mr_rope;

/* Computes the frequencies (64 bits) and uploads them. */
int mr_rope_create(mr_ctx* ctx, const mr_rope_desc* desc, mr_rope** out);
void mr_rope_destroy(mr_rope* rope);
/* The rotary_dim / 2 frequencies in radians per position, and the factor on cosine and sine;
 * host memory, valid until mr_rope_destroy. */
const double* mr_rope_frequencies(const mr_rope* rope, uint32_t* n, float* attn_factor);

/* For each token t and head: x = in (RMSNorm over head_dim with weight w and eps where w is given:
 * x = in / sqrt(mean(in^2) + eps) * w, the squares summed in 32 bits, which magnitudes beyond 1e18 leave), then
 * the pairs of x turn by positions[t] * f_i. Angles are reduced in 64 bits: any int32 position. q_norm, k_norm:
 * f32 [head_dim] or NULL (no norm);
 * 0 <= eps <= 1. k and k_out: both NULL for queries alone. Types of inputs and outputs are free,
 * q's and k's alike; q_out may be q (k_out k) with the same type and strides. */
int mr_qk_norm_rope(mr_ctx* ctx, const mr_rope* rope, const mr_heads* q, const mr_heads* k, const float* q_norm,
                    const float* k_norm, float eps, const int32_t* positions, uint32_t n_tokens,
                    const mr_heads* q_out, const mr_heads* k_out);

/* ---- paged cache of keys and values (KvCache, kv_cache.rs:37-60) ----------------- */
/* Formats. A block is 32 adjacent elements of one head of one token; its values are code * 2^e with
 * the least e, no less than -16, that fits the block's largest magnitude m. MXFP4: codes 0, 0.5, 1, 1.5,
 * 2, 3, 4, 6 and their negatives, m <= 7 * 2^e, e up to 13; MXINT8: whole numbers -127..127,
 * m < 127.5 * 2^e, e up to 9. Codes are rounded to nearest, ties to the even code. Every value a cache
 * holds is a finite f16 number: magnitudes beyond the largest (49152, 65024; F16: 65504) are stored
 * as the largest, infinities too, and NaN as zero. */
#define MR_KV_F16 16
#define MR_KV_MXINT8 8
#define MR_KV_MXFP4 4

typedef struct mr_kv_desc {
  uint32_t format;    /* MR_KV_* */
  uint32_t n_pages;   /* n_pages * page_size: up to 2^31 - 1 */
  uint32_t page_size; /* tokens of a page: 64, 128, 256, 512 or 1024 */
  uint32_t n_heads;   /* key/value heads, 1..1024 */
  uint32_t head_dim;  /* 64, 128 or 256 */
} mr_kv_desc;

typedef struct mr_kv mr_kv;

/* One layer's cache: n_pages pages of page_size tokens, zeros at first. Slot s is token s % page_size
 * of page s / page_size. */
int mr_kv_create(mr_ctx* ctx, const mr_kv_desc* desc, mr_kv** out);
void mr_kv_destroy(mr_kv* kv);
/* Device bytes of the pages of such a cache; 0 for a description mr_kv_create refuses. */
uint64_t mr_kv_bytes(const mr_kv_desc* desc);
/* Quantises token t of k and v (n_heads heads each, any types) into slot slots[t]. A negative slot
 * leaves the token out; so does one past the last page, with an error at mr_sync. The slots of a call
 * differ from each other: a slot named twice holds some mixture of the tokens. n_tokens of a call, here
 * and below: up to 2^30 - 64. */
int mr_kv_write(mr_ctx* ctx, mr_kv* kv, const mr_heads* k, const mr_heads* v, uint32_t n_tokens,
                const int32_t* slots);
/* The values of slot slots[t] to token t of k and v (any types; either may be NULL): zeros for a
 * negative slot, and for one past the last page, with an error at mr_sync. */
int mr_kv_read(mr_ctx* ctx, const mr_kv* kv, uint32_t n_tokens, const int32_t* slots, const mr_heads* k,
               const mr_heads* v);

/* ---- attention (SDPA with shared heads, sinks and windows, attention.rs:178-271) -- */
/* Query head h reads key/value head h / (query heads / key heads). A position sees the keys at its own
 * and at earlier positions, with window > 0 the last `window` of them, its own among them.
 * out = sum_j p_j v_j, p = softmax(scale * q.k); a sink is one more score of the softmax with no value (-infinity:
 * none; +infinity or NaN: the head's rows are NaN). A row that sees no key is zero.
 *
 * Numerics. Scores, maxima and sums are 32-bit floats; scores of any size that 32 bits hold are right to their
 * own rounding. Weights are rounded to 16 bits for the product with the values, and the divisor is the sum of the
 * rounded ones. Over the cache they are f16: 11 bits down to 2^-28 of the largest, and what lies below 2^-39 of it
 * is dropped. Over prompts they have the inputs' type: f16, 11 bits down to 2^-21 and nothing below 2^-32, or bf16,
 * 8 bits and the range of 32. mr_attn_decode takes a query head as f16 times a power of two: all its bits down to
 * 2^-30 of its largest element. The same call gives the same bits. */
typedef struct mr_attn_opts {
  float scale;        /* 0: 1 / sqrt(head_dim) */
  uint32_t window;    /* 0: all earlier positions */
  const float* sinks; /* f32 [query heads] or NULL */
} mr_attn_opts;

/* One token of each of n_seqs sequences over the cache. q, out: [n_seqs, query heads, head_dim], F16
 * or BF16, both the same; sequence b has seq_len[b] tokens in the cache, its own among them (0: the
 * row is zero), token i in slot block_table[b * max_pages + i / page_size] * page_size + i % page_size.
 * A length below 0 or beyond max_pages * page_size is taken as the nearest that is not, a page out of
 * range as tokens that are not there; both give an error at mr_sync. opts NULL: defaults.
 *
 * Long sequences are spread over the CUs in calls of up to 1024 sequences whose tables hold less than 2^37
 * tokens in all (n_seqs * max_pages * page_size). In others a sequence is one workgroup's for each key head:
 * 100,001 tokens among 1023 and among 1024 others of one token take 0.23 and 0.48 ms (MXFP4, 4 heads of 128), 0.17
 * and 1.2 ms (MXINT8, 2 of 256). Whether a call is split is decided by what the table holds, not by the lengths:
 * for 1280 tokens or less (heads of 256: 512), or a window of 1217 (449) or less, there is one launch and not
 * two (8 sequences of 250 tokens: 7.5 and 10.4 us). */
int mr_attn_decode(mr_ctx* ctx, const mr_kv* kv, const mr_heads* q, uint32_t n_seqs, const int32_t* seq_len,
                   const int32_t* block_table, uint32_t max_pages, const mr_attn_opts* opts, const mr_heads* out);

/* Packed prompts: sequence s has query rows cu_q[s] .. cu_q[s + 1] - 1 of the n_q rows of q and out, and
 * key/value rows cu_k[s] .. cu_k[s + 1] - 1 of the n_k rows of k and v; its queries are its last
 * positions (as many as keys: a whole prompt; fewer: the next part of one; more: the first ones see
 * nothing). cu_q, cu_k: n_seqs + 1 offsets that do not decrease. Offsets outside the rows are taken as
 * the nearest inside and decreasing ones as empty sequences, both with an error at mr_sync; rows that two
 * sequences claim then hold either's result or none. Rows of `out` in no sequence are left as they are.
 * Keys and values that are not finite reach the rows that see them and no others: an element of a row that sees a value of
 * infinity or NaN is one of the two. q, k, v and out: F16 or BF16, all the same; head_dim 64, 128 or 256; token strides
 * of k and v below 2^24 elements. opts NULL: defaults. */
int mr_attn_prefill(mr_ctx* ctx, uint32_t head_dim, const mr_heads* q, uint32_t n_q, const mr_heads* k,
                    const mr_heads* v, uint32_t n_k, uint32_t n_seqs, const int32_t* cu_q, const int32_t* cu_k,
                    const mr_attn_opts* opts, const mr_heads* out);

#ifdef __cplusplus
}
#endif
#endif /* MOE_ROCM_ATTN_H */
