/*
 * moe_rocm_state.h -- C ABI of what takes new tokens of many sequences over what those sequences keep, on
 * the MI355X (gfx950): attention of packed chunks over the paged cache of moe_rocm_attn.h, and the two steps of
 * a layer whose attention is linear, the short causal convolution and the gated delta rule, over states (the
 * reference's deltanet_forward, deltanet.rs:148-543). Contexts, status codes, streams, graphs and conventions are
 * those of moe_rocm.h and moe_rocm_attn.h.
 *
 *   mr_attn_extend   the next tokens of each sequence over the cache, which holds them already
 *   mr_causal_conv   a causal convolution of a few tokens' width for each channel
 *   mr_delta_rule    linear attention whose state is corrected, not added to
 *
 * Further conventions
 *  - New tokens are packed: sequence s has rows cu[s] .. cu[s + 1] - 1 of the n rows of a call, one token or
 *    many, or none; cu holds n_seqs + 1 offsets that do not decrease. Rows of an output in no sequence are left as they
 *    are. Offsets outside the rows are taken as the nearest inside, with an error at mr_sync. Decreasing ones end in an
 *    error too, and the call's rows of output and target states then hold a result, some mixture of results, or what was there
 *    before, those of sequences behind and before the offset among them; nothing else is written.
 *  - States are the caller's: n_slots of them, f32, dense, 16-byte aligned. Sequence s starts from the state of
 *    slot source[s], from zeros if that is negative, and leaves its last one in slot target[s], nowhere if that
 *    is negative. The two may be one slot, or two: the state before a draft that is not taken is then still
 *    there. source and target may be NULL, for negative ones throughout, and states where both are. A slot past the
 *    last is taken as a negative one, with an error at mr_sync. No slot is another sequence's target in the
 *    same call: it would hold some mixture. A sequence without tokens takes its state from source to target.
 *  - Kernel names for mr_profile_read: "attn_extend", "extend_join", "causal_conv", "delta_step", "delta_list",
 *    "delta_prepare", "delta_chunks".
 */
#ifndef MOE_ROCM_STATE_H
#define MOE_ROCM_STATE_H

#include "moe_rocm_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- attention of new tokens over the cache ---------------------------------------- */
/* Rows of q and out are packed as above (F16 or BF16, both the same); sequence s has seq_len[s] tokens in the
 * cache, its new ones (the last of them) among them, placed as for mr_attn_decode. Its i-th of n rows stands
 * at position seq_len[s] - n + i and sees the keys at its own and at earlier positions, with a window the last of
 * those; a row before position 0, of more new tokens than cached ones, sees nothing and is zero. Lengths, pages,
 * window, sinks and numerics are mr_attn_decode's; where sequences have more than 32 rows (new tokens times the
 * query heads of a key head) on average, weights keep their 11 bits down to 2^-25 of the largest only. n_seqs: up to
 * 65535; n_q times the query heads of a key head: below 2^24; a sixteenth of that, n_seqs and 2048, times the key
 * heads: below 2^24 (more is refused). opts NULL: defaults. Shares its scratch with mr_attn_decode: one call of a
 * context at a time.
 *
 * Long sequences are spread over the CUs in calls of up to 1024 sequences; in others a tile of rows is one workgroup's for each key
 * head: 100,001 tokens among 1023 and among 1024 others of one token take 0.24 and 0.50 ms (MXFP4, 4 heads of 128), 0.37 and
 * 1.16 ms (MXINT8, 2 of 256). */
int mr_attn_extend(mr_ctx* ctx, const mr_kv* kv, const mr_heads* q, uint32_t n_q, uint32_t n_seqs, const int32_t* cu_q,
                   const int32_t* seq_len, const int32_t* block_table, uint32_t max_pages, const mr_attn_opts* opts,
                   const mr_heads* out);

/* ---- short causal convolution (deltanet.rs:204-330) --------------------------------- */
/* Rows [tokens, width] of any type; the elements of a row are adjacent. data 16-byte aligned, stride (elements; 0:
 * width) a multiple of 16 bytes. */
typedef struct mr_rows {
  void* data;
  uint32_t dtype; /* MR_F32, MR_F16, MR_BF16 */
  uint32_t width; /* multiple of 8, up to 2^20 */
  uint64_t stride;
} mr_rows;

/* out_t = act(bias + sum_j w[c][j] x_(t - taps + 1 + j)) for each channel c and token t, 2 <= taps <= 4; act is
 * x / (1 + exp(-x)) with silu, else none. w: f32 [channels, taps], bias: f32 [channels] or NULL, both 16-byte aligned.
 * A state is the last taps - 1 inputs, the oldest first: f32 [taps - 1, channels]. Sums in 32 bits. Types of x and
 * out are free; out overlaps no input. n_tokens: up to 2^24 - 1; n_seqs: up to 65535. */
int mr_causal_conv(mr_ctx* ctx, const mr_rows* x, const float* w, uint32_t taps, const float* bias, uint32_t silu,
                   uint32_t n_tokens, uint32_t n_seqs, const int32_t* cu, float* states, uint32_t n_slots,
                   const int32_t* source, const int32_t* target, const mr_rows* out);

/* ---- gated delta rule (deltanet.rs:330-543) ------------------------------------------- */
typedef struct mr_delta_desc {
  uint32_t n_key_heads;   /* heads of q and k */
  uint32_t n_value_heads; /* a multiple; value head h goes with key head h / (value heads / key heads); up to 256 */
  uint32_t key_dim;       /* 64 or 128 */
  uint32_t value_dim;     /* 64 or 128 */
  float scale;            /* 0: 1 / sqrt(key_dim) */
  float unit_eps;         /* above 0 (up to 1): rows of q and k are divided by sqrt(sum of squares + unit_eps) first */
  uint64_t gate_stride;   /* elements between the tokens of decay and beta; 0: n_value_heads */
  const float* a_log;     /* f32 [n_value_heads], or NULL. Given (with dt_bias): decay holds raw a, beta raw b, and */
  const float* dt_bias;   /* g = -exp(a_log) ln(1 + exp(a + dt_bias)), beta = 1 / (1 + exp(-b)). Borrowed. */
} mr_delta_desc;

typedef struct mr_delta mr_delta;

/* One layer's rule. Allocates the context's workspace for long sequences (256 MiB, all rules' calls in turn) with the
 * first one. */
int mr_delta_create(mr_ctx* ctx, const mr_delta_desc* desc, mr_delta** out);
void mr_delta_destroy(mr_delta* delta);
/* For each value head, a state S [key_dim, value_dim] (f32, a slot is [n_value_heads, key_dim, value_dim]) and token t
 * with its key k, query q, value v, g = decay (a log: 0 or less, -infinity among them) and beta:
 *   S' = exp(g) S, S = S' + beta k (v - S'^T k)^T, out = scale S^T q.
 * q, k, v and out: F16 or BF16, all the same, token strides below 2^24 elements; decay, beta: f32 [tokens, value
 * heads] with gate_stride. States, sums, and all that the next state comes from are held to 32 bits or the like:
 * products of more than a few tokens run on 16-bit matrix instructions in three parts of 8 bits a number, those for
 * out alone in two, and out is rounded once. Decays above 0 (growth) are taken as they are; 64 tokens whose growth is more
 * than a factor of two go one by one, 0.7 us each. -infinity forgets. What is not finite, of the inputs or because 32
 * bits do not hold it, reaches no earlier token: a value makes its column NaN or infinite from its token on; a key,
 * another decay or a beta all columns; a query its own row. Squares of keys stay within 32 bits: elements below 10^18.
 * n_tokens: up to 2^24 - 1; n_seqs: up to 65535. */
int mr_delta_rule(mr_ctx* ctx, const mr_delta* delta, const mr_heads* q, const mr_heads* k, const mr_heads* v,
                  const float* decay, const float* beta, uint32_t n_tokens, uint32_t n_seqs, const int32_t* cu,
                  float* states, uint32_t n_slots, const int32_t* source, const int32_t* target, const mr_heads* out);

#ifdef __cplusplus
}
#endif
#endif /* MOE_ROCM_STATE_H */
