// mr_api_common.h -- argument checks that the C ABIs of the attention side and of kept states share.
#pragma once

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "mr_attn.h"

namespace mr {
namespace api {

inline int fail(mr_ctx* c, int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(c, code, buf);
}

inline int hip_fail(mr_ctx* c, hipError_t e, const char* what) {
  return fail(c, e == hipErrorOutOfMemory ? MR_E_NOMEM : MR_E_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// Makes the context's device current for this host thread.
inline int bind(mr_ctx* c) {
  if (c->device < 0) return fail(c, MR_E_NODEV, "host-only context");
  int cur = -1;
  if (hipGetDevice(&cur) != hipSuccess) return fail(c, MR_E_LAUNCH, "hipGetDevice failed");
  if (cur != c->device) {
    const hipError_t e = hipSetDevice(c->device);
    if (e != hipSuccess) return hip_fail(c, e, "hipSetDevice");
  }
  return MR_OK;
}

// Whether work on the context's stream is being captured, by mr_graph_begin or by the stream's owner.
inline bool capturing(mr_ctx* c) {
  if (c->capturing) return true;
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(c->stream, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

inline bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

inline uint32_t elem_bytes(uint32_t dtype) { return dtype == MR_F32 ? 4 : 2; }

// Checks rows of heads and fills in the default strides.
inline int take(mr_ctx* c, const char* name, const mr_heads* h, uint32_t D, Heads* out) {
  if (!h || !h->data) return fail(c, MR_E_INVAL, "%s is NULL", name);
  if (h->dtype > MR_BF16) return fail(c, MR_E_INVAL, "%s: type %u unknown", name, h->dtype);
  if (h->n_heads == 0 || h->n_heads > 1024) return fail(c, MR_E_INVAL, "%s: %u heads, not 1..1024", name, h->n_heads);
  const uint32_t per16 = 16 / elem_bytes(h->dtype);
  out->p = h->data, out->dtype = h->dtype, out->n = h->n_heads;
  out->hs = h->head_stride ? h->head_stride : D;
  out->ts = h->token_stride ? h->token_stride : (uint64_t)h->n_heads * D;
  if (misaligned(h->data, 16) || out->hs % per16 || out->ts % per16)
    return fail(c, MR_E_INVAL, "%s must be 16-byte aligned, its strides multiples of 16 bytes", name);
  if (out->hs >= 1ull << 40 || out->ts >= 1ull << 40) return fail(c, MR_E_INVAL, "%s: a stride of 2^40 elements or more", name);
  return MR_OK;
}

inline int check_kv(mr_ctx* c, const mr_kv* kv) {
  if (!kv) return fail(c, MR_E_INVAL, "cache is NULL");
  if (kv->ctx != c) return fail(c, MR_E_INVAL, "cache belongs to another context");
  return MR_OK;
}

inline KvPages pages(const mr_kv* kv) {
  uint32_t shift = 6;
  while ((1u << shift) < kv->d.page_size) ++shift;
  return KvPages{kv->base, kv->d.n_pages, shift, kv->d.n_heads, kv_chunk_bytes(kv->d.format, kv->d.head_dim)};
}

inline int take_opts(mr_ctx* c, const mr_attn_opts* o, uint32_t D, AttnOpts* out) {
  out->scale = o && o->scale != 0.f ? o->scale : 1.f / std::sqrt((float)D);
  out->window = o ? o->window : 0;
  out->sinks = o ? o->sinks : nullptr;
  if (!std::isfinite(out->scale)) return fail(c, MR_E_INVAL, "scale is not finite");
  if (misaligned(out->sinks, 4)) return fail(c, MR_E_INVAL, "sinks must be 4-byte aligned");
  return MR_OK;
}

// Query and output of an attention call: one 16-bit type, heads in whole groups.
inline int check_qo(mr_ctx* c, const Heads& q, const Heads& out, uint32_t n_kv) {
  if (q.dtype == MR_F32 || out.dtype != q.dtype)
    return fail(c, MR_E_UNSUPPORTED, "q and out must be both F16 or both BF16");
  if (out.n != q.n) return fail(c, MR_E_INVAL, "out has %u heads, q %u", out.n, q.n);
  if (q.n % n_kv) return fail(c, MR_E_INVAL, "%u query heads do not share %u key heads evenly", q.n, n_kv);
  return MR_OK;
}

// Lengths and pages of an attention call over a cache.
inline int check_lengths(mr_ctx* c, const mr_kv* kv, const int32_t* seq_len, const int32_t* block_table, uint32_t max_pages, uint32_t n_seqs) {
  if (!seq_len || !block_table || misaligned(seq_len, 4) || misaligned(block_table, 4))
    return fail(c, MR_E_INVAL, "seq_len or block_table is NULL or not 4-byte aligned");
  if (max_pages == 0 || (uint64_t)max_pages * kv->d.page_size > 0x7FFFFFFFull)
    return fail(c, MR_E_INVAL, "max_pages %u of %u tokens are not 1 .. 2^31 - 1 tokens", max_pages, kv->d.page_size);
  if (n_seqs > 65535) return fail(c, MR_E_INVAL, "n_seqs %u is above 65535", n_seqs);
  return MR_OK;
}

}  // namespace api
}  // namespace mr
