// mr_state_api.cpp -- C ABI of include/moe_rocm_state.h: handles, argument validation and dispatch. Arguments are
// checked before the device is touched, so a host-only context (MR_DEVICE_NONE) exercises every refusal
// without a GPU.
#include <cmath>
#include <new>

#include "mr_api_common.h"
#include "mr_state.h"

using namespace mr::api;

namespace {

constexpr uint32_t kMaxRows = (1u << 24) - 1;

int take_rows(mr_ctx* c, const char* name, const mr_rows* r, mr::RowsOf* out) {
  if (!r || !r->data) return fail(c, MR_E_INVAL, "%s is NULL", name);
  if (r->dtype > MR_BF16) return fail(c, MR_E_INVAL, "%s: type %u unknown", name, r->dtype);
  if (r->width == 0 || r->width % 8 || r->width > 1u << 20)
    return fail(c, MR_E_INVAL, "%s: width %u is not a multiple of 8 up to 2^20", name, r->width);
  out->p = r->data, out->dtype = r->dtype, out->width = r->width;
  out->stride = r->stride ? r->stride : r->width;
  if (misaligned(r->data, 16) || out->stride % (16 / elem_bytes(r->dtype)))
    return fail(c, MR_E_INVAL, "%s must be 16-byte aligned, its stride a multiple of 16 bytes", name);
  if (out->stride >= 1ull << 40) return fail(c, MR_E_INVAL, "%s: a stride of 2^40 elements or more", name);
  return MR_OK;
}

int take_sequences(mr_ctx* c, uint32_t n_rows, uint32_t n_seqs, const int32_t* cu, float* states, uint32_t n_slots,
                   const int32_t* source, const int32_t* target, mr::Sequences* out) {
  if (!cu || misaligned(cu, 4)) return fail(c, MR_E_INVAL, "cu is NULL or not 4-byte aligned");
  if (n_rows > kMaxRows) return fail(c, MR_E_INVAL, "n_tokens %u is 2^24 or more", n_rows);
  if (n_seqs > 65535) return fail(c, MR_E_INVAL, "n_seqs %u is above 65535", n_seqs);
  if (misaligned(source, 4) || misaligned(target, 4)) return fail(c, MR_E_INVAL, "source or target is not 4-byte aligned");
  if ((source || target) && (!states || misaligned(states, 16)))
    return fail(c, MR_E_INVAL, "states is NULL or not 16-byte aligned");
  if (n_slots > 0x7FFFFFFFu) return fail(c, MR_E_INVAL, "2^31 slots or more");
  *out = mr::Sequences{cu, n_seqs, (int)n_rows, states, n_slots, source, target, c->attn_err};
  return MR_OK;
}

}  // namespace

extern "C" {

int mr_attn_extend(mr_ctx* c, const mr_kv* kv, const mr_heads* q, uint32_t nq, uint32_t n_seqs, const int32_t* cu_q,
                   const int32_t* seq_len, const int32_t* block_table, uint32_t max_pages, const mr_attn_opts* opts,
                   const mr_heads* out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  int rc = check_kv(c, kv);
  if (rc) return rc;
  mr::Heads hq, ho;
  mr::AttnOpts o;
  const uint32_t D = kv->d.head_dim;
  if ((rc = take(c, "q", q, D, &hq)) || (rc = take(c, "out", out, D, &ho)) || (rc = check_qo(c, hq, ho, kv->d.n_heads)) ||
      (rc = take_opts(c, opts, D, &o)))
    return rc;
  if (!cu_q || misaligned(cu_q, 4)) return fail(c, MR_E_INVAL, "cu_q is NULL or not 4-byte aligned");
  if ((rc = check_lengths(c, kv, seq_len, block_table, max_pages, n_seqs))) return rc;
  if ((uint64_t)nq * (hq.n / kv->d.n_heads) > kMaxRows)
    return fail(c, MR_E_INVAL, "%u rows of %u heads that share keys are 2^24 or more", nq, hq.n / kv->d.n_heads);
  if (((uint64_t)nq * (hq.n / kv->d.n_heads) / 16 + n_seqs + 2048) * kv->d.n_heads >= 1u << 24)  // 2^32 threads of a launch
    return fail(c, MR_E_INVAL, "%u rows in %u sequences are too many tiles for %u key heads", nq, n_seqs, kv->d.n_heads);
  if (nq == 0 || n_seqs == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_attn_extend(c->launch(), pages(kv), kv->d.format, D, hq, nq, n_seqs, cu_q, seq_len,
                                              block_table, max_pages, o, ho, c->attn_err, c->attn_scratch, c->n_cu);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "attn_extend launch");
}

int mr_causal_conv(mr_ctx* c, const mr_rows* x, const float* w, uint32_t taps, const float* bias, uint32_t silu,
                   uint32_t n_tokens, uint32_t n_seqs, const int32_t* cu, float* states, uint32_t n_slots,
                   const int32_t* source, const int32_t* target, const mr_rows* out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  mr::RowsOf rx, ro;
  mr::Sequences s;
  int rc;
  if ((rc = take_rows(c, "x", x, &rx)) || (rc = take_rows(c, "out", out, &ro))) return rc;
  if (ro.width != rx.width) return fail(c, MR_E_INVAL, "out has %u channels, x %u", ro.width, rx.width);
  if (taps < 2 || taps > 4) return fail(c, MR_E_UNSUPPORTED, "%u taps, not 2 to 4", taps);
  if (!w || misaligned(w, 16) || misaligned(bias, 16)) return fail(c, MR_E_INVAL, "w is NULL, or w or bias not 16-byte aligned");
  if (silu > 1) return fail(c, MR_E_INVAL, "silu %u is not 0 or 1", silu);
  if ((rc = take_sequences(c, n_tokens, n_seqs, cu, states, n_slots, source, target, &s))) return rc;
  if (n_seqs == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_causal_conv(c->launch(), rx, w, taps, bias, silu != 0, s, ro);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "causal_conv launch");
}

int mr_delta_create(mr_ctx* c, const mr_delta_desc* desc, mr_delta** out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (!out) return fail(c, MR_E_INVAL, "out pointer is NULL");
  *out = nullptr;
  if (!desc) return fail(c, MR_E_INVAL, "delta description is NULL");
  mr_delta_desc d = *desc;
  if (d.n_key_heads == 0 || d.n_value_heads == 0 || d.n_value_heads > 256 || d.n_value_heads % d.n_key_heads)
    return fail(c, MR_E_INVAL, "%u value heads do not share %u key heads evenly, or are not 1..256", d.n_value_heads, d.n_key_heads);
  if ((d.key_dim != 64 && d.key_dim != 128) || (d.value_dim != 64 && d.value_dim != 128))
    return fail(c, MR_E_UNSUPPORTED, "key_dim %u or value_dim %u is not 64 or 128", d.key_dim, d.value_dim);
  if (!std::isfinite(d.scale)) return fail(c, MR_E_INVAL, "scale is not finite");
  if (d.scale == 0.f) d.scale = 1.f / std::sqrt((float)d.key_dim);
  if (!(d.unit_eps >= 0.f) || d.unit_eps > 1.f) return fail(c, MR_E_INVAL, "unit_eps %g is not in [0, 1]", (double)d.unit_eps);
  if (d.gate_stride == 0) d.gate_stride = d.n_value_heads;
  if (d.gate_stride < d.n_value_heads || d.gate_stride >= 1ull << 40)
    return fail(c, MR_E_INVAL, "gate_stride %llu is below the value heads, or 2^40 or more", (unsigned long long)d.gate_stride);
  if (!d.a_log != !d.dt_bias) return fail(c, MR_E_INVAL, "only one of a_log and dt_bias is given");
  if (misaligned(d.a_log, 4) || misaligned(d.dt_bias, 4)) return fail(c, MR_E_INVAL, "a_log or dt_bias is not 4-byte aligned");
  if (c->device >= 0 && capturing(c)) return fail(c, MR_E_INVAL, "allocation during graph capture");
  if (c->device >= 0 && !c->delta_scratch) {
    int rc = bind(c);
    if (rc) return rc;
    const hipError_t e = hipMalloc(&c->delta_scratch, mr::delta_scratch_bytes());
    if (e != hipSuccess) return hip_fail(c, e, "delta workspace");
  }
  mr_delta* r = new (std::nothrow) mr_delta;
  if (!r) return fail(c, MR_E_NOMEM, "host allocation failed");
  r->ctx = c, r->d = d;
  *out = r;
  return MR_OK;
}

void mr_delta_destroy(mr_delta* r) { delete r; }

int mr_delta_rule(mr_ctx* c, const mr_delta* r, const mr_heads* q, const mr_heads* k, const mr_heads* v, const float* decay,
                  const float* beta, uint32_t n_tokens, uint32_t n_seqs, const int32_t* cu, float* states, uint32_t n_slots,
                  const int32_t* source, const int32_t* target, const mr_heads* out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (!r) return fail(c, MR_E_INVAL, "delta is NULL");
  if (r->ctx != c) return fail(c, MR_E_INVAL, "delta belongs to another context");
  const mr_delta_desc& d = r->d;
  mr::Heads hq, hk, hv, ho;
  mr::Sequences s;
  int rc;
  if ((rc = take(c, "q", q, d.key_dim, &hq)) || (rc = take(c, "k", k, d.key_dim, &hk)) ||
      (rc = take(c, "v", v, d.value_dim, &hv)) || (rc = take(c, "out", out, d.value_dim, &ho)))
    return rc;
  if (hq.dtype == MR_F32 || hk.dtype != hq.dtype || hv.dtype != hq.dtype || ho.dtype != hq.dtype)
    return fail(c, MR_E_UNSUPPORTED, "q, k, v and out must be all F16 or all BF16");
  if (hq.n != d.n_key_heads || hk.n != d.n_key_heads || hv.n != d.n_value_heads || ho.n != d.n_value_heads)
    return fail(c, MR_E_INVAL, "heads of q, k, v and out are %u, %u, %u, %u, not %u, %u, %u, %u", hq.n, hk.n, hv.n, ho.n,
                d.n_key_heads, d.n_key_heads, d.n_value_heads, d.n_value_heads);
  for (const mr::Heads* x : {&hq, &hk, &hv, &ho})  // 64 rows within 32-bit offsets
    if (x->ts >= 1ull << 24) return fail(c, MR_E_INVAL, "q, k, v or out has a token stride of 2^24 elements or more");
  if (!decay || !beta || misaligned(decay, 4) || misaligned(beta, 4))
    return fail(c, MR_E_INVAL, "decay or beta is NULL or not 4-byte aligned");
  if ((rc = take_sequences(c, n_tokens, n_seqs, cu, states, n_slots, source, target, &s))) return rc;
  if (n_seqs == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const mr::DeltaShape shape{d.n_key_heads, d.n_value_heads, d.key_dim, d.value_dim, d.scale, d.unit_eps, d.gate_stride, d.a_log, d.dt_bias};
  const hipError_t e = mr::launch_delta_rule(c->launch(), shape, hq, hk, hv, decay, beta, s, ho, c->delta_scratch);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "delta_rule launch");
}

}  // extern "C"
