// mr_attn_api.cpp -- C ABI of include/moe_rocm_attn.h: handles, argument validation and dispatch of the
// attention-side operators. Arguments are checked before the device is touched, so a host-only context
// (MR_DEVICE_NONE) exercises every refusal without a GPU.
#include <cmath>
#include <new>

#include "mr_api_common.h"
#include "mr_state.h"

using namespace mr::api;

namespace {

constexpr uint32_t kMaxWork = 1u << 24;  // workgroups of 256 threads that a launch's 2^32 threads allow
constexpr uint32_t kMaxTokens = (kMaxWork - 1) * 64;  // of a cache write or read, 64 to a workgroup

int check_eps(mr_ctx* c, float eps) {
  if (!(eps >= 0.f) || eps > 1.f) return fail(c, MR_E_INVAL, "eps %g is not in [0, 1]", (double)eps);
  return MR_OK;
}

int check_kv_desc(mr_ctx* c, const mr_kv_desc* d) {
  if (!d) return fail(c, MR_E_INVAL, "cache description is NULL");
  if (d->format != MR_KV_F16 && d->format != MR_KV_MXINT8 && d->format != MR_KV_MXFP4)
    return fail(c, MR_E_INVAL, "cache format %u unknown", d->format);
  if (d->page_size < 64 || d->page_size > 1024 || (d->page_size & (d->page_size - 1)))
    return fail(c, MR_E_INVAL, "page size %u is not 64, 128, 256, 512 or 1024", d->page_size);
  if (d->n_pages == 0 || (uint64_t)d->n_pages * d->page_size > 0x7FFFFFFFull)
    return fail(c, MR_E_INVAL, "%u pages of %u tokens are not 1 .. 2^31 - 1 tokens", d->n_pages, d->page_size);
  if (d->n_heads == 0 || d->n_heads > 1024) return fail(c, MR_E_INVAL, "%u heads, not 1..1024", d->n_heads);
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return fail(c, MR_E_UNSUPPORTED, "head_dim %u is not 64, 128 or 256", d->head_dim);
  return MR_OK;
}

}  // namespace

extern "C" {

int mr_rope_create(mr_ctx* c, const mr_rope_desc* desc, mr_rope** out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (!out) return fail(c, MR_E_INVAL, "out pointer is NULL");
  *out = nullptr;
  if (!desc) return fail(c, MR_E_INVAL, "rope description is NULL");
  mr_rope_desc d = *desc;
  if (d.head_dim == 0 || d.head_dim > 512 || d.head_dim % 8)
    return fail(c, MR_E_INVAL, "head_dim %u is not a multiple of 8 up to 512", d.head_dim);
  if (d.rotary_dim == 0) d.rotary_dim = d.head_dim;
  if (d.rotary_dim > d.head_dim || d.rotary_dim % 8)
    return fail(c, MR_E_INVAL, "rotary_dim %u is not a multiple of 8 up to head_dim %u", d.rotary_dim, d.head_dim);
  if (d.layout > MR_ROPE_INTERLEAVED) return fail(c, MR_E_INVAL, "rope layout %u unknown", d.layout);
  if (d.scaling > MR_ROPE_YARN_EXACT) return fail(c, MR_E_INVAL, "rope scaling %u unknown", d.scaling);
  if (!(d.base > 1.0) || !std::isfinite(d.base)) return fail(c, MR_E_INVAL, "rope base %g is not above 1", d.base);
  const bool yarn = d.scaling >= MR_ROPE_YARN;
  if (d.scaling != MR_ROPE_PLAIN && (!(d.factor >= 1.0) || !std::isfinite(d.factor)))
    return fail(c, MR_E_INVAL, "rope factor %g is not 1 or more", d.factor);
  if (yarn && d.orig_context == 0) return fail(c, MR_E_INVAL, "YaRN needs orig_context");
  if (d.beta_fast == 0.f) d.beta_fast = 32.f;
  if (d.beta_slow == 0.f) d.beta_slow = 1.f;
  if (yarn && (!(d.beta_slow > 0.f) || !(d.beta_fast >= d.beta_slow) || !std::isfinite(d.beta_fast)))
    return fail(c, MR_E_INVAL, "beta_fast %g and beta_slow %g are not in order", (double)d.beta_fast, (double)d.beta_slow);
  if (!std::isfinite(d.attn_factor) || d.attn_factor < 0.f)
    return fail(c, MR_E_INVAL, "attn_factor %g is negative or not finite", (double)d.attn_factor);
  if (c->device >= 0 && capturing(c)) return fail(c, MR_E_INVAL, "allocation during graph capture");
  mr_rope* r = new (std::nothrow) mr_rope;
  if (!r) return fail(c, MR_E_NOMEM, "host allocation failed");
  r->ctx = c, r->d = d;
  r->mul = d.attn_factor != 0.f ? d.attn_factor : yarn ? (float)(0.1 * std::log(d.factor) + 1.0) : 1.f;
  const int n = (int)d.rotary_dim / 2;
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  double low = 0, high = 1;
  if (yarn) {
    // the pair that turns `beta` times over the original context: base^(-2i/rotary) * orig = 2 pi beta
    auto pair = [&](double beta) { return d.rotary_dim * std::log(d.orig_context / (beta * kTwoPi)) / (2.0 * std::log(d.base)); };
    low = pair(d.beta_fast), high = pair(d.beta_slow);
    if (d.scaling == MR_ROPE_YARN) low = std::floor(low), high = std::ceil(high);
    low = std::max(low, 0.0), high = std::max(low, std::min(high, d.rotary_dim - 1.0));
    if (low == high) high += 0.001;
  }
  std::vector<double> turns;
  try {
    r->freq.resize(n), turns.resize(n);
  } catch (const std::bad_alloc&) {
    delete r;
    return fail(c, MR_E_NOMEM, "host allocation failed");
  }
  for (int i = 0; i < n; ++i) {
    double f = std::pow(d.base, -2.0 * i / d.rotary_dim);
    if (d.scaling == MR_ROPE_LINEAR) f /= d.factor;
    if (yarn) {
      const double ramp = std::min(1.0, std::max(0.0, (i - low) / (high - low)));
      f = f / d.factor * ramp + f * (1.0 - ramp);
    }
    r->freq[i] = f, turns[i] = f / kTwoPi;
  }
  if (c->device >= 0) {
    int rc = bind(c);
    hipError_t e = rc ? hipSuccess : hipMalloc(&r->d_turns, n * sizeof(double));
    if (!rc && e == hipSuccess) e = hipMemcpy(r->d_turns, turns.data(), n * sizeof(double), hipMemcpyHostToDevice);
    if (!rc && e != hipSuccess) rc = hip_fail(c, e, "rope frequencies");
    if (rc) {
      if (r->d_turns) (void)hipFree(r->d_turns);
      delete r;
      return rc;
    }
  }
  *out = r;
  return MR_OK;
}

void mr_rope_destroy(mr_rope* r) {
  if (!r) return;
  if (r->d_turns && bind(r->ctx) == MR_OK) {
    (void)hipStreamSynchronize(r->ctx->stream);
    (void)hipFree(r->d_turns);
  }
  delete r;
}

const double* mr_rope_frequencies(const mr_rope* r, uint32_t* n, float* attn_factor) {
  if (!r) return nullptr;
  if (n) *n = (uint32_t)r->freq.size();
  if (attn_factor) *attn_factor = r->mul;
  return r->freq.data();
}

int mr_qk_norm_rope(mr_ctx* c, const mr_rope* r, const mr_heads* q, const mr_heads* k, const float* q_norm,
                    const float* k_norm, float eps, const int32_t* positions, uint32_t T, const mr_heads* q_out,
                    const mr_heads* k_out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (!r) return fail(c, MR_E_INVAL, "rope is NULL");
  if (r->ctx != c) return fail(c, MR_E_INVAL, "rope belongs to another context");
  const uint32_t D = r->d.head_dim;
  mr::Heads in[2] = {}, o[2] = {};
  int rc;
  if ((rc = take(c, "q", q, D, &in[0])) || (rc = take(c, "q_out", q_out, D, &o[0]))) return rc;
  if (!k != !k_out) return fail(c, MR_E_INVAL, "only one of k and k_out is given");
  if (k && ((rc = take(c, "k", k, D, &in[1])) || (rc = take(c, "k_out", k_out, D, &o[1])))) return rc;
  if (o[0].n != in[0].n || o[1].n != in[1].n) return fail(c, MR_E_INVAL, "outputs have other head counts than inputs");
  if (k && (in[0].dtype != in[1].dtype || o[0].dtype != o[1].dtype))
    return fail(c, MR_E_INVAL, "q and k (q_out and k_out) must have one type");
  if (misaligned(q_norm, 16) || misaligned(k_norm, 16)) return fail(c, MR_E_INVAL, "norm weights must be 16-byte aligned");
  if (k_norm && !k) return fail(c, MR_E_INVAL, "k_norm without k");
  if ((rc = check_eps(c, eps))) return rc;
  if (!positions || misaligned(positions, 4)) return fail(c, MR_E_INVAL, "positions is NULL or not 4-byte aligned");
  if (T >= kMaxWork) return fail(c, MR_E_INVAL, "n_tokens %u is 2^24 or more", T);
  if (T == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_qk_norm_rope(c->launch(), *r, in[0], in[1], q_norm, k_norm, eps, positions, T, o[0], o[1]);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "qk_norm_rope launch");
}

uint64_t mr_kv_bytes(const mr_kv_desc* d) {
  if (check_kv_desc(nullptr, d)) return 0;
  return (uint64_t)d->n_pages * d->n_heads * (d->page_size / 64) * mr::kv_chunk_bytes(d->format, d->head_dim);
}

int mr_kv_create(mr_ctx* c, const mr_kv_desc* desc, mr_kv** out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (!out) return fail(c, MR_E_INVAL, "out pointer is NULL");
  *out = nullptr;
  int rc = check_kv_desc(c, desc);
  if (rc) return rc;
  if (c->device >= 0 && capturing(c)) return fail(c, MR_E_INVAL, "allocation during graph capture");
  mr_kv* kv = new (std::nothrow) mr_kv;
  if (!kv) return fail(c, MR_E_NOMEM, "host allocation failed");
  kv->ctx = c, kv->d = *desc, kv->bytes = mr_kv_bytes(desc);
  if (c->device >= 0) {
    rc = bind(c);
    if (!rc) {
      hipError_t e = hipSuccess;
      if (!c->attn_scratch)
        e = hipMalloc(&c->attn_scratch, std::max(mr::attn_decode_scratch_bytes(), mr::attn_extend_scratch_bytes()));
      if (e == hipSuccess) e = hipMalloc(&kv->base, kv->bytes);
      if (e == hipSuccess) e = mr::launch_zero(mr::Launch{c->stream, nullptr}, kv->base, kv->bytes);
      if (e == hipSuccess) e = hipStreamSynchronize(c->stream);  // the next call may be on another stream
      if (e != hipSuccess) rc = hip_fail(c, e, "cache pages");
    }
    if (rc) {
      if (kv->base) (void)hipFree(kv->base);
      delete kv;
      return rc;
    }
  }
  *out = kv;
  return MR_OK;
}

void mr_kv_destroy(mr_kv* kv) {
  if (!kv) return;
  if (kv->base && bind(kv->ctx) == MR_OK) {
    (void)hipStreamSynchronize(kv->ctx->stream);
    (void)hipFree(kv->base);
  }
  delete kv;
}

int mr_kv_write(mr_ctx* c, mr_kv* kv, const mr_heads* k, const mr_heads* v, uint32_t T, const int32_t* slots) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  int rc = check_kv(c, kv);
  if (rc) return rc;
  mr::Heads hk, hv;
  if ((rc = take(c, "k", k, kv->d.head_dim, &hk)) || (rc = take(c, "v", v, kv->d.head_dim, &hv))) return rc;
  if (hk.n != kv->d.n_heads || hv.n != kv->d.n_heads)
    return fail(c, MR_E_INVAL, "k has %u heads, v %u, the cache %u", hk.n, hv.n, kv->d.n_heads);
  if (!slots || misaligned(slots, 4)) return fail(c, MR_E_INVAL, "slots is NULL or not 4-byte aligned");
  if (T > kMaxTokens) return fail(c, MR_E_INVAL, "n_tokens %u is above 2^30 - 64", T);
  if (T == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_kv_write(c->launch(), pages(kv), kv->d.format, kv->d.head_dim, hk, hv, T, slots, c->attn_err);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "kv_write launch");
}

int mr_kv_read(mr_ctx* c, const mr_kv* kv, uint32_t T, const int32_t* slots, const mr_heads* k, const mr_heads* v) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  int rc = check_kv(c, kv);
  if (rc) return rc;
  if (!k && !v) return fail(c, MR_E_INVAL, "k and v are NULL");
  mr::Heads hk{}, hv{};
  if (k && (rc = take(c, "k", k, kv->d.head_dim, &hk))) return rc;
  if (v && (rc = take(c, "v", v, kv->d.head_dim, &hv))) return rc;
  if ((k && hk.n != kv->d.n_heads) || (v && hv.n != kv->d.n_heads))
    return fail(c, MR_E_INVAL, "k or v has another head count than the cache's %u", kv->d.n_heads);
  if (!slots || misaligned(slots, 4)) return fail(c, MR_E_INVAL, "slots is NULL or not 4-byte aligned");
  if (T > kMaxTokens) return fail(c, MR_E_INVAL, "n_tokens %u is above 2^30 - 64", T);
  if (T == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_kv_read(c->launch(), pages(kv), kv->d.format, kv->d.head_dim, T, slots, hk, hv, c->attn_err);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "kv_read launch");
}

int mr_attn_decode(mr_ctx* c, const mr_kv* kv, const mr_heads* q, uint32_t B, const int32_t* seq_len,
                   const int32_t* block_table, uint32_t max_pages, const mr_attn_opts* opts, const mr_heads* out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  int rc = check_kv(c, kv);
  if (rc) return rc;
  mr::Heads hq, ho;
  mr::AttnOpts o;
  const uint32_t D = kv->d.head_dim;
  if ((rc = take(c, "q", q, D, &hq)) || (rc = take(c, "out", out, D, &ho)) || (rc = check_qo(c, hq, ho, kv->d.n_heads)) ||
      (rc = take_opts(c, opts, D, &o)))
    return rc;
  if ((rc = check_lengths(c, kv, seq_len, block_table, max_pages, B))) return rc;
  if (B == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_attn_decode(c->launch(), pages(kv), kv->d.format, D, hq, B, seq_len, block_table,
                                              max_pages, o, ho, c->attn_err, c->attn_scratch, c->n_cu);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "attn_decode launch");
}

int mr_attn_prefill(mr_ctx* c, uint32_t D, const mr_heads* q, uint32_t nq, const mr_heads* k, const mr_heads* v,
                    uint32_t nk, uint32_t n_seqs, const int32_t* cu_q, const int32_t* cu_k, const mr_attn_opts* opts,
                    const mr_heads* out) {
  if (!c) return fail(nullptr, MR_E_INVAL, "context is NULL");
  if (D != 64 && D != 128 && D != 256) return fail(c, MR_E_UNSUPPORTED, "head_dim %u is not 64, 128 or 256", D);
  mr::Heads hq, hk, hv, ho;
  mr::AttnOpts o;
  int rc;
  if ((rc = take(c, "q", q, D, &hq)) || (rc = take(c, "k", k, D, &hk)) || (rc = take(c, "v", v, D, &hv)) ||
      (rc = take(c, "out", out, D, &ho)))
    return rc;
  if (hk.n != hv.n) return fail(c, MR_E_INVAL, "k has %u heads, v %u", hk.n, hv.n);
  if ((rc = check_qo(c, hq, ho, hk.n)) || (rc = take_opts(c, opts, D, &o))) return rc;
  if (hk.dtype != hq.dtype || hv.dtype != hq.dtype)
    return fail(c, MR_E_UNSUPPORTED, "k and v must have the type of q");
  if (hk.ts >= 1ull << 24 || hv.ts >= 1ull << 24)  // 64 rows within the 32-bit offsets of a buffer load
    return fail(c, MR_E_INVAL, "k or v has a token stride of 2^24 elements or more");
  if (!cu_q || !cu_k || misaligned(cu_q, 4) || misaligned(cu_k, 4))
    return fail(c, MR_E_INVAL, "cu_q or cu_k is NULL or not 4-byte aligned");
  if (nq > 0x7FFFFFFFu || nk > 0x7FFFFFFFu || n_seqs >= 0x7FFFFFFFu) return fail(c, MR_E_INVAL, "2^31 rows or more");
  if (((uint64_t)nq / mr::kPrefillRows + n_seqs + 1) * hq.n > kMaxWork - 8)  // the launch takes eights of them
    return fail(c, MR_E_INVAL, "%u rows of %u heads in %u sequences are more than 2^24 - 8 tiles", nq, hq.n, n_seqs);
  if (nq == 0 || n_seqs == 0) return MR_OK;
  if ((rc = bind(c))) return rc;
  const hipError_t e = mr::launch_attn_prefill(c->launch(), D, hq, nq, hk, hv, nk, n_seqs, cu_q, cu_k, o, ho, c->attn_err);
  return e == hipSuccess ? MR_OK : hip_fail(c, e, "attn_prefill launch");
}

}  // extern "C"
