// mr_attn_decode.hip -- attention of one query token per sequence over the paged cache.
#include "mr_attn_device.h"

namespace mr {

namespace {

// One wave for a sequence and query head: a lane takes a key of each 64 and, for the sum, D/64
// elements of the values.
template <int FMT, int D>
__global__ __launch_bounds__(64) void k_attn_decode(KvPages kv, Heads q, Heads out, const int32_t* __restrict__ len,
                                                    const int32_t* __restrict__ table, uint32_t max_pages, AttnOpts o,
                                                    uint32_t* err) {
  __shared__ float qs[D], ps[64];
  const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hk = h / (q.n / kv.n_heads);
  const int64_t cap = (int64_t)max_pages << kv.page_shift;
  const int64_t raw = len[b], n = raw < 0 ? 0 : raw > cap ? cap : raw;
  if (raw != n && lane == 0) atomicOr(err, kErrLength);
  for (int d = lane * 4; d < D; d += 256) {
    const f32x4 v = load4(q.p, q.dtype, (uint64_t)b * q.ts + (uint64_t)h * q.hs + d);
    qs[d] = v.x, qs[d + 1] = v.y, qs[d + 2] = v.z, qs[d + 3] = v.w;
  }
  __syncthreads();
  float m = o.sinks ? o.sinks[h] : -INFINITY, l = o.sinks ? 1.f : 0.f, acc[D / 64] = {};
  const int64_t first = o.window && n > o.window ? n - o.window : 0;
  for (int64_t k0 = first & ~63ll; k0 < n; k0 += 64) {
    const int32_t page = table[(uint64_t)b * max_pages + (k0 >> kv.page_shift)];
    const bool there = page >= 0 && (uint32_t)page < kv.n_pages;
    if (!there) {
      if (lane == 0) atomicOr(err, kErrPage);
      continue;
    }
    const uint8_t* chunk = kv.at(page, hk, (uint32_t)((k0 & ((1ll << kv.page_shift) - 1)) >> 6));
    const int64_t key = k0 + lane;
    float s = -INFINITY;
    if (key >= first && key < n) {
      s = 0.f;
      for (int d = 0; d < D; ++d) s += qs[d] * kv_value<FMT, D>(chunk, true, lane, d);
      s *= o.scale;
    }
    const float top = fmaxf(m, wave_max(s));
    const float p = s == -INFINITY ? 0.f : expf(s - top), f = m == -INFINITY ? 0.f : expf(m - top);
    l = l * f + wave_sum(p), m = top;
    ps[lane] = p;
    __syncthreads();
    for (int i = 0; i < D / 64; ++i) {
      acc[i] *= f;
      for (int j = 0; j < 64; ++j) acc[i] += ps[j] * kv_value<FMT, D>(chunk, false, j, lane + 64 * i);
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(out.p) + (uint64_t)b * out.ts + (uint64_t)h * out.hs;
  for (int i = 0; i < D / 64; ++i) {
    const float v = acc[i] * inv;
    dst[lane + 64 * i] = (uint16_t)(out.dtype == MR_F16 ? pack_f16(v, 0.f) : pack_bf16(v, 0.f));
  }
}

template <int FMT>
hipError_t decode_fmt(const Launch& K, const KvPages& kv, uint32_t D, const Heads& q, uint32_t B, const int32_t* len,
                      const int32_t* table, uint32_t max_pages, const AttnOpts& o, const Heads& out, uint32_t* err) {
  const dim3 g(B, q.n);
  if (D == 64) hipLaunchKernelGGL((k_attn_decode<FMT, 64>), g, dim3(64), 0, K.s, kv, q, out, len, table, max_pages, o, err);
  if (D == 128) hipLaunchKernelGGL((k_attn_decode<FMT, 128>), g, dim3(64), 0, K.s, kv, q, out, len, table, max_pages, o, err);
  if (D == 256) hipLaunchKernelGGL((k_attn_decode<FMT, 256>), g, dim3(64), 0, K.s, kv, q, out, len, table, max_pages, o, err);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_decode(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& q, uint32_t B,
                              const int32_t* len, const int32_t* table, uint32_t max_pages, const AttnOpts& o,
                              const Heads& out, uint32_t* err) {
  ProfScope ps(K, "attn_decode");
  if (format == MR_KV_F16) return decode_fmt<MR_KV_F16>(K, kv, D, q, B, len, table, max_pages, o, out, err);
  if (format == MR_KV_MXINT8) return decode_fmt<MR_KV_MXINT8>(K, kv, D, q, B, len, table, max_pages, o, out, err);
  return decode_fmt<MR_KV_MXFP4>(K, kv, D, q, B, len, table, max_pages, o, out, err);
}

}  // namespace mr
