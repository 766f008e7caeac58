// mr_attn_prefill.hip -- causal attention over packed prompts.
#include "mr_attn_device.h"

namespace mr {

namespace {

// One wave for a query row and head. blockIdx.x counts the rows; the row's sequence is found in cu_q.
template <int D>
__global__ __launch_bounds__(64) void k_attn_prefill(Heads q, Heads k, Heads v, Heads out, int nq, int nk, int n_seqs,
                                                     const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k,
                                                     AttnOpts o, uint32_t* err) {
  __shared__ float qs[D], ps[64];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hk = h / (q.n / k.n);
  auto clamp = [](int x, int hi) { return min(max(x, 0), hi); };
  int seq = -1;
  for (int s = 0; s < n_seqs && seq < 0; ++s) {
    if (cu_q[s] != clamp(cu_q[s], nq) || cu_q[s + 1] != clamp(cu_q[s + 1], nq) || cu_q[s + 1] < cu_q[s] ||
        cu_k[s] != clamp(cu_k[s], nk) || cu_k[s + 1] != clamp(cu_k[s + 1], nk) || cu_k[s + 1] < cu_k[s])
      if (lane == 0) atomicOr(err, kErrOffset);
    if (row >= clamp(cu_q[s], nq) && row < clamp(cu_q[s + 1], nq)) seq = s;
  }
  if (seq < 0) return;
  const int q1 = clamp(cu_q[seq + 1], nq), k0 = clamp(cu_k[seq], nk), k1 = clamp(cu_k[seq + 1], nk);
  for (int d = lane * 4; d < D; d += 256) {
    const f32x4 x = load4(q.p, q.dtype, (uint64_t)row * q.ts + (uint64_t)h * q.hs + d);
    qs[d] = x.x, qs[d + 1] = x.y, qs[d + 2] = x.z, qs[d + 3] = x.w;
  }
  __syncthreads();
  float m = o.sinks ? o.sinks[h] : -INFINITY, l = o.sinks ? 1.f : 0.f, acc[D / 64] = {};
  const int64_t last = (int64_t)k1 - (q1 - row), first = max((int64_t)k0, o.window ? last + 1 - (int64_t)o.window : 0);
  for (int64_t j0 = first; j0 <= last; j0 += 64) {
    const int64_t key = j0 + lane;
    float s = -INFINITY;
    if (key <= last) {
      s = 0.f;
      for (int d = 0; d < D; d += 4) {
        const f32x4 x = load4(k.p, k.dtype, (uint64_t)key * k.ts + (uint64_t)hk * k.hs + d);
        s += x.x * qs[d] + x.y * qs[d + 1] + x.z * qs[d + 2] + x.w * qs[d + 3];
      }
      s *= o.scale;
    }
    const float top = fmaxf(m, wave_max(s));
    const float p = s == -INFINITY ? 0.f : expf(s - top), f = m == -INFINITY ? 0.f : expf(m - top);
    l = l * f + wave_sum(p), m = top;
    ps[lane] = p;
    __syncthreads();
    for (int i = 0; i < D / 64; ++i) {
      acc[i] *= f;
      for (int j = 0; j < 64 && j0 + j <= last; ++j) {
        const uint16_t w = static_cast<const uint16_t*>(v.p)[(uint64_t)(j0 + j) * v.ts + (uint64_t)hk * v.hs + lane + 64 * i];
        acc[i] += ps[j] * (v.dtype == MR_F16 ? h2f(w) : bits_f32((uint32_t)w << 16));
      }
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(out.p) + (uint64_t)row * out.ts + (uint64_t)h * out.hs;
  for (int i = 0; i < D / 64; ++i) {
    const float x = acc[i] * inv;
    dst[lane + 64 * i] = (uint16_t)(out.dtype == MR_F16 ? pack_f16(x, 0.f) : pack_bf16(x, 0.f));
  }
}

}  // namespace

hipError_t launch_attn_prefill(const Launch& K, uint32_t D, const Heads& q, uint32_t nq, const Heads& k, const Heads& v,
                               uint32_t nk, uint32_t n_seqs, const int32_t* cu_q, const int32_t* cu_k, const AttnOpts& o,
                               const Heads& out, uint32_t* err) {
  ProfScope ps(K, "attn_prefill");
  const dim3 g(nq, q.n);
  if (D == 64) hipLaunchKernelGGL((k_attn_prefill<64>), g, dim3(64), 0, K.s, q, k, v, out, (int)nq, (int)nk, (int)n_seqs, cu_q, cu_k, o, err);
  if (D == 128) hipLaunchKernelGGL((k_attn_prefill<128>), g, dim3(64), 0, K.s, q, k, v, out, (int)nq, (int)nk, (int)n_seqs, cu_q, cu_k, o, err);
  if (D == 256) hipLaunchKernelGGL((k_attn_prefill<256>), g, dim3(64), 0, K.s, q, k, v, out, (int)nq, (int)nk, (int)n_seqs, cu_q, cu_k, o, err);
  return hipGetLastError();
}

}  // namespace mr
