// mr_rope.hip -- RMSNorm of query and key heads and their rotary positions in one pass.
//
// x = in * (1 / sqrt(mean(in^2) + eps)) * w per head (where w is given), then the pairs (a, b) of x turn
// by t = position * f: (a cos t - b sin t, b cos t + a sin t), both times the attention factor.
#include "mr_attn_device.h"

namespace mr {

namespace {

struct RopeArgs {
  Heads in[2], out[2];  // queries, keys
  const float* w[2];
  const double* turns;  // [rotary / 2] turns per position
  const int32_t* pos;
  float eps, mul;
  int D, rotary, interleaved, rows;  // rows: heads of one token, queries first
};

// One token and blockIdx.y's share of its heads to a workgroup; L lanes (a power of two) to a head, each
// with 8 of its elements as two quads: in the half layout elements 4u.. and rotary/2 + 4u.., so that a
// lane holds both members of its pairs; adjacent quads in the interleaved layout and behind the rotated
// part. The angle is reduced to a fraction of a turn in 64 bits (f32 would lose 2^-24 of a far position's
// angle), the sine and cosine of that fraction are taken in f32, once per token and pair, while the first R
// heads of each lane group are on their way from memory. Memory bounds it: 4096 tokens of 36 heads of 128, f32 to
// bf16 with norms, 28.6 us, 113 MB at 4.0 TB/s (a large copy: 4.9); one token of 72 heads of 64: 2.9 us.
template <int R>
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs a, int L) {
  __shared__ __attribute__((aligned(16))) float cs[256], sn[256];
  const int t = blockIdx.x, half = a.rotary / 2, per = 256 / L;
  const int u = threadIdx.x & (L - 1);
  const bool turn = u < a.rotary / 8, apart = turn && !a.interleaved;
  const int e0 = apart ? 4 * u : 8 * u, e1 = apart ? half + 4 * u : 8 * u + 4;
  const int row0 = blockIdx.y * per * R + threadIdx.x / L;
  auto live = [&](int i) { return row0 + i * per < a.rows && u < a.D / 8; };
  f32x4 x[R], y[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i * per, q = row < (int)a.in[0].n;
    if (!live(i)) continue;
    const uint64_t o = q ? (uint64_t)t * a.in[0].ts + (uint64_t)row * a.in[0].hs
                         : (uint64_t)t * a.in[1].ts + (uint64_t)(row - (int)a.in[0].n) * a.in[1].hs;
    const void* p = q ? a.in[0].p : a.in[1].p;
    x[i] = load4(p, a.in[0].dtype, o + e0);
    y[i] = load4(p, a.in[0].dtype, o + e1);
  }
  if ((int)threadIdx.x < half) {
    const double z = (double)a.pos[t] * a.turns[threadIdx.x];
    float s, c;
    sincospif(2.f * (float)(z - rint(z)), &s, &c);
    cs[threadIdx.x] = c * a.mul, sn[threadIdx.x] = s * a.mul;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i * per, q = row < (int)a.in[0].n;
    const float* w = q ? a.w[0] : a.w[1];
    f32x4 v = x[i], z = y[i];
    float s = v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w + z.x * z.x + z.y * z.y + z.z * z.z + z.w * z.w;
    if (a.w[0] || a.w[1]) {
      if (!live(i)) s = 0.f;
      for (int o = L / 2; o >= 1; o >>= 1) s += __shfl_xor(s, o, kWave);
    }
    if (!live(i)) continue;
    if (w) {
      const float inv = 1.f / sqrtf(s / (float)a.D + a.eps);
      v = v * inv * *reinterpret_cast<const f32x4*>(w + e0);
      z = z * inv * *reinterpret_cast<const f32x4*>(w + e1);
    }
    if (turn) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(cs + 4 * u), n = *reinterpret_cast<const f32x4*>(sn + 4 * u);
      if (apart) {
        const f32x4 b = v * c - z * n;
        z = z * c + v * n, v = b;
      } else {
        v = f32x4{v.x * c.x - v.y * n.x, v.y * c.x + v.x * n.x, v.z * c.y - v.w * n.y, v.w * c.y + v.z * n.y};
        z = f32x4{z.x * c.z - z.y * n.z, z.y * c.z + z.x * n.z, z.z * c.w - z.w * n.w, z.w * c.w + z.z * n.w};
      }
    }
    const uint64_t o = q ? (uint64_t)t * a.out[0].ts + (uint64_t)row * a.out[0].hs
                         : (uint64_t)t * a.out[1].ts + (uint64_t)(row - (int)a.in[0].n) * a.out[1].hs;
    void* p = q ? a.out[0].p : a.out[1].p;
    store4(p, a.out[0].dtype, o + e0, v);
    store4(p, a.out[0].dtype, o + e1, z);
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(const Launch& K, const mr_rope& r, const Heads& q, const Heads& k, const float* qn,
                               const float* kn, float eps, const int32_t* pos, uint32_t T, const Heads& qo,
                               const Heads& ko) {
  ProfScope ps(K, "qk_norm_rope");
  RopeArgs a{{q, k}, {qo, ko}, {qn, kn}, r.d_turns, pos, eps, r.mul, (int)r.d.head_dim, (int)r.d.rotary_dim,
             r.d.layout == MR_ROPE_INTERLEAVED, (int)(q.n + k.n)};
  int L = 1;
  while (L < a.D / 8) L *= 2;
  // Up to four heads to a lane group, so that one workgroup's sines serve more of them, as long as that leaves
  // each CU eight workgroups.
  const int per = 256 / L, need = (a.rows + per - 1) / per;
  const int R = (int)std::max<uint64_t>(1, std::min<uint64_t>(std::min(4, need), (uint64_t)T * need / 2048));
  const dim3 g(T, (need + R - 1) / R);
  if (R == 1) hipLaunchKernelGGL(k_qk_norm_rope<1>, g, dim3(256), 0, K.s, a, L);
  if (R == 2) hipLaunchKernelGGL(k_qk_norm_rope<2>, g, dim3(256), 0, K.s, a, L);
  if (R == 3) hipLaunchKernelGGL(k_qk_norm_rope<3>, g, dim3(256), 0, K.s, a, L);
  if (R == 4) hipLaunchKernelGGL(k_qk_norm_rope<4>, g, dim3(256), 0, K.s, a, L);
  return hipGetLastError();
}

}  // namespace mr
