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
// angle), the sine and cosine of that fraction are taken in f32, once per token and pair.
__global__ __launch_bounds__(256) void k_qk_norm_rope(RopeArgs a, int L, int rows_per_wg) {
  __shared__ float cs[256], sn[256];
  const int t = blockIdx.x, half = a.rotary / 2;
  if ((int)threadIdx.x < half) {
    const double x = (double)a.pos[t] * a.turns[threadIdx.x];
    float s, c;
    sincospif(2.f * (float)(x - rint(x)), &s, &c);
    cs[threadIdx.x] = c * a.mul, sn[threadIdx.x] = s * a.mul;
  }
  __syncthreads();
  const int u = threadIdx.x & (L - 1), U = a.D / 8;
  const int row0 = blockIdx.y * rows_per_wg, row1 = min(a.rows, row0 + rows_per_wg);
  const bool turn = u < a.rotary / 8, apart = turn && !a.interleaved;
  const int e0 = apart ? 4 * u : 8 * u, e1 = apart ? half + 4 * u : 8 * u + 4;
  for (int base = row0; base < row1; base += 256 / L) {
    const int row = base + threadIdx.x / L;
    const bool live = row < row1 && u < U;
    const int side = row >= (int)a.in[0].n, h = side ? row - a.in[0].n : row;
    f32x4 x = {0, 0, 0, 0}, y = x;
    if (live) {
      const uint64_t o = (uint64_t)t * a.in[side].ts + (uint64_t)h * a.in[side].hs;
      x = load4(a.in[side].p, a.in[side].dtype, o + e0);
      y = load4(a.in[side].p, a.in[side].dtype, o + e1);
    }
    const float* w = a.w[side];
    float s = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
    for (int o = L / 2; o >= 1; o >>= 1) s += __shfl_xor(s, o, kWave);
    if (!live) continue;
    if (w) {
      const float inv = 1.f / sqrtf(s / (float)a.D + a.eps);
      const f32x4 wx = *reinterpret_cast<const f32x4*>(w + e0), wy = *reinterpret_cast<const f32x4*>(w + e1);
      x = x * inv * wx, y = y * inv * wy;
    }
    if (apart) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(cs + 4 * u), n = *reinterpret_cast<const f32x4*>(sn + 4 * u);
      const f32x4 p = x * c - y * n, q = y * c + x * n;
      x = p, y = q;
    } else if (turn) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(cs + 4 * u), n = *reinterpret_cast<const f32x4*>(sn + 4 * u);
      x = f32x4{x.x * c.x - x.y * n.x, x.y * c.x + x.x * n.x, x.z * c.y - x.w * n.y, x.w * c.y + x.z * n.y};
      y = f32x4{y.x * c.z - y.y * n.z, y.y * c.z + y.x * n.z, y.z * c.w - y.w * n.w, y.w * c.w + y.z * n.w};
    }
    const uint64_t o = (uint64_t)t * a.out[side].ts + (uint64_t)h * a.out[side].hs;
    store4(a.out[side].p, a.out[side].dtype, o + e0, x);
    store4(a.out[side].p, a.out[side].dtype, o + e1, y);
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
  const int per = 256 / L;
  hipLaunchKernelGGL(k_qk_norm_rope, dim3(T, (a.rows + per - 1) / per), dim3(256), 0, K.s, a, L, per);
  return hipGetLastError();
}

}  // namespace mr
