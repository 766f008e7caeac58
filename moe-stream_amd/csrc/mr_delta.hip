// mr_delta.hip -- the gated delta rule over packed sequences.
//
//   S' = exp(g) S,  S = S' + beta k (v - S'^T k)^T,  out = scale S^T q
//
// One token at a time, a workgroup for each sequence and head, its state in registers.
#include "mr_state_device.h"

namespace mr {

namespace {

struct DeltaArgs {
  DeltaShape d;
  Heads q, k, v, out;
  const float *decay, *beta;
  Sequences s;
};

// Log decay and beta of token t for head h.
__device__ __forceinline__ void gates(const DeltaArgs& a, uint64_t t, uint32_t h, float& g, float& beta) {
  g = a.decay[t * a.d.gate_stride + h], beta = a.beta[t * a.d.gate_stride + h];
  if (!a.d.a_log) return;
  const float x = g + a.d.dt_bias[h];
  g = -expf(a.d.a_log[h]) * (fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))));
  beta = 1.f / (1.f + expf(-beta));
}

// A state's rows lie across the lanes, four columns each; a thread has every G-th row. S'^T k and S'^T q are taken
// together, as out = scale (S'^T q + (k . q) correction): one exchange between the lanes for each token.
template <int DK, int DV, bool BF>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a) {
  constexpr int L = DV / 4, G = 256 / L, N = DK / G, E = DK / 64;
  constexpr int kT = 8;  // tokens staged at once
  constexpr uint32_t kType = BF ? MR_BF16 : MR_F16;
  __shared__ __attribute__((aligned(16))) float key[kT][DK], query[kT][DK], red[2][4][2][DV];
  __shared__ float fade[kT], gain[kT], both[kT];
  const Sequences& sq = a.s;
  const uint32_t h = blockIdx.x, s = blockIdx.y, hk = h / (a.d.value_heads / a.d.key_heads);
  if (h == 0 && s == 0) check_offsets(sq.cu, sq.n_seqs, sq.n_rows, sq.err, kErrPacked);
  int q0, q1;
  rows_of(sq.cu, sq.n_rows, s, q0, q1);
  const int n = q1 - q0;
  const int source = slot_of(sq, sq.source, s), target = slot_of(sq, sq.target, s);
  if (n == 0 && (target < 0 || target == source)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = tid / L, col = 4 * (tid % L);

  f32x4 S[N] = {};
  if (source >= 0) {
    const float* p = sq.states + ((uint64_t)source * a.d.value_heads + h) * (DK * DV) + col;
#pragma unroll
    for (int i = 0; i < N; ++i) S[i] = *reinterpret_cast<const f32x4*>(p + (g + G * i) * DV);
  }
  for (int t0 = 0; t0 < n; t0 += kT) {
    const int m = min(kT, n - t0);
    __syncthreads();
    for (int t = wave; t < m; t += 4) {
      const uint64_t row = (uint64_t)(q0 + t0 + t);
      float x[E], y[E], xx = 0.f, yy = 0.f, xy = 0.f;
      const uint16_t* qp = static_cast<const uint16_t*>(a.q.p) + row * a.q.ts + (uint64_t)hk * a.q.hs + E * lane;
      const uint16_t* kp = static_cast<const uint16_t*>(a.k.p) + row * a.k.ts + (uint64_t)hk * a.k.hs + E * lane;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = BF ? bits_f32((uint32_t)qp[e] << 16) : h2f(qp[e]);
        y[e] = BF ? bits_f32((uint32_t)kp[e] << 16) : h2f(kp[e]);
        xx = fmaf(x[e], x[e], xx), yy = fmaf(y[e], y[e], yy), xy = fmaf(x[e], y[e], xy);
      }
      float fx = a.d.scale, fy = 1.f;
      if (a.d.unit_eps > 0.f) {
        fx /= sqrtf(wave_sum_fast(xx) + a.d.unit_eps);
        fy /= sqrtf(wave_sum_fast(yy) + a.d.unit_eps);
      }
      xy = wave_sum_fast(xy);
#pragma unroll
      for (int e = 0; e < E; ++e) query[t][E * lane + e] = x[e] * fx, key[t][E * lane + e] = y[e] * fy;
      if (lane == 0) {
        float lg, b;
        gates(a, row, h, lg, b);
        fade[t] = expf(lg), gain[t] = b, both[t] = xy * fx * fy;
      }
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const uint64_t row = (uint64_t)(q0 + t0 + t);
      const f32x4 v = load4(a.v.p, kType, row * a.v.ts + (uint64_t)h * a.v.hs + col);
      f32x4 sk = {}, sq4 = {};
#pragma unroll
      for (int i = 0; i < N; ++i) sk += S[i] * key[t][g + G * i], sq4 += S[i] * query[t][g + G * i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sk[j] = add_xor32(sk[j]), sq4[j] = add_xor32(sq4[j]);
        if (L == 16) sk[j] = add_xor16(sk[j]), sq4[j] = add_xor16(sq4[j]);
      }
      float(&r)[4][2][DV] = red[t & 1];
      if (lane < L) *reinterpret_cast<f32x4*>(&r[wave][0][col]) = sk, *reinterpret_cast<f32x4*>(&r[wave][1][col]) = sq4;
      __syncthreads();
      sk = f32x4{}, sq4 = f32x4{};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sk += *reinterpret_cast<const f32x4*>(&r[w][0][col]), sq4 += *reinterpret_cast<const f32x4*>(&r[w][1][col]);
      const float f = fade[t];
      const f32x4 d = (v - sk * f) * gain[t];
      if (tid < L) store4(a.out.p, kType, row * a.out.ts + (uint64_t)h * a.out.hs + col, sq4 * f + d * both[t]);
#pragma unroll
      for (int i = 0; i < N; ++i) S[i] = S[i] * f + d * key[t][g + G * i];
    }
  }
  if (target >= 0) {
    float* p = sq.states + ((uint64_t)target * a.d.value_heads + h) * (DK * DV) + col;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<f32x4*>(p + (g + G * i) * DV) = S[i];
  }
}

template <int DK, int DV>
void launch(const Launch& K, bool bf, const DeltaArgs& a) {
  const dim3 g(a.d.value_heads, a.s.n_seqs), b(256);
  hipLaunchKernelGGL((bf ? k_delta_step<DK, DV, true> : k_delta_step<DK, DV, false>), g, b, 0, K.s, a);
}

}  // namespace

uint64_t delta_scratch_bytes() { return 256; }

hipError_t launch_delta_rule(const Launch& K, const DeltaShape& d, const Heads& q, const Heads& k, const Heads& v,
                             const float* decay, const float* beta, const Sequences& s, const Heads& out, void* scratch) {
  (void)scratch;
  const DeltaArgs a{d, q, k, v, out, decay, beta, s};
  const bool bf = q.dtype == MR_BF16;
  ProfScope ps(K, "delta_step");
  if (d.key_dim == 64 && d.value_dim == 64) launch<64, 64>(K, bf, a);
  if (d.key_dim == 64 && d.value_dim == 128) launch<64, 128>(K, bf, a);
  if (d.key_dim == 128 && d.value_dim == 64) launch<128, 64>(K, bf, a);
  if (d.key_dim == 128 && d.value_dim == 128) launch<128, 128>(K, bf, a);
  return hipGetLastError();
}

}  // namespace mr
