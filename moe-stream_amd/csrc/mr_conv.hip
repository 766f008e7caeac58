// mr_conv.hip -- short causal convolutions of each channel over packed sequences.
//
// out_t = act(bias + sum_j w_j x_(t - taps + 1 + j)): each input is used `taps` times, so memory bounds it. A lane has 8
// adjacent channels of a run of rows of one sequence, the last inputs in registers; only a run's first rows read
// inputs of the run before again. A sequence's first run has no fewer than taps - 1 rows, or all of them: it alone
// reads the old state, and the same lane writes the new one after that, so that both may be one slot. Seven prompts, 8192 channels,
// f32 to bf16, 253 MB: 64 us, 4.0 TB/s; 48 sequences of one token: 6.5 us, launch and three loads in turn.
#include "mr_state_device.h"

namespace mr {

namespace {

constexpr int kV = 8;  // channels of a lane

struct ConvArgs {
  RowsOf x, out;
  const float *w, *bias;
  int silu;
  Sequences s;
};

struct Channels {
  float v[kV];
};

template <int SRC>
__device__ __forceinline__ Channels load8(const void* p, uint64_t i) {
  const f32x4 a = load4(p, SRC, i), b = load4(p, SRC, i + 4);
  return Channels{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ void store8(void* p, uint32_t dtype, uint64_t i, const Channels& c) {
  store4(p, dtype, i, f32x4{c.v[0], c.v[1], c.v[2], c.v[3]});
  store4(p, dtype, i + 4, f32x4{c.v[4], c.v[5], c.v[6], c.v[7]});
}

template <int SRC, int TAPS, int BITS>
__global__ __launch_bounds__(256) void k_causal_conv(ConvArgs a) {
  constexpr int R = 1 << BITS, P = TAPS - 1;
  static_assert(R >= P, "a sequence's first run has all that the old state reaches");
  const Sequences& q = a.s;
  if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(q.cu, q.n_seqs, q.n_rows, q.err, kErrPacked);
  const uint32_t s = find_seq(q.cu, q.n_seqs, q.n_rows, 1, BITS, blockIdx.x);
  int q0, q1;
  rows_of(q.cu, q.n_rows, s, q0, q1);
  const int64_t tile = (int64_t)blockIdx.x - first_tile(q.cu, q.n_rows, s, 1, BITS);
  const int n = q1 - q0, at = (int)(tile << BITS);  // the sequence's rows, the run's first one of them
  if (tile < 0 || (tile > 0 && at >= n)) return;
  const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * kV;
  if (c >= a.x.width) return;

  // the inputs before the run's first one, the oldest first
  Channels before[P] = {};
  const int source = at < P ? slot_of(q, q.source, s) : -1;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (at - P + j >= 0)
      before[j] = load8<SRC>(a.x.p, (uint64_t)(q0 + at - P + j) * a.x.stride + c);
    else if (source >= 0)
      before[j] = load8<MR_F32>(q.states, ((uint64_t)source * P + at + j) * a.x.width + c);
  }
  if (at == 0) {
    const int target = slot_of(q, q.target, s);
    if (target >= 0) {
      Channels last[P];
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (n - P + j >= 0) {
          last[j] = load8<SRC>(a.x.p, (uint64_t)(q0 + n - P + j) * a.x.stride + c);
        } else {
          last[j] = before[j];
#pragma unroll
          for (int i = j + 1; i < P; ++i)
            if (i == n + j) last[j] = before[i];
        }
      }
#pragma unroll
      for (int j = 0; j < P; ++j) store8(q.states, MR_F32, ((uint64_t)target * P + j) * a.x.width + c, last[j]);
    }
  }
  if (at >= n) return;
  Channels w[TAPS], bias = {};
#pragma unroll
  for (int i = 0; i < kV * TAPS; i += 4) {
    const f32x4 x = load4(a.w, MR_F32, (uint64_t)c * TAPS + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[(i + j) % TAPS].v[(i + j) / TAPS] = x[j];
  }
  if (a.bias) bias = load8<MR_F32>(a.bias, c);

  const int rows = min(R, n - at);
  constexpr int B = 4;  // rows on their way at once
  for (int r0 = 0; r0 < rows; r0 += B) {
    Channels x[B];
#pragma unroll
    for (int r = 0; r < B; ++r)
      if (r0 + r < rows) x[r] = load8<SRC>(a.x.p, (uint64_t)(q0 + at + r0 + r) * a.x.stride + c);
#pragma unroll
    for (int r = 0; r < B; ++r) {
      if (r0 + r >= rows) break;
      Channels y = bias;
#pragma unroll
      for (int v = 0; v < kV; ++v) {
#pragma unroll
        for (int j = 0; j < P; ++j) y.v[v] = fmaf(w[j].v[v], before[j].v[v], y.v[v]);
        y.v[v] = fmaf(w[P].v[v], x[r].v[v], y.v[v]);
        if (a.silu) y.v[v] = y.v[v] / (1.f + __expf(-y.v[v]));
      }
      store8(a.out.p, a.out.dtype, (uint64_t)(q0 + at + r0 + r) * a.out.stride + c, y);
#pragma unroll
      for (int j = 0; j + 1 < P; ++j) before[j] = before[j + 1];
      before[P - 1] = x[r];
    }
  }
}

template <int SRC, int TAPS>
void launch(const Launch& K, const ConvArgs& a) {
  const Sequences& s = a.s;
  const uint32_t across = (a.x.width + 256 * kV - 1) / (256 * kV);
  // Runs of 4 rows where sequences are short, so that their first rows' loads do not wait for each other's.
  if ((uint64_t)s.n_rows < 8ull * s.n_seqs)
    hipLaunchKernelGGL((k_causal_conv<SRC, TAPS, 2>), dim3((s.n_rows >> 2) + s.n_seqs, across), dim3(256), 0, K.s, a);
  else
    hipLaunchKernelGGL((k_causal_conv<SRC, TAPS, 4>), dim3((s.n_rows >> 4) + s.n_seqs, across), dim3(256), 0, K.s, a);
}
template <int SRC>
void launch(const Launch& K, uint32_t taps, const ConvArgs& a) {
  if (taps == 2) launch<SRC, 2>(K, a);
  if (taps == 3) launch<SRC, 3>(K, a);
  if (taps == 4) launch<SRC, 4>(K, a);
}

}  // namespace

hipError_t launch_causal_conv(const Launch& K, const RowsOf& x, const float* w, uint32_t taps, const float* bias, bool silu,
                              const Sequences& s, const RowsOf& out) {
  ProfScope ps(K, "causal_conv");
  const ConvArgs a{x, out, w, bias, silu, s};
  if (x.dtype == MR_F32) launch<MR_F32>(K, taps, a);
  if (x.dtype == MR_F16) launch<MR_F16>(K, taps, a);
  if (x.dtype == MR_BF16) launch<MR_BF16>(K, taps, a);
  return hipGetLastError();
}

}  // namespace mr
