// mr_delta.hip -- the gated delta rule over packed sequences.
//
//   S' = exp(g) S,  S = S' + beta k (v - S'^T k)^T,  out = scale S^T q
//
// One token at a time (k_delta_step) for short sequences, a workgroup for each sequence and head, its state in registers; in chunks
// of 64 tokens (k_delta_prepare, k_delta_chunks) for long ones.
#include <type_traits>

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

// A state's rows lie across the lanes, four columns each; a thread has N adjacent rows. S'^T k and S'^T q are taken
// together, as out = scale (S'^T q + (k . q) correction): one exchange between the lanes for each token. For one token the states'
// bytes bound it (48 sequences, 32 heads of 128 by 128, 202 MB: 48 us, 4.2 TB/s; one sequence 6.2 us, launch and loads in turn),
// for a few the products and exchanges of each token in turn (16 sequences of 5 tokens, 69 MB: 22 us).
template <int DK, int DV, bool BF>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a, int most) {
  constexpr int L = DV / 4, G = 256 / L, N = DK / G, E = DK / 64, F = DV / 64;
  constexpr int kT = 8;  // tokens staged at once
  constexpr uint32_t kType = BF ? MR_BF16 : MR_F16;
  __shared__ __attribute__((aligned(16))) float key[kT][DK], query[kT][DK], value[kT][DV], red[2][4][2][DV];
  __shared__ float fade[kT], gain[kT], both[kT];
  const Sequences& sq = a.s;
  const uint32_t h = blockIdx.x, s = blockIdx.y, hk = h / (a.d.value_heads / a.d.key_heads);
  if (h == 0 && s == 0) check_offsets(sq.cu, sq.n_seqs, sq.n_rows, sq.err, kErrPacked);
  int q0, q1;
  rows_of(sq.cu, sq.n_rows, s, q0, q1);
  const int n = q1 - q0;
  const int source = slot_of(sq, sq.source, s), target = slot_of(sq, sq.target, s);
  if (n > most || (n == 0 && (target < 0 || target == source))) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = tid / L, col = 4 * (tid % L);

  f32x4 S[N] = {};
  if (source >= 0) {
    const float* p = sq.states + ((uint64_t)source * a.d.value_heads + h) * (DK * DV) + col;
#pragma unroll
    for (int i = 0; i < N; ++i) S[i] = *reinterpret_cast<const f32x4*>(p + (N * g + i) * DV);
  }
  for (int t0 = 0; t0 < n; t0 += kT) {
    const int m = min(kT, n - t0);
    __syncthreads();
    // Tokens wave and wave + 4: all their loads first.
    float x[2][E], y[2][E], v[2][F], lg[2], b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t row = (uint64_t)(q0 + t0 + min(wave + 4 * j, m - 1));
      const uint16_t* qp = static_cast<const uint16_t*>(a.q.p) + row * a.q.ts + (uint64_t)hk * a.q.hs + E * lane;
      const uint16_t* kp = static_cast<const uint16_t*>(a.k.p) + row * a.k.ts + (uint64_t)hk * a.k.hs + E * lane;
      const uint16_t* vp = static_cast<const uint16_t*>(a.v.p) + row * a.v.ts + (uint64_t)h * a.v.hs + F * lane;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[j][e] = BF ? bits_f32((uint32_t)qp[e] << 16) : h2f(qp[e]);
        y[j][e] = BF ? bits_f32((uint32_t)kp[e] << 16) : h2f(kp[e]);
      }
#pragma unroll
      for (int e = 0; e < F; ++e) v[j][e] = BF ? bits_f32((uint32_t)vp[e] << 16) : h2f(vp[e]);
      gates(a, row, h, lg[j], b[j]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = wave + 4 * j;
      if (t >= m) break;
      float xx = 0.f, yy = 0.f, xy = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) xx = fmaf(x[j][e], x[j][e], xx), yy = fmaf(y[j][e], y[j][e], yy), xy = fmaf(x[j][e], y[j][e], xy);
      float fx = a.d.scale, fy = 1.f;
      if (a.d.unit_eps > 0.f) {
        fx /= sqrtf(wave_sum_fast(xx) + a.d.unit_eps);
        fy /= sqrtf(wave_sum_fast(yy) + a.d.unit_eps);
      }
      xy = wave_sum_fast(xy);
#pragma unroll
      for (int e = 0; e < E; ++e) query[t][E * lane + e] = x[j][e] * fx, key[t][E * lane + e] = y[j][e] * fy;
#pragma unroll
      for (int e = 0; e < F; ++e) value[t][F * lane + e] = v[j][e];
      if (lane == 0) fade[t] = expf(lg[j]), gain[t] = b[j], both[t] = xy * fx * fy;
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const uint64_t row = (uint64_t)(q0 + t0 + t);
      f32x4 sk = {}, sq4 = {}, k[N / 4];
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        k[i] = *reinterpret_cast<const f32x4*>(&key[t][N * g + 4 * i]);
        const f32x4 x = *reinterpret_cast<const f32x4*>(&query[t][N * g + 4 * i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) sk += S[4 * i + j] * k[i][j], sq4 += S[4 * i + j] * x[j];
      }
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
      const f32x4 d = (*reinterpret_cast<const f32x4*>(&value[t][col]) - sk * f) * gain[t];
      if (tid < L) store4(a.out.p, kType, row * a.out.ts + (uint64_t)h * a.out.hs + col, sq4 * f + d * both[t]);
#pragma unroll
      for (int i = 0; i < N; ++i) S[i] = S[i] * f + d * k[i / 4][i % 4];
    }
  }
  if (target >= 0) {
    float* p = sq.states + ((uint64_t)target * a.d.value_heads + h) * (DK * DV) + col;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<f32x4*>(p + (N * g + i) * DV) = S[i];
  }
}

// ---- many tokens: chunks of 64 -------------------------------------------------------------
// With G_i the sum of the chunk's log decays up to token i, S the state before it, and
//   A_ij = beta_i k_i.k_j e^(G_i - G_j) for j < i,  T = (I + A)^-1,
// the corrections of the chunk's tokens are V' = T beta (V - e^G K S), and
//   out = scale (e^G Q S + P V'), P_ij = q_i.k_j e^(G_i - G_j) for j <= i;   S' = e^(G_63) S + (e^(G_63 - G) K)^T V'.
// T and P do not need the state: k_delta_prepare works them out for all chunks at once; k_delta_chunks then goes
// through a sequence's chunks, a workgroup for 16 columns of a head's state.
//
// Where decays above 0 add up to more than a factor of two within a chunk, A, T and the powers above could leave 32 bits though
// the rule itself does not (64 tokens of g = 2, beta 0 but for the last one's): such a chunk of a head goes token by token through
// k_delta_chunks, as k_delta_step would take it (1024 tokens, 32 heads of 128, all growing: 680 us, else 50 us).
//
// States are held to 32 bits: S, T, V - K S and V' enter the 16-bit matrix instructions as sums of three bf16 parts (8 bits each),
// in as many products as reach 2^-24; P, and S and V' for the outputs alone, as two. k and q are exact: themselves in bf16, or,
// for f16, two bf16 parts. Two parts are 16 bits, which leave outputs of 8 or 11 bits as they would be: off from 64 bits by what the
// plain 32-bit form is, 1.7e-3 and 2.1e-4 of their norm (4096 tokens in bf16, seven prompts in f16).
constexpr int kChunk = 64;

typedef u32x4 Operand;  // 8 numbers of 16 bits of a lane: lane (m, g), row (or column) m, the 8 at 8 g of 32

__device__ __forceinline__ f32x4 mfma_bf16(Operand a, Operand b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
typedef short bf16x4_bits __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma_bf16(u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16x4_bits, a), __builtin_bit_cast(bf16x4_bits, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f16(Operand a, Operand b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Four numbers as N sums of bf16 parts, the largest first.
template <int N>
__device__ __forceinline__ void split(f32x4 x, u32x2 (&part)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    part[i] = u32x2{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w)};
    asm("" : "+v"(part[i]));  // taken apart again below, not rounded anew
    if (i + 1 < N) {
      const f32x2 a = unpack_bf16(part[i].x), b = unpack_bf16(part[i].y);
      x -= f32x4{a.x, a.y, b.x, b.y};
    }
  }
}

constexpr float kFits = 0x1.ffp127f;  // from here on a first part of 8 bits is infinite

// What k_delta_prepare leaves, in the order of the lanes that read it: operands of 1 KB.
// A chunk's tokens 32 s + 4 g + r and 32 s + 16 + 4 g + r (r = 0..3) are, in turn, the 8 numbers of lane group g in step s of a sum
// over tokens: what the lanes of a product's result hold of two tiles of 16.
// The state's row 16 t + 4 g + r is the key's element 32 (t / 2) + 8 g + 4 (t % 2) + r: so the sums over a key's elements
// read 8 adjacent ones.
template <int DK, int NP>
struct DeltaImage {
  static constexpr int kT = 0;                // [tile and step][3 parts]: T beta
  static constexpr int kP = 18 * 1024;        // [tile and step][2 parts]: scale P
  static constexpr int kVec = 30 * 1024;      // f32: [64] of K S, [64] of Q S, [64] of V', [0] of S
  static constexpr int kSlow = 31 * 1024;     // of a chunk token by token: kVec has [64] -1, [64] of a query, [64] beta, here are [64] of a key, [64] exp(g)
  static constexpr int kValue = kSlow + 512;  // bytes of a value head's chunk
  static constexpr int kK = 0;                // [tile of tokens][step][NP]
  static constexpr int kQ = DK / 8 * NP * 1024;
  static constexpr int kKT = 2 * kQ;          // [tile of the state's rows][step][NP]
  static constexpr int kKey = 3 * kQ;         // bytes of a key head's chunk
  // Tile w of T and P needs the steps 0 .. w / 2.
  static __device__ __forceinline__ int lower(int w, int s) { return w < 2 ? w : 2 * (w - 1) + s; }
};

struct Long {
  uint32_t s, start;  // a sequence of this path, the number of its first chunk
};

struct ChunkArgs {
  DeltaArgs a;
  uint8_t *values, *keys;  // images [chunk][value head], [chunk][key head]
  float* carry;            // [2][value head][state]: of the sequences that go on in the next launch
  uint32_t first, last;    // chunks of this launch, by their numbers
  int least;               // sequences of fewer tokens are not this path's
  int dense;               // chunks and sequences are numbered among those that are
  Long* list;              // of many sequences: those of this path, n_long entries
  uint32_t n_long;
};

// Each workgroup looks through so many; of more, k_delta_list lists the long ones first. Launches for as many as there are sequences
// instead grew with the square of these (4000 single tokens, 32 heads of 128: 28 ms, with the list 0.48 ms).
constexpr uint32_t kDenseSeqs = 1024;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// The list's last entry whose first chunk is `chunk` or before, 64 candidates at a time; all 64 lanes active.
__device__ __forceinline__ uint32_t find_long(const ChunkArgs& c, uint32_t chunk) {
  uint32_t lo = 0, n = c.n_long;
  for (;;) {
    const uint32_t step = (n + 63) / 64, at = (threadIdx.x & 63) * step;
    const int k = __popcll(__ballot(at < n && c.list[lo + at].start <= chunk));
    const uint32_t past = k > 0 ? (uint32_t)(k - 1) * step : 0;
    lo += past, n = min(step, n - past);
    if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
  }
}

// Sequence number i of this path (chunk: the one that chunk number i is in), the number of its first chunk, its rows. With a list,
// sequences are numbered from the one that the launch's first chunk is in.
struct Chunked {
  uint32_t s, start;
  int q0, q1;
};
__device__ __forceinline__ bool find_sequence(const ChunkArgs& c, uint32_t i, bool chunk, Chunked& r) {
  const Sequences& q = c.a.s;
  if (c.list) {
    const uint32_t at = chunk ? find_long(c, i) : find_long(c, c.first) + i;
    if (at >= c.n_long || c.list[at].start == kNone) return false;
    r.s = __builtin_amdgcn_readfirstlane(c.list[at].s), r.start = __builtin_amdgcn_readfirstlane(c.list[at].start);
    rows_of(q.cu, q.n_rows, r.s, r.q0, r.q1);
    return true;
  }
  if (!c.dense) {
    r.s = chunk ? find_seq(q.cu, q.n_seqs, q.n_rows, 1, 6, i) : i;
    r.start = first_tile(q.cu, q.n_rows, r.s, 1, 6);
    rows_of(q.cu, q.n_rows, r.s, r.q0, r.q1);
    return r.q1 - r.q0 >= c.least;
  }
  uint32_t seqs = 0, chunks = 0;
  for (uint32_t s0 = 0; s0 < q.n_seqs; s0 += 64) {
    const uint32_t s = s0 + (threadIdx.x & 63);
    int q0 = 0, q1 = 0;
    if (s < q.n_seqs) rows_of(q.cu, q.n_rows, s, q0, q1);
    const uint32_t here = s < q.n_seqs && q1 - q0 >= c.least, n = here ? (uint32_t)(q1 - q0 + kChunk - 1) / kChunk : 0;
    const uint32_t at = wave_prefix(here), sum = wave_prefix(n);
    const uint64_t past = __ballot(chunk ? chunks + sum > i : seqs + at > i);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      r.s = s0 + l, r.start = chunks + __builtin_amdgcn_readlane(sum - n, l);
      r.q0 = __builtin_amdgcn_readlane(q0, l), r.q1 = __builtin_amdgcn_readlane(q1, l);
      return true;
    }
    seqs += __builtin_amdgcn_readlane(at, 63), chunks += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The long sequences of many, in order, by one workgroup: a thread counts those of a few adjacent ones, then writes them behind what
// the threads before it have. Entries behind the last have no first chunk.
__global__ __launch_bounds__(1024) void k_delta_list(ChunkArgs c) {
  __shared__ uint32_t sums[16][2];
  const Sequences& q = c.a.s;
  const uint32_t each = (q.n_seqs + 1023) / 1024, s0 = min(threadIdx.x * each, q.n_seqs), s1 = min(s0 + each, q.n_seqs);
  const int wave = threadIdx.x >> 6;
  auto chunks_of = [&](uint32_t s) {
    int q0, q1;
    rows_of(q.cu, q.n_rows, s, q0, q1);
    return q1 - q0 >= c.least ? (uint32_t)(q1 - q0 + kChunk - 1) / kChunk : 0;
  };
  uint32_t seqs = 0, chunks = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t n = chunks_of(s);
    seqs += n > 0, chunks += n;
  }
  const uint32_t at = wave_prefix(seqs), sum = wave_prefix(chunks);
  if ((threadIdx.x & 63) == 63) sums[wave][0] = at, sums[wave][1] = sum;
  __syncthreads();
  uint32_t i = at - seqs, start = sum - chunks, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < wave) i += sums[w][0], start += sums[w][1];
    all += sums[w][0];
  }
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t n = chunks_of(s);
    if (n && i < c.n_long) c.list[i] = Long{s, start};
    i += n > 0, start += n;
  }
  for (uint32_t j = all + threadIdx.x; j < c.n_long; j += 1024) c.list[j] = Long{0, kNone};
}

// Chunk number `at`: its first row and its rows.
__device__ __forceinline__ bool find_chunk(const ChunkArgs& c, uint32_t at, int& row, int& n) {
  Chunked r;
  if (!find_sequence(c, at, true, r)) return false;
  const int64_t i = (int64_t)at - r.start;
  if (i < 0 || i * kChunk >= r.q1 - r.q0) return false;
  row = r.q0 + (int)i * kChunk, n = min(kChunk, r.q1 - row);
  return true;
}

// The sum of lanes 0 .. l in lane l, by wave_prefix's moves.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_moved(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const u32x2 x = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, ROWS, 0xF, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, ROWS, 0xF, false)};
  return v + __builtin_bit_cast(double, x);
}
__device__ __forceinline__ double wave_prefix(double v) {
  v = add_moved<0x111, 0xF>(v), v = add_moved<0x112, 0xF>(v), v = add_moved<0x114, 0xF>(v), v = add_moved<0x118, 0xF>(v);
  return add_moved<0x143, 0xC>(add_moved<0x142, 0xA>(v));
}

// A chunk of a value head; the first head that shares a key head also lays out that one's operands. 4096 tokens, 16 key heads and
// 32 value heads of 128 in bf16: 48 us, two rounds of workgroups, for 114 MB written (2.4 TB/s) and 16 GFLOP; what bounds it is
// the way of a workgroup through its short serial steps, not one of these rates.
//
// A^T and T lie in one square: A^T above the diagonal, T = (I + A)^-1 on it and below.
template <int DK, bool BF>
__global__ __launch_bounds__(256, 4) void k_delta_prepare(ChunkArgs c) {
  constexpr int NP = BF ? 1 : 2, NS = DK / 32, kPad = 68;
  using I = DeltaImage<DK, NP>;
  __shared__ union {
    float m[kChunk][kPad];
    uint16_t keys[kChunk][DK + 8];
  } lds __attribute__((aligned(16)));
  __shared__ __attribute__((aligned(16))) float hi[kChunk], lo[kChunk], beta[kChunk], unit_k[kChunk], unit_q[kChunk];
  __shared__ __attribute__((aligned(16))) int bad[kChunk], slow;
  const DeltaArgs& a = c.a;
  const uint32_t h = blockIdx.x, group = a.d.value_heads / a.d.key_heads, hk = h / group;
  int row, n;
  if (!find_chunk(c, c.first + blockIdx.y, row, n)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  uint8_t* image = c.values + ((uint64_t)blockIdx.y * a.d.value_heads + h) * I::kValue;
  uint8_t* key_image = c.keys + ((uint64_t)blockIdx.y * a.d.key_heads + hk) * I::kKey;

  // rows of keys and queries as operands, zeros behind the last
  auto rows16 = [&](const Heads& x, int t, int s) {
    const int i = 16 * t + m;
    const uint8_t* p = static_cast<const uint8_t*>(x.p) + ((uint64_t)row * x.ts + (uint64_t)hk * x.hs) * 2;
    const Operand v = *reinterpret_cast<const Operand*>(p + (uint32_t)(min(i, n - 1) * (int)x.ts * 2 + 64 * s + 16 * g));
    return i < n ? v : Operand{0, 0, 0, 0};
  };
  auto squares = [&](const Operand (&x)[NS]) {
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 y = BF ? unpack_bf16(x[s][e]) : unpack_f16(x[s][e]);
        v = fmaf(y.x, y.x, v), v = fmaf(y.y, y.y, v);
      }
    return add_xor16(add_xor32(v));
  };
  auto dot = [](Operand x, Operand y, f32x4 z) { return BF ? mfma_bf16(x, y, z) : mfma_f16(x, y, z); };
  Operand kw[NS], qw[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) kw[s] = rows16(a.k, wave, s), qw[s] = rows16(a.q, wave, s);
  float lg = 0.f, b = 0.f;
  if (wave == 0 && lane < n) gates(a, (uint64_t)(row + lane), h, lg, b);  // the wave with the fewest products below
  // Products of this wave's 16 tokens with the earlier ones: rows are the earlier tokens, this wave's the columns.
  f32x4 kk[4] = {}, pt[4] = {};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t > wave) break;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const Operand k = t == wave ? kw[s] : rows16(a.k, t, s);
      kk[t] = dot(k, kw[s], kk[t]), pt[t] = dot(k, qw[s], pt[t]);
    }
  }
  {
    const float k2 = squares(kw), q2 = squares(qw);
    if (g == 0) {
      unit_k[16 * wave + m] = a.d.unit_eps > 0.f ? 1.f / sqrtf(k2 + a.d.unit_eps) : 1.f;
      unit_q[16 * wave + m] = a.d.scale * (a.d.unit_eps > 0.f ? 1.f / sqrtf(q2 + a.d.unit_eps) : 1.f);
      bad[16 * wave + m] = !(k2 < INFINITY);
    }
    if (h % group == 0) {
#pragma unroll
      for (int s = 0; s < NS; ++s) *reinterpret_cast<Operand*>(&lds.keys[16 * wave + m][32 * s + 8 * g]) = kw[s];
    }
  }
  __syncthreads();
  if (h % group == 0) {
    // A key head's operands: f16 numbers as two bf16 ones.
    auto put = [&](uint8_t* to, Operand x) {
      if constexpr (BF) {
        *reinterpret_cast<Operand*>(to + lane * 16) = x;
      } else {
        u32x2 part[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x2 y = unpack_f16(x[2 * e]), z = unpack_f16(x[2 * e + 1]);
          split(f32x4{y.x, y.y, z.x, z.y}, part[e]);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
          *reinterpret_cast<Operand*>(to + p * 1024 + lane * 16) = Operand{part[0][p].x, part[0][p].y, part[1][p].x, part[1][p].y};
      }
    };
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      put(key_image + I::kK + (wave * NS + s) * NP * 1024, kw[s]);
      put(key_image + I::kQ + (wave * NS + s) * NP * 1024, qw[s]);
    }
    for (int t = wave; t < DK / 16; t += 4) {
      const int e = 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Operand x;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int j = 32 * s + 16 * (y >> 1) + 4 * g + 2 * (y & 1);
          x[y] = (uint32_t)lds.keys[j][e] | (uint32_t)lds.keys[j + 1][e] << 16;
        }
        put(key_image + I::kKT + (t * 2 + s) * NP * 1024, x);
      }
    }
  }
  if (wave == 0) {
    // Sums of the decays in powers of two and 64 bits, kept as two numbers of 32: what two sums differ by is what counts. A token whose
    // key, decay or beta is not finite counts as none here, and as NaN for all that comes after it.
    const bool wrong = bad[lane] || !(lg < INFINITY) || !(fabsf(b) < INFINITY);
    if (wrong) lg = 0.f, b = 0.f;
    const bool grows = __any(lg > 0.f) && wave_sum_fast(fmaxf(lg, 0.f)) > 0.6931f;
    if (lane == 0) slow = grows;
    const double sum = wave_prefix(fmax((double)lg, -1e4) * 1.4426950408889634);
    hi[lane] = (float)sum, lo[lane] = (float)(sum - (double)(float)sum), beta[lane] = b, bad[lane] = wrong;
    const double end = __shfl(sum, 63, 64);
    const float rise = __builtin_amdgcn_exp2f((float)sum), fall = __builtin_amdgcn_exp2f((float)(end - sum));
    float* vec = reinterpret_cast<float*>(image + I::kVec);
    vec[lane] = wrong ? NAN : rise * unit_k[lane];
    vec[64 + lane] = rise * unit_q[lane];
    vec[128 + lane] = fall * unit_k[lane];
    if (lane == 0) vec[192] = __builtin_amdgcn_exp2f((float)end);
  }
  __syncthreads();
  auto go_by_tokens = [&] {  // what a token needs by itself; NaN and infinities as they are
    float g1 = 0.f, b1 = 0.f;
    if (lane < n) gates(a, (uint64_t)(row + lane), h, g1, b1);
    float *vec = reinterpret_cast<float*>(image + I::kVec), *more = reinterpret_cast<float*>(image + I::kSlow);
    vec[lane] = -1.f, vec[64 + lane] = unit_q[lane], vec[128 + lane] = b1;
    more[lane] = unit_k[lane], more[64 + lane] = expf(g1);
  };
  if (slow) {
    if (wave == 0) go_by_tokens();
    return;
  }
  const int i = 16 * wave + m;
  {
    const float hi_i = hi[i], lo_i = lo[i], gain = unit_k[i] * beta[i], of_q = unit_q[i];
    const bool bad_i = bad[i];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t > wave) break;
      const int j0 = 16 * t + 4 * g;
      const f32x4 hi_j = *reinterpret_cast<const f32x4*>(hi + j0), lo_j = *reinterpret_cast<const f32x4*>(lo + j0);
      const f32x4 unit_j = *reinterpret_cast<const f32x4*>(unit_k + j0);
      const i32x4 bad_j = *reinterpret_cast<const i32x4*>(bad + j0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = unit_j[r] * __builtin_amdgcn_exp2f((hi_i - hi_j[r]) + (lo_i - lo_j[r]));
        const float x = bad_i || bad_j[r] ? 0.f : kk[t][r] * f * gain;
        if (t < wave || 4 * g + r < m) lds.m[j0 + r][i] = x;
        pt[t][r] = (t < wave || 4 * g + r <= m) && !bad_j[r] ? pt[t][r] * f * of_q : 0.f;
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s > wave / 2) break;
    u32x2 x[2], y[2];
    split(pt[2 * s], x), split(pt[2 * s + 1], y);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *reinterpret_cast<Operand*>(image + I::kP + (I::lower(wave, s) * 2 + p) * 1024 + lane * 16) = Operand{x[p].x, x[p].y, y[p].x, y[p].y};
  }
  __syncthreads();
  // Blocks of 16 on the diagonal, column m of the transposed one from its last row up; then, a diagonal of blocks after the
  // other and in products of 32 bits, T^T_je = -T^T_jj sum_(k = j + 1 .. e) A^T_jk T^T_ke.
  {
    float w[16], column[16];  // lane m has the block's column m: row r's numbers come from the lanes
#pragma unroll
    for (int r = 0; r < 15; ++r) column[r] = lds.m[16 * wave + r][i];
#pragma unroll
    for (int r = 15; r >= 0; --r) {
      float v = r == m ? 1.f : 0.f;
#pragma unroll
      for (int k = r + 1; k < 16; ++k) v = fmaf(-bits_f32(__builtin_amdgcn_readlane(__float_as_uint(column[r]), k)), w[k], v);
      w[r] = v;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (g == r >> 2 && r <= m) lds.m[i][16 * wave + r] = w[r];
  }
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int j = wave, e = wave + d;
    if (e < 4) {
      f32x4 y = {}, z = {};
      for (int k = j + 1; k <= e; ++k) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(&lds.m[16 * j + m][16 * k + 4 * g]);
        f32x4 w = *reinterpret_cast<const f32x4*>(&lds.m[16 * e + m][16 * k + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (k == e && 4 * g + r > m) w[r] = 0.f;  // the other matrix's side of the diagonal
          y = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], w[r], y, 0, 0, 0);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = 4 * g + r >= m ? lds.m[16 * j + 4 * g + r][16 * j + m] : 0.f;
        z = __builtin_amdgcn_mfma_f32_16x16x4f32(x, y[r], z, 0, 0, 0);
      }
      *reinterpret_cast<f32x4*>(&lds.m[16 * e + m][16 * j + 4 * g]) = -z;
    }
    __syncthreads();
  }
  bool over = false;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s > wave / 2) break;
    u32x2 part[2][3];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x4 v = {};
      if (2 * s + x <= wave) {
        const int j = 32 * s + 16 * x + 4 * g;
        v = *reinterpret_cast<const f32x4*>(&lds.m[i][j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = j + r <= i ? v[r] * beta[j + r] : 0.f;
          over |= !(fabsf(v[r]) < kFits);
        }
      }
      split(v, part[x]);
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<Operand*>(image + I::kT + (I::lower(wave, s) * 3 + p) * 1024 + lane * 16) =
          Operand{part[0][p].x, part[0][p].y, part[1][p].x, part[1][p].y};
  }
  // What two tokens do to each other, long keys or a large beta, can leave 32 bits too, and would be multiplied with zeros then.
  if (__any(over) && lane == 0) slow = 1;
  __syncthreads();
  if (slow && wave == 0) go_by_tokens();
}

// A sequence's chunks for 16 columns of a head's state. What the next chunk waits for is the state alone, through three steps:
// V - K S, V', S. Four waves take them, each result going from one wave's registers through LDS to all: wave w has the state's
// tiles of 16 rows from w * (DK / 64) on, whose part of K S it works out for the whole chunk, and the chunk's tokens from 16 w on
// after that. Four others work out the tokens' outputs beside them, a step behind. A chunk takes 1.8 us (4096 tokens of one sequence,
// 32 heads of 128, all 256 CUs: 115 us): three barriers, exchanges through LDS and 78 KB of operands by the CU's loads, 580 cycles
// of each wave's matrix instructions. In 128 registers two workgroups share a CU, where there are so many: seven prompts of 12 heads,
// f16 keys of 64, 73 us with one and 60 us with two; 32 heads of 128 in bf16, 156 and 132 us, though 3 and 5 registers are spilled for it. f16 keys
// of 128, in two parts, would spill 96 (214 us with one, 524 us).
template <int DK, int NP, bool BF>
__global__ __launch_bounds__(512, (DK == 64 || NP == 1 ? 4 : 2)) void k_delta_chunks(ChunkArgs c, uint32_t slices, int parity) {
  constexpr int NS = DK / 32, NT = DK / 64;
  constexpr bool kLate = DK == 128 && NP == 1;  // T is asked for a step later: there is no room for it before
  using I = DeltaImage<DK, NP>;
  __shared__ __attribute__((aligned(16))) uint8_t state[NS][2][1024], rest[2][3][1024], faded[2][3][1024];
  __shared__ f32x4 fresh[4][64], sums[4][4][64];
  __shared__ __attribute__((aligned(16))) int first_bad[4][16], any_bad[4];
  const DeltaArgs& a = c.a;
  const Sequences& q = a.s;
  // Workgroups go to the 8 XCDs in turn: the slices of a head, which read the same operands, to one of them.
  const uint32_t unit = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), h = unit / slices, slice = unit % slices;
  if (c.least == 0 && blockIdx.x == 0 && blockIdx.y == 0) check_offsets(q.cu, q.n_seqs, q.n_rows, q.err, kErrPacked);  // else k_delta_step has
  Chunked seq;
  if (h >= a.d.value_heads || !find_sequence(c, blockIdx.y, false, seq)) return;
  const uint32_t hk = h / (a.d.value_heads / a.d.key_heads), DV = a.d.value_dim;
  const int number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = number & 3;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const bool outputs = number >= 4;
  const uint32_t s = seq.s, start = seq.start;
  const int q0 = seq.q0, q1 = seq.q1, n = q1 - q0;
  const uint32_t count = (n + kChunk - 1) / kChunk;
  const uint32_t end = start + max(count, 1u);  // a sequence without tokens takes part in one launch
  if (end <= c.first || start >= c.last) return;
  const uint32_t begin = max(start, c.first), stop = min(start + count, c.last);

  auto operand = [&](const uint8_t* p) { return *reinterpret_cast<const Operand*>(p + lane * 16); };
  // The operands of a chunk are on their way while the chunk before is worked on: each part is asked for as soon as its
  // registers have been read. The last chunk loads itself again: a wait for one load must know how many others there
  // are behind it.
  const uint64_t value_step = (uint64_t)a.d.value_heads * I::kValue, key_step = (uint64_t)a.d.key_heads * I::kKey;
  const uint8_t* image = c.values + (uint64_t)(begin - c.first) * value_step + (uint64_t)h * I::kValue;
  const uint8_t* key_image = c.keys + (uint64_t)(begin - c.first) * key_step + (uint64_t)hk * I::kKey;
  const int t0 = 16 * wave + 4 * g;
  int row = q0 + (int)(begin - start) * kChunk;

  if (outputs) {
    if (begin >= stop) return;
    Operand Q[NS][NP], P[2][2];
    f32x4 of_q;
    float slow;
    auto load = [&] {
      slow = *reinterpret_cast<const float*>(image + I::kVec);
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int p = 0; p < NP; ++p) Q[x][p] = operand(key_image + I::kQ + ((wave * NS + x) * NP + p) * 1024);
      of_q = *reinterpret_cast<const f32x4*>(image + I::kVec + 256 + (uint32_t)(4 * t0));
    };
    auto load_mix = [&] {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int p = 0; p < 2; ++p) P[x][p] = operand(image + I::kP + (I::lower(wave, min(x, wave / 2)) * 2 + p) * 1024);
    };
    const int step = (int)a.out.ts * 2;  // bytes from a token to the next
    f32x4 o = {};
    auto store = [&](int row) {
      uint8_t* out = static_cast<uint8_t*>(a.out.p) + ((uint64_t)row * a.out.ts + (uint64_t)h * a.out.hs + 16 * slice) * 2;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (row + t0 + r < q1)
          *reinterpret_cast<uint16_t*>(out + (uint32_t)((t0 + r) * step + 2 * m)) = (uint16_t)(BF ? pack_bf16(o[r], 0.f) : pack_f16(o[r], 0.f));
    };
    load(), load_mix();
    __syncthreads();
    bool left = false;  // outputs of the chunk before to be stored
    for (uint32_t chunk = begin; chunk < stop; ++chunk, row += kChunk) {
      const bool more = chunk + 1 < stop;
      if (__builtin_expect(slow < 0.f, 0)) {
        // the other waves take this chunk, with a barrier for each token
        if (left) store(row - kChunk);
        left = false;
        image += more ? value_step : 0, key_image += more ? key_step : 0;
        load(), load_mix();
        for (int t = min(kChunk, q1 - row); t > 0; --t) __syncthreads();
        __syncthreads();
        continue;
      }
      f32x4 qs[2] = {};  // sums of products of like size, so that they do not wait for each other
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const Operand S2[2] = {operand(state[x][0]), operand(state[x][1])};
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int z = 0; z + p < 2; ++z) qs[z + p] = mfma_bf16(Q[x][p], S2[z], qs[z + p]);
      }
      const f32x4 before = (qs[1] + qs[0]) * of_q;
      image += more ? value_step : 0, key_image += more ? key_step : 0;
      load();
      __syncthreads();
      if (left) store(row - kChunk);
      __syncthreads();
      const i32x4 bads = *reinterpret_cast<const i32x4*>(any_bad);
      f32x4 sum[2] = {};
      auto mix = [&](int x, f32x4 v0, f32x4 v1) {
        u32x2 lo[2], hi[2];
        split(v0, lo), split(v1, hi);
        const Operand v[2] = {{lo[0].x, lo[0].y, hi[0].x, hi[0].y}, {lo[1].x, lo[1].y, hi[1].x, hi[1].y}};
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int z = 0; z + p < 2; ++z) sum[z + p] = mfma_bf16(P[x][p], v[z], sum[z + p]);
      };
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > wave / 2) break;
        mix(x, fresh[2 * x][lane], fresh[2 * x + 1][lane]);
      }
      int first = kChunk;  // the column's first token that is not finite
      if (__builtin_expect(__any(!(fabsf(sum[0].x) + fabsf(sum[0].y) + fabsf(sum[0].z) + fabsf(sum[0].w) < INFINITY)), 0)) {
        // Corrections that are sums beyond 32 bits, as with V - K S below; all products again without them.
        sum[0] = f32x4{}, sum[1] = f32x4{};
#pragma unroll 1
        for (int x = 0; x <= wave / 2; ++x) {
          f32x4 now[2] = {fresh[2 * x][lane], fresh[2 * x + 1][lane]};
#pragma unroll
          for (int r = 7; r >= 0; --r)
            if (!(fabsf(now[r / 4][r % 4]) < kFits)) first = min(first, 32 * x + 16 * (r / 4) + 4 * g + r % 4), now[r / 4][r % 4] = 0.f;
          x ? mix(1, now[0], now[1]) : mix(0, now[0], now[1]);
        }
        first = min(first, __shfl_xor(first, 16, 64));
        first = min(first, __shfl_xor(first, 32, 64));
      }
      load_mix();
      o = before + (sum[1] + sum[0]);
      if (__builtin_amdgcn_readfirstlane(bads.x | bads.y | bads.z | bads.w)) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (bads[w]) first = min(first, first_bad[w][m]);
      }
      if (__any(first < kChunk)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + r >= first) o[r] = NAN;
      }
      left = true;
      __syncthreads();
    }
    if (left) store(row - kChunk);
    return;
  }

  const int source = slot_of(q, q.source, s), target = slot_of(q, q.target, s);
  const uint64_t state_size = (uint64_t)DK * DV;
  // this lane's numbers of a state: rows 4 g + r of each of the wave's tiles, one column
  auto at = [&](float* base, int t, int r) {
    const int x = wave * NT + t;
    return base + (uint64_t)(32 * (x >> 1) + 8 * g + 4 * (x & 1) + r) * DV + 16 * slice + m;
  };
  auto in_slot = [&](int slot) { return q.states + ((uint64_t)slot * a.d.value_heads + h) * state_size; };
  auto carry = [&](int parity) { return c.carry + ((uint64_t)parity * a.d.value_heads + h) * state_size; };
  f32x4 S[NT] = {};
  if (float* from = start < c.first ? carry(parity ^ 1) : source >= 0 ? in_slot(source) : nullptr) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] = *at(from, t, r);
  }
  if (begin < stop) {
    using Part = std::conditional_t<NT == 2, Operand, u32x2>;  // the wave's rows of the state as an operand
    Operand T[2][3], KT[NT][2][NP];
    Part K[4][NP];
    f32x4 of_k, of_v;
    float fade;
    uint16_t vals[4];
    const int step = (int)a.v.ts * 2;
    auto load_keys = [&] {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          K[t][p] = *reinterpret_cast<const Part*>(key_image + I::kK + ((t * NS + wave * NT / 2) * NP + p) * 1024 + lane * 16 + (NT == 1 ? 8 * (wave & 1) : 0));
    };
    auto vec = [&](int i) { return *reinterpret_cast<const f32x4*>(image + I::kVec + 256 * i + (uint32_t)(4 * t0)); };
    auto load_values = [&](int row) {
      of_k = vec(0);
      const uint8_t* v = static_cast<const uint8_t*>(a.v.p) + ((uint64_t)row * a.v.ts + (uint64_t)h * a.v.hs + 16 * slice) * 2;
#pragma unroll
      for (int r = 0; r < 4; ++r) vals[r] = *reinterpret_cast<const uint16_t*>(v + (uint32_t)(min(t0 + r, q1 - 1 - row) * step + 2 * m));
    };
    auto load_solution = [&] {
      of_v = vec(2);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int p = 0; p < 3; ++p) T[x][p] = operand(image + I::kT + (I::lower(wave, min(x, wave / 2)) * 3 + p) * 1024);
    };
    auto load_fade = [&](const uint8_t* keys) {
      fade = reinterpret_cast<const float*>(image + I::kVec)[192];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int p = 0; p < NP; ++p) KT[t][x][p] = operand(keys + I::kKT + (((wave * NT + t) * 2 + x) * NP + p) * 1024);
    };
    // The wave's part of K S for the next chunk. The state's tiles 2 s and 2 s + 1 are step s of the sums over a key's elements: as
    // an operand they are what their lanes hold.
    auto look = [&] {
      u32x2 part[NT][3];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        split(S[t], part[t]);
        const int x = wave * NT + t;
#pragma unroll
        for (int p = 0; p < 2; ++p) *reinterpret_cast<u32x2*>(&state[x >> 1][p][lane * 16 + 8 * (x & 1)]) = part[t][p];
      }
      f32x4 sum[4] = {};
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int z = 2 - p; z >= 0; --z) {
          Part y;
          if constexpr (NT == 2) y = Operand{part[0][z].x, part[0][z].y, part[1][z].x, part[1][z].y};
          else y = part[0][z];
#pragma unroll
          for (int t = 0; t < 4; ++t) sum[t] = mfma_bf16(K[t][p], y, sum[t]);
        }
#pragma unroll
      for (int t = 0; t < 4; ++t) sums[wave][t][lane] = sum[t];
    };
    // A chunk token by token: each wave's rows of the state, sums over the lanes and, through LDS, over the waves. The call's
    // arguments are read and the lane's places worked out here: kept through the other chunks they would push those's registers out.
    auto go_by_tokens = [&] {
      const __attribute__((address_space(4))) auto* c2 = (const __attribute__((address_space(4))) ChunkArgs*)__builtin_amdgcn_kernarg_segment_ptr();
      int lane2 = lane;
      asm volatile("" : "+s"(c2), "+v"(lane2));
      constexpr uint32_t kType = BF ? MR_BF16 : MR_F16;
      const uint32_t m = lane2 & 15, g = lane2 >> 4;
      const uint16_t* kp = static_cast<const uint16_t*>(c2->a.k.p) + (uint64_t)row * c2->a.k.ts + (uint64_t)hk * c2->a.k.hs;
      const uint16_t* qp = static_cast<const uint16_t*>(c2->a.q.p) + (uint64_t)row * c2->a.q.ts + (uint64_t)hk * c2->a.q.hs;
      const uint16_t* vp = static_cast<const uint16_t*>(c2->a.v.p) + (uint64_t)row * c2->a.v.ts + (uint64_t)h * c2->a.v.hs + 16 * slice;
      uint16_t* op = static_cast<uint16_t*>(c2->a.out.p) + (uint64_t)row * c2->a.out.ts + (uint64_t)h * c2->a.out.hs + 16 * slice;
      float(*red)[4][3][16] = reinterpret_cast<float(*)[4][3][16]>(&rest[0][0][0]);
      const float *vec = reinterpret_cast<const float*>(image + I::kVec), *of_key = reinterpret_cast<const float*>(image + I::kSlow);
      const int tokens = min(kChunk, q1 - row);
#pragma unroll 1
      for (int t = 0; t < tokens; ++t, kp += c2->a.k.ts, qp += c2->a.q.ts, vp += c2->a.v.ts, op += c2->a.out.ts) {
        f32x4 k[NT];
        float sum[3] = {};  // of S k, S q, k q
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int x = wave * NT + i;
          const uint32_t e = 32 * (x >> 1) + 8 * g + 4 * (x & 1);
          k[i] = load4(kp, kType, e) * of_key[t];
          const f32x4 y = load4(qp, kType, e) * vec[64 + t];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            sum[0] = fmaf(S[i][r], k[i][r], sum[0]), sum[1] = fmaf(S[i][r], y[r], sum[1]), sum[2] = fmaf(k[i][r], y[r], sum[2]);
        }
        const float v = BF ? bits_f32((uint32_t)vp[m] << 16) : (float)__builtin_bit_cast(_Float16, vp[m]);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          sum[i] = add_xor16(add_xor32(sum[i]));
          if (g == 0) red[t & 1][wave][i][m] = sum[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) sum[i] = (red[t & 1][0][i][m] + red[t & 1][1][i][m]) + (red[t & 1][2][i][m] + red[t & 1][3][i][m]);
        const float f = of_key[64 + t], d = (v - sum[0] * f) * vec[128 + t], o = fmaf(d, sum[2], sum[1] * f);
        if (wave == 0 && g == 0) op[m] = (uint16_t)(BF ? pack_bf16(o, 0.f) : pack_f16(o, 0.f));
#pragma unroll
        for (int i = 0; i < NT; ++i) S[i] = S[i] * f + k[i] * d;
      }
    };
    load_keys(), load_values(row), load_solution(), load_fade(key_image);
    look();
    __syncthreads();
    for (uint32_t chunk = begin; chunk < stop; ++chunk, row += kChunk) {
      const bool more = chunk + 1 < stop;
      const int half = lane * 16 + 8 * (wave & 1);  // of the step that the wave's tokens are in
      // Loads are asked for behind a step's reads of LDS, while these are on their way.
      const f32x4 part0 = sums[0][wave][lane], part1 = sums[1][wave][lane], part2 = sums[2][wave][lane], part3 = sums[3][wave][lane];
      __builtin_amdgcn_sched_barrier(0);
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(__float_as_int(of_k[0])) == __float_as_int(-1.f), 0)) {
        go_by_tokens();
        key_image += more ? key_step : 0, image += more ? value_step : 0;
        load_keys(), load_values(row + (more ? kChunk : 0)), load_solution(), load_fade(key_image);
        look();
        __syncthreads();
        continue;
      }
      key_image += more ? key_step : 0, image += more ? value_step : 0;
      load_keys();
      __builtin_amdgcn_sched_barrier(0);
      f32x4 R = (part0 + part1) + (part2 + part3);
      bool wrong = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = row + t0 + r < q1 ? (BF ? bits_f32((uint32_t)vals[r] << 16) : (float)__builtin_bit_cast(_Float16, vals[r])) : 0.f;
        R[r] = fmaf(-of_k[r], R[r], v);
        wrong |= !(fabsf(R[r]) < kFits);
      }
      const bool any = __any(wrong);
      if (any) {
        // NaN would reach earlier tokens by the zeros it is multiplied with: it is taken out, and the column's tokens from here
        // on are NaN at the end
        int bad = kChunk;
#pragma unroll
        for (int r = 3; r >= 0; --r)
          if (!(fabsf(R[r]) < kFits)) bad = t0 + r, R[r] = 0.f;
        bad = min(bad, __shfl_xor(bad, 16, 64));
        bad = min(bad, __shfl_xor(bad, 32, 64));
        if (g == 0) first_bad[wave][m] = bad;
      }
      if (lane == 0) any_bad[wave] = any;
      {
        u32x2 part[3];
        split(R, part);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2*>(&rest[wave >> 1][p][half]) = part[p];
      }
      __syncthreads();
      const i32x4 bads = *reinterpret_cast<const i32x4*>(any_bad);
      f32x4 V;
      {
        f32x4 sum[3] = {};  // sums of products of like size, so that they do not wait for each other
        Operand y[2][3];
#pragma unroll
        for (int p = 0; p < 3; ++p) y[0][p] = operand(rest[0][p]), y[1][p] = operand(rest[1][p]);
        __builtin_amdgcn_sched_barrier(0);
        load_values(row + (more ? kChunk : 0));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (x > wave / 2) break;
#pragma unroll
          for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int z = 0; z + p < 3; ++z) sum[z + p] = mfma_bf16(T[x][p], y[x][z], sum[z + p]);
        }
        V = (sum[2] + sum[1]) + sum[0];
      }
      fresh[wave][lane] = V;
      {
        u32x2 part[3];
        split(V * of_v, part);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2*>(&faded[wave >> 1][p][half]) = part[p];
      }
      bool lost = false;
      if (__builtin_amdgcn_readfirstlane(bads.x | bads.y | bads.z | bads.w)) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          lost |= bads[w] && first_bad[w][m] < kChunk;
      }
      __syncthreads();
      {
        Operand y[2][3];
#pragma unroll
        for (int p = 0; p < 3; ++p) y[0][p] = operand(faded[0][p]), y[1][p] = operand(faded[1][p]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!kLate) { load_solution(); __builtin_amdgcn_sched_barrier(0); }
        const float keep = lost ? NAN : fade;
        f32x4 sum[NT][3] = {};
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int z = 0; z + p < 3; ++z)
#pragma unroll
              for (int t = 0; t < NT; ++t) sum[t][z + p] = mfma_bf16(KT[t][x][p], y[x][z], sum[t][z + p]);
#pragma unroll
        for (int t = 0; t < NT; ++t) S[t] = S[t] * keep + ((sum[t][2] + sum[t][1]) + sum[t][0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_fade(key_image);
      __builtin_amdgcn_sched_barrier(0);
      look();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kLate) load_solution();
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
    }
  }
  float* to = end > c.last ? carry(parity) : target >= 0 ? in_slot(target) : nullptr;
  if (!to || (n == 0 && target == source)) return;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) *at(to, t, r) = S[t][r];
}

template <int DK, int DV>
void launch_step(const Launch& K, bool bf, const DeltaArgs& a, int most) {
  const dim3 g(a.d.value_heads, a.s.n_seqs), b(256);
  hipLaunchKernelGGL((bf ? k_delta_step<DK, DV, true> : k_delta_step<DK, DV, false>), g, b, 0, K.s, a, most);
}

// Sequences of up to so many tokens go through k_delta_step, whose workgroups of one sequence take 1.1 us a token; the other two
// kernels take 19 us for a sequence's first chunk, each further sequence about 3.5 us of all CUs. 32 heads of 128, step : chunks (us):
// one sequence of 16 tokens 22 : 18, of 32, 40 : 19 (of 33); 4 sequences of 32, 44 : 30 (of 33); 16 of 16, 38, of 32, 63 : 72 (of 40).
int step_tokens(uint32_t n_seqs, uint32_t value_heads) { return (int)std::min<uint64_t>(32, 12 + (uint64_t)n_seqs * value_heads / 16); }
constexpr uint64_t kScratch = 256ull << 20;

template <int DK, bool BF>
hipError_t launch_chunks(const Launch& K, const DeltaArgs& a, int least, uint8_t* scratch) {
  using I = DeltaImage<DK, BF ? 1 : 2>;
  const uint32_t vh = a.d.value_heads, kh = a.d.key_heads, dv = a.d.value_dim;
  const uint32_t longest = least ? (uint32_t)a.s.n_rows / (uint32_t)least : a.s.n_seqs;  // sequences of so many tokens at most
  const uint32_t seqs = std::min(a.s.n_seqs, longest);
  const bool listed = least && a.s.n_seqs > kDenseSeqs;
  const uint64_t list = listed ? ((uint64_t)seqs * sizeof(Long) + 1023) / 1024 * 1024 : 0;
  const uint64_t carry = 2ull * vh * DK * dv * sizeof(float), chunk = (uint64_t)vh * I::kValue + (uint64_t)kh * I::kKey;
  const uint32_t all = ((uint32_t)a.s.n_rows >> 6) + seqs, room = (uint32_t)std::min<uint64_t>((kScratch - list - carry) / chunk, 65535);
  ChunkArgs c{a, nullptr, nullptr, reinterpret_cast<float*>(scratch + list), 0, 0, least, least > 0, nullptr, 0};
  if (listed) {
    ProfScope ps(K, "delta_list");
    c.list = reinterpret_cast<Long*>(scratch), c.n_long = seqs;
    hipLaunchKernelGGL(k_delta_list, dim3(1), dim3(1024), 0, K.s, c);
  }
  int parity = 0;
  for (c.first = 0; c.first < all; c.first = c.last, parity ^= 1) {
    c.last = std::min(all, c.first + room);
    c.values = scratch + list + carry;
    c.keys = c.values + (uint64_t)(c.last - c.first) * vh * I::kValue;
    {
      ProfScope ps(K, "delta_prepare");
      hipLaunchKernelGGL((k_delta_prepare<DK, BF>), dim3(vh, c.last - c.first), dim3(256), 0, K.s, c);
    }
    ProfScope ps(K, "delta_chunks");
    hipLaunchKernelGGL((k_delta_chunks<DK, BF ? 1 : 2, BF>), dim3((vh * (dv / 16) + 7) / 8 * 8, listed ? std::min(seqs, c.last - c.first) : seqs), dim3(512), 0, K.s, c, dv / 16, parity);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

uint64_t delta_scratch_bytes() { return kScratch; }

hipError_t launch_delta_rule(const Launch& K, const DeltaShape& d, const Heads& q, const Heads& k, const Heads& v,
                             const float* decay, const float* beta, const Sequences& s, const Heads& out, void* scratch) {
  const DeltaArgs a{d, q, k, v, out, decay, beta, s};
  const bool bf = q.dtype == MR_BF16;
  // One sequence takes one path, and so do a few rows of sequences that are all short if none is without tokens: two more launches
  // would cost batches of single tokens 7 us (48 sequences: of 47; 160: of 131). If some are, one long sequence of so few rows, 1.1 us a
  // token, goes token by token.
  const int few = step_tokens(s.n_seqs, d.value_heads);
  const bool chunks = (int64_t)s.n_rows - s.n_seqs + 1 > few || s.n_rows > 8 * few, steps = !chunks || s.n_seqs > 1;
  if (steps) {
    ProfScope ps(K, "delta_step");
    const int most = chunks ? few : s.n_rows;
    if (d.key_dim == 64 && d.value_dim == 64) launch_step<64, 64>(K, bf, a, most);
    if (d.key_dim == 64 && d.value_dim == 128) launch_step<64, 128>(K, bf, a, most);
    if (d.key_dim == 128 && d.value_dim == 64) launch_step<128, 64>(K, bf, a, most);
    if (d.key_dim == 128 && d.value_dim == 128) launch_step<128, 128>(K, bf, a, most);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !chunks) return e;
  }
  const int least = steps ? few + 1 : 0;
  uint8_t* w = static_cast<uint8_t*>(scratch);
  if (d.key_dim == 64) return bf ? launch_chunks<64, true>(K, a, least, w) : launch_chunks<64, false>(K, a, least, w);
  return bf ? launch_chunks<128, true>(K, a, least, w) : launch_chunks<128, false>(K, a, least, w);
}

}  // namespace mr
