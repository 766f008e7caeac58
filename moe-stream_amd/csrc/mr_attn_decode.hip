// mr_attn_decode.hip -- attention of one query token per sequence over the paged cache.
//
// The cache is read once: 2 D FMT / 8 bytes (and the scales) a token and key head, and 4 D operations for each
// query head on them, so memory bounds it. The query heads that share a key head (up to 16) are the columns of
// 16x16x32 f16 matrix instructions, S = K Q^T and O = V^T P; the cached values are f16 numbers, so turning
// codes into operands rounds nothing. Pages lie in the order in which the lanes read them (KvLayout): no LDS,
// no barrier and no exchange of elements between lanes; a wave takes chunks of 64 tokens by itself.
//
// 32 sequences of 16000 tokens, 4 heads of 128: MXFP4 279 MB in 54 us, 5.2 TB/s, MXINT8 541 MB in 105 us, 5.2 TB/s; 16
// of 16000, 2 heads of 256, F16: 524 MB in 101 us, 5.2 TB/s; of the 6 TB/s that reading alone reaches here; what is missing
// is the launch and the first and last chunks, about 8 us.
// One short sequence is latency: 5.6 us.
//
// Weights are rounded to f16 for the second product, the largest of them 2^14 (kLift), and their sum is that of the rounded ones.
//
// The sequences' chunks are dealt out to the workgroups in parts of one size, so that a long sequence next to
// short ones is spread over many CUs; the parts of a sequence are joined by a second launch.
#include "mr_kv_operand.h"

namespace mr {

namespace {

struct DecodeArgs {
  KvPages kv;
  Heads q, out;
  const int32_t *len, *table;
  uint32_t max_pages, n_seqs;
  uint32_t heads;      // query heads of a key head
  uint32_t head_tiles; // tiles of 16 of them
  uint32_t parts;      // parts that the CUs hold at once; 1: a sequence a part
  AttnOpts o;
  uint32_t* err;
  float* part;         // [slot][key head][head tile][16][D] sums, then [slot][..][16][2] maximum and sum
};

constexpr int kWaves = 4;
constexpr uint32_t kPartUnits = 1024;  // most parts, times key heads and head tiles
constexpr uint32_t kMinPart = kWaves;  // chunks of a part at least: one for each wave
// Sequences that cannot have more chunks stay whole, which spares the second launch. One sequence of 1200 tokens whole
// and in parts: 11.8 and 13.9 us (MXFP4, 4 heads of 128), 24.7 and 16.7 us (MXINT8, 2 heads of 256, where a chunk
// takes a wave 4 us).
__host__ __device__ inline uint32_t whole_chunks(uint32_t D) { return D == 256 ? 2 * kWaves : 5 * kWaves; }
// With more sequences none is split: each workgroup looks through their lengths to find its part.
constexpr uint32_t kSplitSeqs = 1024;
// Parts of all sequences at most. Those of split sequences, two or more of each, are then no more than `parts`.
__host__ __device__ inline uint32_t part_limit(uint32_t parts, uint32_t n_seqs) {
  const uint32_t some = n_seqs + parts / 2;
  return parts > some ? parts : some;
}

// Which tokens of sequence b are seen, in chunks.
struct Span {
  int n, first;     // length, first token seen
  int c0, chunks;   // first chunk, number of chunks
  int bad;          // the length was out of range
};
__device__ __forceinline__ Span span_of(const DecodeArgs& a, uint32_t b) {
  const int64_t cap = (int64_t)a.max_pages << a.kv.page_shift;
  Span s;
  const int64_t len = a.len[b];
  s.n = (int)min(max(len, (int64_t)0), cap);
  s.bad = s.n != len;
  s.first = a.o.window && (uint32_t)s.n > a.o.window ? s.n - (int)a.o.window : 0;
  s.c0 = s.first >> 6;
  s.chunks = s.n ? ((s.n - 1) >> 6) + 1 - s.c0 : 0;
  return s;
}

// The sequence and part of index `i` among all parts (split_only: of the sequences of several parts, in
// which case the part is 0). Parts of `size` chunks; a sequence of no more than that is one part, one of no
// chunks too. slot: the number of parts of split sequences in front. A lane looks at a sequence; the lengths of
// up to 64 are read once.
struct Part {
  uint32_t b, part, parts, slot, size;
  Span sp;
};
__device__ __forceinline__ bool find_part(const DecodeArgs& a, uint32_t i, bool split_only, Part& r) {
  const uint32_t lane = threadIdx.x & 63;
  if (a.parts == 1) {
    if (split_only || i >= a.n_seqs) return false;
    r = Part{i, 0, 1, 0, 0x7FFFFFFFu, span_of(a, i)};
    return true;
  }
  auto span = [&](uint32_t b) { return b < a.n_seqs ? span_of(a, b) : Span{}; };
  Span s = span(lane);
  // f(chunks) of every sequence, summed
  auto sum_of = [&](auto f) {
    uint32_t v = lane < a.n_seqs ? f((uint32_t)s.chunks) : 0;
    for (uint32_t b0 = 64; b0 < a.n_seqs; b0 += 64)
      if (b0 + lane < a.n_seqs) v += f((uint32_t)span_of(a, b0 + lane).chunks);
    return wave_total(v);
  };
  // The smallest size, in steps of an eighth, at which the CUs hold all parts at once: a part more would run after
  // the others, alone (32 sequences up to 24000: 54 -> 49 us). Next to many sequences, the long ones are still split.
  const uint32_t all = sum_of([](uint32_t c) { return c; }), most = part_limit(a.parts, a.n_seqs);
  r.size = max(kMinPart, (all + a.parts - 1) / a.parts);
  while (r.size < all && sum_of([&](uint32_t c) { return max(1u, (c + r.size - 1) / r.size); }) > most) r.size += (r.size + 7) / 8;
  uint32_t before = 0, slots = 0;
  for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += 64) {
    if (b0) s = span(b0 + lane);
    const uint32_t n = b0 + lane < a.n_seqs ? max(1u, ((uint32_t)s.chunks + r.size - 1) / r.size) : 0;
    const uint32_t split = n > 1 ? n : 0, count = split_only ? split > 0 : n;
    const uint32_t sum = wave_prefix(count), ssum = wave_prefix(split);
    const uint64_t past = __ballot(before + sum > i);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      r.b = b0 + l;
      r.parts = __builtin_amdgcn_readlane(n, l);
      r.part = split_only ? 0 : i - before - __builtin_amdgcn_readlane(sum - count, l);
      r.slot = slots + __builtin_amdgcn_readlane(ssum - split, l);
      r.sp = Span{__builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.c0, l),
                  __builtin_amdgcn_readlane(s.chunks, l), __builtin_amdgcn_readlane(s.bad, l)};
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(ssum, 63);
  }
  return false;
}

// Waves of a SIMD, as many as the registers of a chunk and of the sums leave room for, and whether the next
// chunk's keys are on their way while this one's values are used. Measured: MXFP4, heads of 128, two waves and three:
// 62 and 54 us (32 sequences up to 24000); MXINT8, of 256, one wave and ahead, two and not: 34.6 and 31.6 us (100001
// tokens); F16, of 256, the same: 100 and 108 us (16 of 16000).
template <int FMT, int D>
struct Tuning {
  static constexpr int kPerSimd = D == 64 ? (FMT == 16 ? 3 : 4) : D == 128 ? (FMT == 4 ? 3 : 2) : FMT == 16 ? 1 : 2;
  static constexpr bool kAhead = !(D == 256 && FMT == 8);
};

template <int FMT, int D>
__global__ __launch_bounds__(64 * kWaves, (Tuning<FMT, D>::kPerSimd)) void k_attn_decode(DecodeArgs a) {
  constexpr int NT = D / 16;
  constexpr bool kAhead = Tuning<FMT, D>::kAhead;
  __shared__ __attribute__((aligned(16))) float sums[kWaves / 2][16 * D];
  __shared__ float stats[kWaves / 2][16][2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  Part pt;
  if (!find_part(a, blockIdx.x, false, pt)) return;
  const Span sp = pt.sp;
  if (threadIdx.x == 0 && blockIdx.y == 0 && pt.part == 0 && sp.bad) note_error(a.err, kErrLength);
  const uint32_t hk = blockIdx.y / a.head_tiles, h0 = 16 * (blockIdx.y % a.head_tiles);  // first query head within the group
  const uint32_t heads = min(16u, a.heads - h0);
  const uint32_t hq = hk * a.heads + h0 + min((uint32_t)n, heads - 1);  // this lane's query head (the last one repeated)

  // The query as f16, scaled by a power of two so that its largest element lies in [2^14, 2^15): exact for
  // f16, and for bf16 all but what lies 2^-30 below the largest.
  u32x4 qf[D / 32];
  float c;
  {
    const uint64_t o = (uint64_t)pt.b * a.q.ts + (uint64_t)hq * a.q.hs + g * (D / 4);
    f32x4 x[D / 16];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      x[i] = load4(a.q.p, a.q.dtype, o + 4 * i);
      top = fmaxf(fmaxf(fmaxf(top, fabsf(x[i].x)), fmaxf(fabsf(x[i].y), fabsf(x[i].z))), fabsf(x[i].w));
    }
    top = max_xor16(max_xor32(top));
    const int e = top > 0.f ? ilogbf(fminf(top, 3.0e38f)) - 14 : 0;
    const float sign = a.o.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = ldexpf(x[2 * i + (j >> 2)][j & 3], -e) * sign;
      qf[i] = u32x4{pack_f16(y[0], y[1]), pack_f16(y[2], y[3]), pack_f16(y[4], y[5]), pack_f16(y[6], y[7])};
    }
    // above zero and finite: a masked score times c stays -inf, a score of zero zero
    c = fminf(fmaxf(ldexpf(fabsf(a.o.scale) * 1.44269504088896340736f, e), 0x1p-126f), kLargest);
  }

  // m: the largest score so far. A weight is 2^((s - m) c + kLift), the difference first: s c - m c would be off by the
  // rounding of m c, which for scores of 2^28 and more is more than the range of the weights' 16 bits.
  f32x4 acc[NT] = {};
  float m = -INFINITY, l = 0.f;
  const int begin = sp.c0 + (int)(pt.part * pt.size), end = sp.c0 + (int)min((uint32_t)sp.chunks, (pt.part + 1) * pt.size);
  const int cpp = 1 << (a.kv.page_shift - 6);
  // this wave's chunks: begin + wave, + kWaves, ..; lane i has the page of the i-th of the next 64
  auto page_of = [&](int chunk) -> int {
    if (chunk >= end) return -1;
    const int p = a.table[(uint64_t)pt.b * a.max_pages + (uint32_t)(chunk >> (a.kv.page_shift - 6))];
    if (p >= 0 && (uint32_t)p < a.kv.n_pages) return p;
    note_error(a.err, kErrPage);
    return -1;
  };
  auto address = [&](int page, int chunk) { return a.kv.at(page < 0 ? 0 : page, hk, chunk & (cpp - 1)); };
  Chunk<FMT, D> ch;
  int pages = -1, page = -1;
  for (int i = 0, cidx = begin + wave; cidx < end; ++i, cidx += kWaves) {
    if ((i & 63) == 0) {
      pages = page_of(cidx + kWaves * lane);
      page = __builtin_amdgcn_readlane(pages, 0);
      if (kAhead) ch.load_k(address(page, cidx), lane);
    }
    const bool there = page >= 0;
    const uint8_t* chunk = address(page, cidx);
    if (!kAhead) ch.load_k(chunk, lane);
    ch.load_v(chunk, lane, 0);
    if (kAhead) ch.load_v(chunk, lane, 1);
    f32x4 s[4] = {};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) s[t] = mfma16(ch.key(t, j), qf[j], s[t]);
    if (!kAhead) ch.load_v(chunk, lane, 1);
    if ((i & 63) != 63 && cidx + kWaves < end) {
      page = __builtin_amdgcn_readlane(pages, (i + 1) & 63);
      if (kAhead) ch.load_k(address(page, cidx + kWaves), lane);
    }
    const int k0 = cidx << 6;
    if (!there || k0 < sp.first || k0 + 64 > sp.n) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + 16 * t + 4 * g + j;
          if (!there || key < sp.first || key >= sp.n) s[t][j] = -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 16; ++t) top = fmaxf(top, s[t >> 2][t & 3]);
    top = max_xor16(max_xor32(top));
    const float m1 = fmaxf(m, top);
    if (__any(m1 > m)) {
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m1) * c);
      l *= f;
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] *= f;
      m = m1;
    }
    const float base = m == -INFINITY ? 0.f : m;
    u32x4 pf[2];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[t][j] - base, c, kLift));
      const uint32_t w0 = pack_f16(p[0], p[1]), w1 = pack_f16(p[2], p[3]);
      pf[t >> 1][2 * (t & 1)] = w0, pf[t >> 1][2 * (t & 1) + 1] = w1;
      l = add_f16(w1, add_f16(w0, l));
    }
#pragma unroll
    for (int G = 0; G < 2; ++G)
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        u32x4 lo, hi;
        ch.value(G, b, lo, hi);
        acc[2 * b] = mfma16(lo, pf[G], acc[2 * b]);
        acc[2 * b + 1] = mfma16(hi, pf[G], acc[2 * b + 1]);
      }
  }
  l = add_xor16(add_xor32(l));

  // The waves' results are joined in pairs: (0, 2) and (1, 3), then (0, 1). acc: element 16 t + 4 g + j of head n.
#pragma unroll
  for (int w = kWaves / 2; w >= 1; w /= 2) {
    if (wave >= w && wave < 2 * w) {
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(&sums[wave - w][n * D + 16 * t + 4 * g]) = acc[t];
      if (g == 0) stats[wave - w][n][0] = m, stats[wave - w][n][1] = l;
    }
    __syncthreads();
    if (wave < w) {
      const float m2 = stats[wave][n][0], l2 = stats[wave][n][1], m1 = fmaxf(m, m2);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m1) * c);
      const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m2 - m1) * c);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t] = acc[t] * f + *reinterpret_cast<const f32x4*>(&sums[wave][n * D + 16 * t + 4 * g]) * f2;
      l = l * f + l2 * f2, m = m1;
    }
    __syncthreads();
  }
  if (wave > 0 || (uint32_t)n >= heads) return;
  // What the weights are relative to, for sinks and other parts; its rounding is one of the score.
  if (m > -INFINITY) m = fminf(fmaxf(m * c, -kLargest), kLargest) - kLift;
  if (pt.parts > 1) {
    const uint64_t unit = ((uint64_t)(pt.slot + pt.part) * gridDim.y + blockIdx.y) * 16 + n;
    float* dst = a.part + unit * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(dst + 16 * t + 4 * g) = acc[t];
    float* st = a.part + (uint64_t)a.parts * gridDim.y * 16 * D + unit * 2;
    if (g == 0) st[0] = m, st[1] = l;
    return;
  }
  if (a.o.sinks) {
    const float sink = sink_of(a.o.sinks, hq), m1 = fmaxf(m, sink);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m1);
    l = l * f + (sink == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - m1));
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] *= f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    store4(a.out.p, a.out.dtype, (uint64_t)pt.b * a.out.ts + (uint64_t)hq * a.out.hs + 16 * t + 4 * g, acc[t] * inv);
}

// Joins the parts of split sequence blockIdx.x for one query head: first all parts' weights, then the weighted
// sums, D/4 lanes to a part and kJoin / (D/4) parts at a time, many loads in flight (a running maximum would
// make each part wait for the one before: 36 us for 391 parts of 256, instead of 7 us for 224).
constexpr int kJoin = 256;
template <int D>
__global__ __launch_bounds__(kJoin) void k_attn_join(DecodeArgs a) {
  constexpr int L = D / 4, G = kJoin / L;
  __shared__ __attribute__((aligned(16))) float sums[G * D];
  __shared__ float weight[kPartUnits], wave_m[kJoin / 64], wave_l[kJoin / 64];
  Part pt;
  if (!find_part(a, blockIdx.x, true, pt)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t h = blockIdx.y, hk = h / a.heads, in = h % a.heads, units = a.kv.n_heads * a.head_tiles;
  const uint64_t unit0 = ((uint64_t)pt.slot * units + hk * a.head_tiles + in / 16) * 16 + in % 16;
  const float* stat = a.part + (uint64_t)a.parts * units * 16 * D;
  float m[kPartUnits / kJoin], l = 0.f, top = -INFINITY;
#pragma unroll
  for (int i = 0; i < (int)(kPartUnits / kJoin); ++i) {
    const uint32_t p = tid + i * kJoin;
    m[i] = p < pt.parts ? stat[2 * (unit0 + (uint64_t)p * units * 16)] : -INFINITY;
    top = fmaxf(top, m[i]);
  }
  top = wave_max(top);
  if (lane == 0) wave_m[wave] = top;
  __syncthreads();
  const float sink = sink_of(a.o.sinks, h);
  float base = sink;
  for (int w = 0; w < kJoin / 64; ++w) base = fmaxf(base, wave_m[w]);
  if (base == -INFINITY) base = 0.f;
#pragma unroll
  for (int i = 0; i < (int)(kPartUnits / kJoin); ++i) {
    const uint32_t p = tid + i * kJoin;
    if (p >= pt.parts) break;
    weight[p] = __builtin_amdgcn_exp2f(m[i] - base);
    l += stat[2 * (unit0 + (uint64_t)p * units * 16) + 1] * weight[p];
  }
  l = wave_sum(l);
  if (lane == 0) wave_l[wave] = l;
  __syncthreads();
  f32x4 acc = {0, 0, 0, 0};
  const float* src = a.part + unit0 * D + 4 * (tid % L);
#pragma unroll 8
  for (uint32_t p = tid / L; p < pt.parts; p += G)
    acc += *reinterpret_cast<const f32x4*>(src + (uint64_t)p * units * 16 * D) * weight[p];
  *reinterpret_cast<f32x4*>(&sums[4 * tid]) = acc;
  __syncthreads();
  if (tid >= D) return;
  float s = 0.f;
  l = __builtin_amdgcn_exp2f(sink - base);
  for (int g = 0; g < G; ++g) s += sums[g * D + tid];
  for (int x = 0; x < kJoin / 64; ++x) l += wave_l[x];
  const float v = l == 0.f ? 0.f : s / l;
  uint16_t* dst = static_cast<uint16_t*>(a.out.p) + (uint64_t)pt.b * a.out.ts + (uint64_t)h * a.out.hs + tid;
  *dst = (uint16_t)(a.out.dtype == MR_F16 ? pack_f16(v, 0.f) : pack_bf16(v, 0.f));
}

using DecodeKernel = void (*)(DecodeArgs);
// The kernel of a format and width, and how many of its workgroups a CU holds.
template <int FMT, int D>
DecodeKernel pick(int& per_cu) {
  static const int n = [] {
    int v = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, k_attn_decode<FMT, D>, 64 * kWaves, 0) == hipSuccess && v > 0 ? v : 1;
  }();
  per_cu = n;
  return k_attn_decode<FMT, D>;
}
template <int FMT>
DecodeKernel pick(uint32_t D, int& per_cu) {
  return D == 64 ? pick<FMT, 64>(per_cu) : D == 128 ? pick<FMT, 128>(per_cu) : pick<FMT, 256>(per_cu);
}

}  // namespace

uint64_t attn_decode_scratch_bytes() { return (uint64_t)kPartUnits * 16 * (256 + 2) * sizeof(float); }

hipError_t launch_attn_decode(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& q, uint32_t B,
                              const int32_t* len, const int32_t* table, uint32_t max_pages, const AttnOpts& o,
                              const Heads& out, uint32_t* err, float* scratch, int n_cu) {
  DecodeArgs a{kv, q, out, len, table, max_pages, B, q.n / kv.n_heads, 0, 0, o, err, scratch};
  a.head_tiles = (a.heads + 15) / 16;
  const uint32_t units = kv.n_heads * a.head_tiles;
  int per_cu = 1;
  const DecodeKernel kernel = format == MR_KV_F16      ? pick<MR_KV_F16>(D, per_cu)
                              : format == MR_KV_MXINT8 ? pick<MR_KV_MXINT8>(D, per_cu)
                                                       : pick<MR_KV_MXFP4>(D, per_cu);
  const uint64_t cap = (uint64_t)max_pages << (kv.page_shift - 6);
  const uint64_t chunks = o.window ? std::min<uint64_t>(cap, (o.window + 62ull) / 64 + 1) : cap;  // of a sequence at most
  const uint32_t room = std::min<uint32_t>(kPartUnits, per_cu * n_cu);
  // the parts are counted in 32 bits
  const bool whole = chunks <= whole_chunks(D) || B > kSplitSeqs || B * chunks >= 1ull << 31;
  a.parts = whole ? 1 : std::max<uint32_t>(1, room / units);
  hipError_t e;
  {
    ProfScope ps(K, "attn_decode");
    hipLaunchKernelGGL(kernel, dim3(a.parts > 1 ? part_limit(a.parts, B) : B, units), dim3(64 * kWaves), 0, K.s, a);
    e = hipGetLastError();
    if (e != hipSuccess || a.parts == 1) return e;
  }
  ProfScope ps(K, "attn_join");
  const dim3 j(std::min(B, a.parts), q.n), blk(kJoin);
  if (D == 64) hipLaunchKernelGGL((k_attn_join<64>), j, blk, 0, K.s, a);
  if (D == 128) hipLaunchKernelGGL((k_attn_join<128>), j, blk, 0, K.s, a);
  if (D == 256) hipLaunchKernelGGL((k_attn_join<256>), j, blk, 0, K.s, a);
  return hipGetLastError();
}

}  // namespace mr
