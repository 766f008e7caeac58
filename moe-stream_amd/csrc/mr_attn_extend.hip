// mr_attn_extend.hip -- attention of the new tokens of many sequences over the paged cache.
//
// One pass over the keys with each row's running maximum and sum, as in mr_attn_decode.hip. A sequence's rows are its
// new tokens times the query heads that share a key head, token by token; a tile is some of them in a row, whatever
// the number of heads.
#include "mr_kv_operand.h"
#include "mr_state_device.h"

namespace mr {

namespace {

constexpr int kWaves = 4;
constexpr uint32_t kSplitSeqs = 1024;      // with more sequences none is split: each workgroup looks through them all
constexpr uint32_t kScratchRows = 65536;   // rows of partial results
constexpr uint32_t kMinPart = kWaves;      // steps of a part at least
constexpr int kFewRows = 16;               // up to so many rows are a wave's of its own chunks in every kernel

struct ExtendArgs {
  KvPages kv;
  Heads q, out;
  const int32_t *cu, *len, *table;
  uint32_t max_pages, n_seqs;
  int nq;
  Divisor group;       // query heads of a key head
  int bits;            // log2 of a tile's rows
  float slack;         // of k_attn_extend_wide, in powers of two
  uint32_t parts;      // parts that the CUs hold at once; 1: none is split
  AttnOpts o;
  uint32_t* err;
  float* part;         // [slot][key head][row][D] sums, then [slot][..][row][2] maximum and sum
};

// A sequence's rows and keys, in chunks.
struct Span {
  int q0, n, len;       // first row (token) of the call, new tokens, cached tokens
  int c0, chunks;       // chunks that some row sees
  uint32_t tiles, steps;  // steps of a workgroup through the chunks
};
__device__ __forceinline__ int first_seen(const ExtendArgs& a, int pos) {
  return a.o.window && pos >= 0 && (uint32_t)pos >= a.o.window ? pos - (int)a.o.window + 1 : 0;
}
__device__ __forceinline__ Span span_of(const ExtendArgs& a, uint32_t b) {
  Span s;
  int q1;
  rows_of(a.cu, a.nq, b, s.q0, q1);
  s.n = q1 - s.q0;
  const int64_t cap = (int64_t)a.max_pages << a.kv.page_shift;
  s.len = (int)min(max((int64_t)a.len[b], (int64_t)0), cap);
  s.c0 = first_seen(a, s.len - s.n) >> 6;
  s.chunks = s.n && s.len ? ((s.len - 1) >> 6) + 1 - s.c0 : 0;
  const uint32_t rows = (uint32_t)s.n * a.group.d;
  s.tiles = (rows + (1u << a.bits) - 1) >> a.bits;
  s.steps = a.bits > 5 && rows <= kFewRows ? (uint32_t)(s.chunks + kWaves - 1) / kWaves : (uint32_t)s.chunks;
  return s;
}

// A workgroup's unit: a tile of a sequence, a part of its keys and a key head, heads in turn: workgroups go to the 8 XCDs in turn, so
// that the tiles of a head, a part after the other, are on few of them and find the keys that they share in one L2 (a prompt's part
// among 32 tokens, 8 heads: 208 us with units in turn, 195 so). split_only: tile blockIdx.x of the sequences of several parts and key
// head blockIdx.y; the part is then 0. slot: parts of split sequences in front of the tile's.
struct Unit {
  uint32_t b, hk, tile, part, parts, slot;
  Span sp;
};
__device__ __forceinline__ bool find_unit(const ExtendArgs& a, bool split_only, Unit& r) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t i = split_only ? blockIdx.x : blockIdx.x / a.kv.n_heads;
  r.hk = split_only ? blockIdx.y : blockIdx.x - i * a.kv.n_heads;
  if (a.parts == 1) {
    if (split_only) return false;
    r.b = find_seq(a.cu, a.n_seqs, a.nq, a.group.d, a.bits, i);
    r.sp = span_of(a, r.b);
    const int64_t tile = (int64_t)i - first_tile(a.cu, a.nq, r.b, a.group.d, a.bits);
    r.tile = (uint32_t)tile, r.part = 0, r.parts = 1, r.slot = 0;
    return tile >= 0 && tile < (int64_t)r.sp.tiles;
  }
  Span s = lane < a.n_seqs ? span_of(a, lane) : Span{};
  // f(tiles, steps) of every sequence, summed
  auto sum_of = [&](auto f) {
    uint32_t v = lane < a.n_seqs ? f(s.tiles, s.steps) : 0;
    for (uint32_t b0 = 64; b0 < a.n_seqs; b0 += 64)
      if (b0 + lane < a.n_seqs) {
        const Span x = span_of(a, b0 + lane);
        v += f(x.tiles, x.steps);
      }
    return wave_total(v);
  };
  // The smallest size, in steps of an eighth, at which the CUs hold all parts at once.
  const uint32_t all = sum_of([](uint32_t t, uint32_t c) { return t * c; }), tiles = sum_of([](uint32_t t, uint32_t) { return t; });
  const uint32_t most = max(a.parts, tiles + a.parts / 2);
  uint32_t size = max(kMinPart, (all + a.parts - 1) / a.parts);
  while (size < all && sum_of([&](uint32_t t, uint32_t c) { return t * max(1u, (c + size - 1) / size); }) > most) size += (size + 7) / 8;
  uint32_t before = 0, slots = 0;
  for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += 64) {
    if (b0) s = b0 + lane < a.n_seqs ? span_of(a, b0 + lane) : Span{};
    const uint32_t parts = max(1u, (s.steps + size - 1) / size), n = s.tiles * parts;
    const uint32_t split = parts > 1 ? n : 0, count = split_only ? (parts > 1 ? s.tiles : 0) : n;
    const uint32_t sum = wave_prefix(count), ssum = wave_prefix(split);
    const uint64_t past = __ballot(before + sum > i);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      r.b = b0 + l;
      r.parts = __builtin_amdgcn_readlane(parts, l);
      const uint32_t in = i - before - __builtin_amdgcn_readlane(sum - count, l);
      const uint32_t tiles = (uint32_t)__builtin_amdgcn_readlane(s.tiles, l);
      r.part = split_only ? 0 : in / tiles;  // the tiles of a part one after the other
      r.tile = in - r.part * tiles;
      r.slot = slots + __builtin_amdgcn_readlane(ssum - split, l) + r.tile * r.parts;
      r.sp = Span{__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.len, l),
                  __builtin_amdgcn_readlane(s.c0, l), __builtin_amdgcn_readlane(s.chunks, l),
                  (uint32_t)__builtin_amdgcn_readlane(s.tiles, l), 0};
      // Offsets in order leave room: parts beyond the first are half of a.parts at most, or all of them. Overlapping ones may not: sums
      // of their tiles and parts may pass 32 bits even, so that the slot is compared by itself.
      return r.parts == 1 || (r.slot < a.parts && r.parts <= a.parts - r.slot);
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(ssum, 63);
  }
  return false;
}

// What a tile's rows see of the part's keys.
struct Reach {
  int r0, rows;          // first row and rows
  int pos0, pos1;        // positions of the first and last row
  int begin, end;        // chunks
};
__device__ __forceinline__ Reach reach_of(const ExtendArgs& a, const Unit& u) {
  Reach t;
  t.r0 = (int)(u.tile << a.bits);
  t.rows = min(1 << a.bits, (int)((uint32_t)u.sp.n * a.group.d) - t.r0);
  const int ahead = u.sp.len - u.sp.n;
  t.pos0 = ahead + (int)a.group.of(t.r0), t.pos1 = ahead + (int)a.group.of(t.r0 + t.rows - 1);
  const int c0 = first_seen(a, t.pos0) >> 6, chunks = t.pos1 < 0 ? 0 : (t.pos1 >> 6) + 1 - c0;
  const int size = (chunks + (int)u.parts - 1) / (int)u.parts;
  t.begin = c0 + min((int)u.part * size, chunks), t.end = c0 + min(((int)u.part + 1) * size, chunks);
  return t;
}

// Reports offsets and lengths out of range; by every thread of one workgroup.
__device__ __forceinline__ void check_entries(const ExtendArgs& a) {
  check_offsets(a.cu, a.n_seqs, a.nq, a.err, kErrOffset);
  for (uint32_t s = threadIdx.x; s < a.n_seqs; s += blockDim.x)
    if (a.len[s] < 0 || (int64_t)a.len[s] > (int64_t)a.max_pages << a.kv.page_shift) note_error(a.err, kErrLength);
}

template <int NT, int FMT, int D>
constexpr int kPerSimd = NT * D >= 256 ? 1 : 2;

// A tile of NT times 16 rows, the columns of the matrix products S = K Q^T and O = V^T P. A wave takes chunks of 64 tokens by
// itself, operands straight from the pages, and the waves' results are joined at the end. The cache's bytes bound it while a tile has
// 16 rows: two new tokens of 32 sequences behind up to 24000, 32 heads on 4 of 128: MXFP4 52 us (4.2 TB/s), F16 154 us (5.3 TB/s);
// turning codes into operands for more rows than that is then most of it.
template <int NT, int FMT, int D>
__device__ __forceinline__ void attend_few(const ExtendArgs& a, const Unit& u, const Reach& t, float (*sums)[16 * D], float (*stats)[16][2]) {
  constexpr int ND = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t hk = u.hk;

  // This lane's row of each 16: its place in q and out, and which keys it sees. The query as f16 times a power of
  // two, its largest element in [2^14, 2^15): exact for f16, for bf16 all but what lies 2^-30 below the largest.
  u32x4 qf[NT][D / 32];
  float c[NT];
  int pos[NT];
  auto place = [&](int j, uint64_t& row, uint32_t& head) {
    const uint32_t r = (uint32_t)(t.r0 + min(16 * j + n, t.rows - 1)), i = a.group.of(r);
    row = (uint64_t)(u.sp.q0 + (int)i), head = hk * a.group.d + (r - i * a.group.d);
    return u.sp.len - u.sp.n + (int)i;
  };
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    uint64_t row;
    uint32_t head;
    pos[j] = place(j, row, head);
    const uint64_t o = row * a.q.ts + (uint64_t)head * a.q.hs + g * (D / 4);
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
      for (int k = 0; k < 8; ++k) y[k] = ldexpf(x[2 * i + (k >> 2)][k & 3], -e) * sign;
      qf[j][i] = u32x4{pack_f16(y[0], y[1]), pack_f16(y[2], y[3]), pack_f16(y[4], y[5]), pack_f16(y[6], y[7])};
    }
    // above zero and finite: a masked score times c stays -inf, a score of zero zero
    c[j] = fminf(fmaxf(ldexpf(fabsf(a.o.scale) * 1.44269504088896340736f, e), 0x1p-126f), kLargest);
  }

  f32x4 acc[NT][ND] = {};
  float m[NT], l[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) m[j] = -INFINITY, l[j] = 0.f;
  const int cpp = 1 << (a.kv.page_shift - 6);
  auto page_of = [&](int chunk) -> int {
    if (chunk >= t.end) return -1;
    const int p = a.table[(uint64_t)u.b * a.max_pages + (uint32_t)(chunk >> (a.kv.page_shift - 6))];
    if (p >= 0 && (uint32_t)p < a.kv.n_pages) return p;
    note_error(a.err, kErrPage);
    return -1;
  };
  Chunk<FMT, D> ch;
  int pages = -1;
  for (int i = 0, cidx = t.begin + wave; cidx < t.end; ++i, cidx += kWaves) {
    if ((i & 63) == 0) pages = page_of(cidx + kWaves * lane);
    const int page = __builtin_amdgcn_readlane(pages, i & 63);
    const bool there = page >= 0;
    const uint8_t* chunk = a.kv.at(there ? page : 0, hk, cidx & (cpp - 1));
    ch.load_k(chunk, lane);
    ch.load_v(chunk, lane, 0), ch.load_v(chunk, lane, 1);
    f32x4 s[NT][4] = {};
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const u32x4 k = ch.key(x, i);
#pragma unroll
        for (int j = 0; j < NT; ++j) s[j][x] = mfma16(k, qf[j][i], s[j][x]);
      }
    const int k0 = cidx << 6;
    // some row does not see some key
    const bool edge = !there || k0 + 63 > t.pos0 || k0 < first_seen(a, t.pos1);
    u32x4 pf[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (edge) {
        const int from = first_seen(a, pos[j]);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int key = k0 + 16 * x + 4 * g + y;
            if (!there || key < from || key > pos[j]) s[j][x][y] = -INFINITY;
          }
      }
      float top = s[j][0][0];
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, s[j][x >> 2][x & 3]);
      top = max_xor16(max_xor32(top));
      const float m1 = fmaxf(m[j], top);
      if (__any(m1 > m[j])) {
        const float f = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[j] - m1) * c[j]);
        l[j] *= f;
#pragma unroll
        for (int x = 0; x < ND; ++x) acc[j][x] *= f;
        m[j] = m1;
      }
      const float base = m[j] == -INFINITY ? 0.f : m[j];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float p[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) p[y] = __builtin_amdgcn_exp2f(fmaf(s[j][x][y] - base, c[j], kLift));
        const uint32_t w0 = pack_f16(p[0], p[1]), w1 = pack_f16(p[2], p[3]);
        pf[j][x >> 1][2 * (x & 1)] = w0, pf[j][x >> 1][2 * (x & 1) + 1] = w1;
        l[j] = add_f16(w1, add_f16(w0, l[j]));
      }
    }
#pragma unroll
    for (int G = 0; G < 2; ++G)
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        u32x4 lo, hi;
        ch.value(G, b, lo, hi);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][2 * b] = mfma16(lo, pf[j][G], acc[j][2 * b]);
          acc[j][2 * b + 1] = mfma16(hi, pf[j][G], acc[j][2 * b + 1]);
        }
      }
  }

  // The waves' results are joined in pairs, 16 rows after the other: (0, 2) and (1, 3), then (0, 1).
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    l[j] = add_xor16(add_xor32(l[j]));
#pragma unroll
    for (int w = kWaves / 2; w >= 1; w /= 2) {
      if (wave >= w && wave < 2 * w) {
#pragma unroll
        for (int x = 0; x < ND; ++x) *reinterpret_cast<f32x4*>(&sums[wave - w][n * D + 16 * x + 4 * g]) = acc[j][x];
        if (g == 0) stats[wave - w][n][0] = m[j], stats[wave - w][n][1] = l[j];
      }
      __syncthreads();
      if (wave < w) {
        const float m2 = stats[wave][n][0], l2 = stats[wave][n][1], m1 = fmaxf(m[j], m2);
        const float f = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[j] - m1) * c[j]);
        const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m2 - m1) * c[j]);
#pragma unroll
        for (int x = 0; x < ND; ++x)
          acc[j][x] = acc[j][x] * f + *reinterpret_cast<const f32x4*>(&sums[wave][n * D + 16 * x + 4 * g]) * f2;
        l[j] = l[j] * f + l2 * f2, m[j] = m1;
      }
      __syncthreads();
    }
  }
  if (wave > 0) return;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (16 * j + n >= t.rows) continue;
    // What the weights are relative to, for sinks and other parts; its rounding is one of the score.
    if (m[j] > -INFINITY) m[j] = fminf(fmaxf(m[j] * c[j], -kLargest), kLargest) - kLift;
    if (u.parts > 1) {
      const uint64_t unit = (((uint64_t)(u.slot + u.part) * a.kv.n_heads + hk) << a.bits) + 16 * j + n;
      float* dst = a.part + unit * D;
#pragma unroll
      for (int x = 0; x < ND; ++x) *reinterpret_cast<f32x4*>(dst + 16 * x + 4 * g) = acc[j][x];
      float* st = a.part + (uint64_t)kScratchRows * D + unit * 2;
      if (g == 0) st[0] = m[j], st[1] = l[j];
      continue;
    }
    uint64_t row;
    uint32_t head;
    place(j, row, head);
    float f = 1.f;
    const float sink = sink_of(a.o.sinks, head);
    if (a.o.sinks) {
      const float m1 = fmaxf(m[j], sink);
      f = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[j] - m1);
      l[j] = l[j] * f + (sink == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - m1));
    }
    const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
#pragma unroll
    for (int x = 0; x < ND; ++x)
      store4(a.out.p, a.out.dtype, row * a.out.ts + (uint64_t)head * a.out.hs + 16 * x + 4 * g, acc[j][x] * f * inv);
  }
}

template <int NT, int FMT, int D>
__global__ __launch_bounds__(64 * kWaves, (kPerSimd<NT, FMT, D>)) void k_attn_extend(ExtendArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[kWaves / 2][16 * D];
  __shared__ float stats[kWaves / 2][16][2];
  if (blockIdx.x == 0) check_entries(a);
  Unit u;
  if (find_unit(a, false, u)) attend_few<NT, FMT, D>(a, u, reach_of(a, u), sums, stats);
}

// ---- many rows ------------------------------------------------------------------------------
// A tile of 128 rows, 32 to a wave, all waves at the same chunk of 64 tokens. Its codes are turned into operands once, by the
// four waves together, and lie in LDS as the pages have them, so that writes and reads are whole rows of 16-byte pieces.
// Both products are 32x32x16 matrix instructions, keys (then the values' elements) down and rows across: a lane has the scores
// of one row. Of each 32 keys the result's row 16 c + 8 x + 4 h + r stands for key 16 x + 8 c + 4 h + r: lane half h then holds,
// 8 numbers after the other, what the second product's right operand wants for the values of lane group 2 c + h.
//
// Bounds: heads of 256, matrix and vector instructions of the one wave of a SIMD, which hardly overlap (2048 tokens behind 30001,
// 16 heads on 2, MXINT8: 1170 us, 890 TFLOP/s); heads of 128, loads and the last round of units (four parts of prompts, 32 heads
// on 4, F16: 167 us, 760 TFLOP/s); heads of 64, vector instructions (a part of 1000 tokens and 32 single ones, 64 heads on 8,
// MXINT8: 174 us, 620 TFLOP/s).
// Weights go up to 2^15, and the maximum is followed when it has moved by 2^slack: the largest weight lies between 2^(15 - slack) and
// 2^15, and ones down to 2^(slack - 29) of it keep all bits of f16. Where sequences have up to 32 rows, the slack is one, and the bits are
// those of attend_few: 3 new tokens of 32 sequences, 32 heads on 4 of 128, MXFP4 76.5 us with four and 79 us with one
// (16 on 2 of 256, MXINT8: 123 and 139 us). For more rows it is four: 5 new tokens of the same 91.5 and 95 us, four prompts' parts 175 and 181 us.
constexpr float kTopWeight = 15.f, kSlackFew = 1.f, kSlackMany = 4.f;

// A wave's quarter of a chunk on its way from the pages to LDS.
template <int FMT, int D>
struct Quarter {
  static constexpr int NK = D / 32, NV = D / 64;   // operands of keys, pairs of operands of values
  static constexpr int KW = D * FMT / 128, VW = FMT / 2;  // words of a lane's keys (16 of them), of a pair's values
  uint32_t k[KW], v[NV][VW], ks[FMT == MR_KV_F16 ? 1 : D == 256 ? 2 : 1];
  u32x2 vs[NV];

  // Load i of the keys 16 wave + m: 16 bytes of codes (or 8), then the scales.
  static constexpr int kKeyLoads = (KW + 3) / 4 + 1, kValueLoads = NV;
  __device__ __forceinline__ void load_keys(int i, const uint8_t* p, int wave, int lane) {
    using L = KvLayout<FMT, D>;
    const int m = lane & 15, g = lane >> 4;
    const int kb = wave * KW * 4;  // byte of a lane's keys: pieces of 16 bytes are 1 KB apart
    p += (uint32_t)((kb >> 4) * 1024 + (kb & 15));
    if (i + 1 < kKeyLoads) {
      if constexpr (KW == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p + lane * 16);
        k[0] = x.x, k[1] = x.y;
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p + 1024 * i + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[4 * i + j] = x[j];
      }
    } else if (i < kKeyLoads) {
      p -= (uint32_t)((kb >> 4) * 1024 + (kb & 15));
#pragma unroll
      for (int j = 0; j < (D == 256 ? 2 : 1); ++j) {
        const int blk = D == 64 ? g >> 1 : D == 128 ? g : 2 * g + j;
        ks[j] = *reinterpret_cast<const uint32_t*>(p + L::kKs + (blk * 16 + m) * 4);
      }
    }
  }
  // Load i of the pairs of values NV * wave and on.
  __device__ __forceinline__ void load_values(int i, const uint8_t* p, int wave, int lane) {
    using L = KvLayout<FMT, D>;
    if (i >= NV) return;
    const int vb = (wave * NV + i) * VW * 4;
    const uint8_t* at = p + L::kV + (vb >> 4) * 1024 + (vb & 15) + lane * 16;
    if constexpr (VW == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(at);
      v[i][0] = x.x, v[i][1] = x.y;
    } else {
      const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
      for (int j = 0; j < VW; ++j) v[i][j] = x[j & 3];
    }
    vs[i] = *reinterpret_cast<const u32x2*>(p + L::kVs + (lane >> 4) * (D / 2) + (wave * NV + i) * 8);
  }
  // Item i of the quarter as operands to the chunk's keys and values in LDS (a lane's addresses): first the keys', then the pairs
  // of values.
  static constexpr int kItems = NK + NV;
  __device__ __forceinline__ void store(int i, uint32_t keys, uint32_t values, int wave) const {
    if (i < NK) {
      u32x4 x;
      const uint32_t s = ks[D == 256 ? i >> 2 : 0];
      if constexpr (FMT == MR_KV_MXFP4) {
        const uint32_t e = exp_bits_of(s, wave), c = k[i];
        x = u32x4{fp4_pair<0>(c, e), fp4_pair<1>(c, e), fp4_pair<2>(c, e), fp4_pair<3>(c, e)};
      } else if constexpr (FMT == MR_KV_MXINT8) {
        const uint32_t b = s >> (8 * wave) & 0xFFu;
        const f16x2 e = __builtin_bit_cast(f16x2, b << 8 | b << 24);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __builtin_bit_cast(uint32_t, int8_pair(k[2 * i + (j >> 1)], j & 1) * e);
      }
      put16(keys + (wave * NK + i) * 1024, x);
    } else if (i < kItems) {
      const int j = i - NK;
      u32x4 lo, hi;
      value_pair<FMT>(v[j], vs[j].x, vs[j].y, lo, hi);
      put16(values + (wave * NV + j) * 2048, lo), put16(values + (wave * NV + j) * 2048 + 1024, hi);
    }
  }
  static __device__ __forceinline__ void put16(uint32_t at, u32x4 x) { *(__attribute__((address_space(3))) u32x4*)(uintptr_t)at = x; }
  static __device__ __forceinline__ uint32_t exp_bits_of(uint32_t s, int wave) { return s >> (8 * wave) << 23; }
};

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int FMT, int D>
constexpr int kWidePerSimd = D == 256 ? 1 : D == 128 ? 2 : FMT == MR_KV_MXINT8 ? 3 : 4;

// KH: how many of a chunk's halves of 32 keys a wave has: both, or, in tiles of 64 rows, two waves one each of the same rows, whose
// results are joined at the end.
template <int FMT, int D, int KH>
__global__ __launch_bounds__(256, (kWidePerSimd<FMT, D>)) void k_attn_extend_wide(ExtendArgs a) {
  constexpr int ND = D / 32, NI = D / 16, kTile = 64 * D * 2;  // bytes of a chunk's keys as operands
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][kTile];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  if (blockIdx.x == 0) check_entries(a);
  Unit u;
  if (!find_unit(a, false, u)) return;
  const uint32_t hk = u.hk;
  const Reach t = reach_of(a, u);
  if (__builtin_expect(t.rows <= kFewRows, 0)) {
    // single tokens beside a prompt's part: of 32, 194 us as tiles like the others, 174 us so; expected to be the rarer, which
    // leaves the others' code where it is (a part of 2048 tokens, heads of 256: 1175 us, else 1212 us)
    attend_few<1, FMT, D>(a, u, t, reinterpret_cast<float(*)[16 * D]>(&lds[0][0][0]), reinterpret_cast<float(*)[16][2]>(&lds[1][0][0]));
    return;
  }
  const int block = KH == 2 ? wave : wave & 1, first_half = KH == 2 ? 0 : wave >> 1;
  const int mine = 32 * block + n;  // this lane's row of the tile

  auto place = [&](int mine, uint64_t& row, uint32_t& head) {
    const uint32_t r = (uint32_t)(t.r0 + min(mine, t.rows - 1)), i = a.group.of(r);
    row = (uint64_t)(u.sp.q0 + (int)i), head = hk * a.group.d + (r - i * a.group.d);
    return u.sp.len - u.sp.n + (int)i;
  };
  uint64_t row;
  uint32_t head;
  const int pos = place(mine, row, head), from = first_seen(a, pos);
  // of the wave's rows: the first one's position, and the last one's first key
  const int wave_pos0 = __builtin_amdgcn_readfirstlane(pos), wave_pos1 = __builtin_amdgcn_readlane(pos, 31);
  const int wave_last_first = first_seen(a, wave_pos1);

  // The query as f16 times a power of two, its largest element in [2^14, 2^15).
  u32x4 qf[NI];
  float c;
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q.p) + row * a.q.ts + (uint64_t)head * a.q.hs;
    const bool bf = a.q.dtype == MR_BF16;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      // step (e, gp) of the sums has the elements 8 e .. of the quarters 2 gp and 2 gp + 1
      qf[i] = *reinterpret_cast<const u32x4*>(qp + (2 * (i & 1) + half) * (D / 4) + 8 * (i >> 1));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 x = bf ? unpack_bf16(qf[i][j]) : unpack_f16(qf[i][j]);
        top = fmaxf(fmaxf(top, fabsf(x.x)), fabsf(x.y));
      }
    }
    top = max_xor32(top);
    const int e = top > 0.f ? ilogbf(fminf(top, 3.0e38f)) - 14 : 0;
    const float sign = a.o.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 x = bf ? unpack_bf16(qf[i][j]) : unpack_f16(qf[i][j]);
        qf[i][j] = pack_f16(ldexpf(x.x, -e) * sign, ldexpf(x.y, -e) * sign);
      }
    c = fminf(fmaxf(ldexpf(fabsf(a.o.scale) * 1.44269504088896340736f, e), 0x1p-126f), kLargest);
  }

  const int cpp = 1 << (a.kv.page_shift - 6);
  auto page_of = [&](int chunk) -> int {
    if (chunk >= t.end) return -1;
    const int p = a.table[(uint64_t)u.b * a.max_pages + (uint32_t)(chunk >> (a.kv.page_shift - 6))];
    if (p >= 0 && (uint32_t)p < a.kv.n_pages) return p;
    note_error(a.err, kErrPage);
    return -1;
  };
  // lane i has the page of the i-th of 64 chunks
  int pages = -1;
  auto next_page = [&](int i) {
    if ((i & 63) == 0) pages = page_of(t.begin + i + lane);
    return __builtin_amdgcn_readlane(pages, i & 63);
  };
  Quarter<FMT, D> quarter;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&lds[0][0][0];
  const uint64_t page_bytes = ((uint64_t)a.kv.n_heads << (a.kv.page_shift - 6)) * a.kv.chunk;
  const uint8_t* head_base = a.kv.base + ((uint64_t)hk << (a.kv.page_shift - 6)) * a.kv.chunk;
  auto address = [&](int page, int chunk) { return head_base + (uint32_t)max(page, 0) * page_bytes + (uint32_t)(chunk & (cpp - 1)) * (uint32_t)a.kv.chunk; };
  // Loads 4 i + wave of a chunk of f16, straight to buffer b.
  constexpr int kWhole = 2 * kTile / 4096;
  auto fetch_whole = [&](int i, const uint8_t* p, int b) {
    load_lds16((uint64_t)p, 2 * kTile, (uint32_t)((i * 4 + wave) * 1024 + lane * 16), lds0 + b * 2 * kTile + (i * 4 + wave) * 1024);
  };
  // Item i of what was fetched, to a lane's address in a buffer: the keys' first, then the values'.
  constexpr bool kCodes = FMT != MR_KV_F16;
  constexpr int kKeyItems = kCodes ? Quarter<FMT, D>::NK : 0, kItems = kCodes ? Quarter<FMT, D>::kItems : 0;
  auto put = [&](int i, uint32_t to) {
    if constexpr (FMT != MR_KV_F16) quarter.store(i, to, to + kTile, wave);
  };
  const uint32_t to_at = lds0 + lane * 16;

  f32x16 acc[ND];
#pragma unroll
  for (int x = 0; x < ND; ++x) acc[x] = f32x16{};
  // Weights are 2^(s c - base): relative to ref, the largest score so far or up to the slack below it, base = ref c - lift. With one
  // rounding of s c - base they are right to their own size, however base was rounded; that rounding is the same factor for
  // all of a row's. Where it could be 2^-12 or more, ref is taken from the scores first.
  constexpr float kNear = 0x1p12f;
  const float slack = KH == 2 ? kSlackMany : a.slack, lift = kTopWeight - slack;  // tiles of 128 rows have more than 64 on average
  float ref = 0.f, base = -lift, l = 0.f;
  bool seen = false;
  // addresses of operands: keys 32 T + .., elements of step i; values' elements 32 x + n of 16 keys
  const uint32_t k_at = lds0 + first_half * (D / 16) * 1024 + (uint32_t)(((n >> 3) & 1) * (D / 32) * 1024 + (16 * half + ((n >> 4) << 3 | (n & 7))) * 16);
  const uint32_t v_at = lds0 + kTile + first_half * (D / 16) * 1024 + (uint32_t)((n >> 4) * 1024 + (16 * half + (n & 15)) * 16);
  auto key_part = [&](uint32_t base, int T, int i) {
    return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(base + T * (D / 16) * 1024 + (i >> 1) * 1024 + (i & 1) * 512);
  };
  auto value_part = [&](uint32_t base, int cc, int x) {  // keys 16 cc and on
    return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(base + (cc >> 1) * (D / 16) * 1024 + x * 2048 + (cc & 1) * 512);
  };

  // Codes are fetched two chunks ahead and turned into operands one ahead, between the matrix instructions: keys between those of
  // the scores, values between those of the sums. f16 goes straight to LDS, one ahead.
  int page = -1, page1 = -1, page2 = -1;  // of this chunk and the next two
  if (t.begin < t.end) {
    page = next_page(0);
    const uint8_t* p = address(page, t.begin);
    if (t.begin + 1 < t.end) page1 = next_page(1);
    if constexpr (kCodes) {
      auto load_keys = [&](const uint8_t* p) {
#pragma unroll
        for (int x = 0; x < Quarter<FMT, D>::kKeyLoads; ++x) quarter.load_keys(x, p, wave, lane);
      };
      load_keys(p);
#pragma unroll
      for (int x = 0; x < Quarter<FMT, D>::kValueLoads; ++x) quarter.load_values(x, p, wave, lane);
#pragma unroll
      for (int x = 0; x < kItems; ++x) put(x, to_at);
      p = t.begin + 1 < t.end ? address(page1, t.begin + 1) : p;
      load_keys(p);
#pragma unroll
      for (int x = 0; x < Quarter<FMT, D>::kValueLoads; ++x) quarter.load_values(x, p, wave, lane);
    } else {
#pragma unroll
      for (int x = 0; x < kWhole; ++x) fetch_whole(x, p, 0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
  }
  // Where the next chunks' codes come from. Behind the last chunks too, of some chunk that is there: a wait for one load must
  // know how many others there are behind it.
  const uint8_t *next = nullptr, *far = nullptr;  // of the next chunk, of the one after it
  auto look_ahead = [&](int i, int cidx) {
    const bool more = cidx + 1 < t.end, more2 = cidx + 2 < t.end;
    if (more2) page2 = next_page(i + 2);
    next = address(more ? page1 : page, cidx + more);
    far = address(more2 ? page2 : page, more2 ? cidx + 2 : cidx);
  };
  // Load i of the next chunk of f16.
  auto load = [&](int i, int b) {
    if constexpr (!kCodes)
      if (i < kWhole) fetch_whole(i, next, b ^ 1);
  };
  auto end_step = [&] {
    if (!kCodes) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    page = page1, page1 = page2;
  };
  if (32 * block >= t.rows) {
    // a wave without rows has its quarter of the chunks alone
    for (int i = 0, cidx = t.begin, b = 0; cidx < t.end; ++i, ++cidx, b ^= 1) {
      look_ahead(i, cidx);
#pragma unroll
      for (int x = 0; x < NI; ++x) load(x, b);
#pragma unroll
      for (int x = 0; x < kItems; ++x) put(x, to_at + (b ^ 1) * 2 * kTile);
      if constexpr (kCodes) {
#pragma unroll
        for (int x = 0; x < Quarter<FMT, D>::kKeyLoads; ++x) quarter.load_keys(x, far, wave, lane);
#pragma unroll
        for (int x = 0; x < Quarter<FMT, D>::kValueLoads; ++x) quarter.load_values(x, far, wave, lane);
      }
      end_step();
    }
    if (KH == 1) __syncthreads();
    return;
  }
  for (int i = 0, cidx = t.begin, b = 0; cidx < t.end; ++i, ++cidx, b ^= 1) {
    const bool there = page >= 0;
    const int k0 = cidx << 6;
    look_ahead(i, cidx);
    uint32_t kb = k_at + b * 2 * kTile, vb = v_at + b * 2 * kTile, to = to_at + (b ^ 1) * 2 * kTile;
    asm("" : "+v"(kb), "+v"(vb), "+v"(to));  // the parts' addresses are worked out from here, not kept
    constexpr int kAhead = D == 64 ? 1 : 2;  // operands are read so many pairs of products ahead
    u32x4 kf[kAhead + 1][KH], vf[3], pf[2 * KH];
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
#pragma unroll
      for (int y = 0; y < KH; ++y) kf[x][y] = key_part(kb, y, x);
    f32x16 s[KH] = {};
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < NI; ++x) {
      if (x + kAhead < NI) {
#pragma unroll
        for (int y = 0; y < KH; ++y) kf[(x + kAhead) % (kAhead + 1)][y] = key_part(kb, y, x + kAhead);
      }
      if (x >= NI - 2) vf[x - (NI - 2)] = value_part(vb, 0, x - (NI - 2));
      s[0] = mfma32(kf[x % (kAhead + 1)][0], qf[x], s[0]);
      load(x, b);  // between the matrix instructions: waves that wait for their turn to load would keep them waiting
      if constexpr (KH == 2) s[1] = mfma32(kf[x % (kAhead + 1)][1], qf[x], s[1]);
      if (x < kKeyItems) put(x, to);  // behind the last chunk too, of what was fetched last: nobody reads it
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (D == 256) {  // moved out of the accumulators' registers once
#pragma unroll
      for (int y = 0; y < KH; ++y) asm("" : "+v"(s[y]));
    }
    if (!there || k0 + 63 > wave_pos0 || k0 < wave_last_first) {
      // bit i: the row sees the i-th key of the wave's
      int most = pos - k0 - 32 * first_half, least = from - k0 - 32 * first_half;
      asm volatile("" : "+v"(most));  // a branch: the compiler would do this in every step
      uint64_t sees = (most < 0 ? 0 : ~0ull >> (63 - min(most, 63))) & (least > 63 ? 0 : ~0ull << max(least, 0));
      if (!there) sees = 0;
      sees >>= 4 * half;
      const uint32_t sees0 = (uint32_t)sees, sees1 = (uint32_t)(sees >> 32);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int at = 16 * ((x >> 2) & 1) + 8 * (x >> 3) + (x & 3);
        s[0][x] = seen_or_least(s[0][x], sees0, at);
        if (KH == 2) s[KH - 1][x] = seen_or_least(s[KH - 1][x], sees1, at);
      }
    }
    // two chains, so that one does not wait for itself
    float top = s[0][0], top2 = s[0][1];
#pragma unroll
    for (int x = 0; x < 16 * KH; x += 4) {
      const f32x16& y = s[x / 16];
      top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, y[x % 16]), y[x % 16 + 2]);
      top2 = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top2, y[x % 16 + 1]), y[x % 16 + 3]);
    }
    top = __builtin_elementwise_maximum(top, top2);
    top = max_xor32(top);
    const bool move = (top - ref) * c > slack || (!seen && top > -INFINITY);
    if (__any(move)) {
      const float next_base = fabsf(top * c) < kNear ? fmaf(top, c, -lift) : -lift;
      const bool near = fabsf(top * c) < kNear && fabsf(ref * c) < kNear;
      const float f = !move ? 1.f : !seen ? 0.f : __builtin_amdgcn_exp2f(near ? base - next_base : (ref - top) * c);
      l *= f;
#pragma unroll
      for (int x = 0; x < ND; ++x) {
        if constexpr (D == 256) asm volatile("" : "+a"(acc[x]));  // read here, not in every step
        acc[x] *= f;
      }
      ref = move ? top : ref, base = move ? next_base : base;
      seen |= move;
    }
    const bool far_off = fabsf(ref * c) >= kNear;
    if (__any(far_off)) {
      const float off = far_off ? ref : 0.f;
#pragma unroll
      for (int x = 0; x < 16 * KH; ++x) s[x / 16][x % 16] -= off;
    }
    auto weigh = [&](int x) {
      const f32x16& y = s[x / 8];
      const float p0 = __builtin_amdgcn_exp2f(fmaf(y[2 * (x & 7)], c, -base));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(y[2 * (x & 7) + 1], c, -base));
      const uint32_t w = pack_f16(p0, p1);
      pf[x >> 2][x & 3] = w;
      l = add_f16(w, l);
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) weigh(x);
    constexpr int NV = 2 * KH * ND;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (q + 2 < NV) vf[(q + 2) % 3] = value_part(vb, (q + 2) / ND, (q + 2) % ND);
      acc[q % ND] = mfma32(vf[q % 3], pf[q / ND], acc[q % ND]);
      // the next 16 keys' weights
      if (q / ND < 2 * KH - 1) {
#pragma unroll
        for (int x = 4 * (q / ND + 1) + q % ND * 4 / ND; x < 4 * (q / ND + 1) + (q % ND + 1) * 4 / ND; ++x) weigh(x);
      }
      if constexpr (kCodes) {
        // the keys' next codes, then the values as operands, each followed by its next codes
        constexpr int kItem = kItems - kKeyItems, kEach = (NV - 1) / kItem;
        if (q < Quarter<FMT, D>::kKeyLoads) quarter.load_keys(q, far, wave, lane);
        if (q % kEach == kEach - 1 && q / kEach < kItem) put(kKeyItems + q / kEach, to), quarter.load_values(q / kEach, far, wave, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    end_step();
  }

  l = add_xor32(l);
  float m = !seen ? -INFINITY : fabsf(ref * c) < kNear ? base : fminf(fmaxf(ref * c, -kLargest), kLargest) - lift;
  if constexpr (KH == 1) {
    // the second halves' results through LDS: number x of lane i at 64 x + i
    float* other = reinterpret_cast<float*>(&lds[0][0][0]) + block * (ND * 16 + 2) * 64 + lane;
    if (first_half) {
#pragma unroll
      for (int x = 0; x < 16 * ND; ++x) other[64 * x] = acc[x / 16][x % 16];
      other[64 * 16 * ND] = m, other[64 * (16 * ND + 1)] = l;
    }
    __syncthreads();
    if (first_half) return;
    const float m2 = other[64 * 16 * ND], l2 = other[64 * (16 * ND + 1)], m1 = fmaxf(m, m2);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m1), f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - m1);
#pragma unroll
    for (int x = 0; x < 16 * ND; ++x) acc[x / 16][x % 16] = acc[x / 16][x % 16] * f + other[64 * x] * f2;
    l = l * f + l2 * f2, m = m1;
  }
  int after = mine;
  asm volatile("" : "+v"(after));  // the row's place is worked out again here, not kept through the steps
  if (after >= t.rows) return;
  place(after, row, head);
  // this lane's elements: 32 x + 8 (i / 4) + 4 half + i % 4
  if (u.parts > 1) {
    const uint64_t unit = (((uint64_t)(u.slot + u.part) * a.kv.n_heads + hk) << a.bits) + after;
    float* dst = a.part + unit * D + 4 * half;
#pragma unroll
    for (int x = 0; x < ND; ++x)
#pragma unroll
      for (int i = 0; i < 16; i += 4) *reinterpret_cast<f32x4*>(dst + 32 * x + 2 * i) = f32x4{acc[x][i], acc[x][i + 1], acc[x][i + 2], acc[x][i + 3]};
    float* st = a.part + (uint64_t)kScratchRows * D + unit * 2;
    if (half == 0) st[0] = m, st[1] = l;
    return;
  }
  float f = 1.f;
  if (a.o.sinks) {
    const float sink = sink_of(a.o.sinks, head), m1 = fmaxf(m, sink);
    f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m1);
    l = l * f + (sink == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - m1));
  }
  f = l == 0.f ? 0.f : f / l;
#pragma unroll
  for (int x = 0; x < ND; ++x)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      store4(a.out.p, a.out.dtype, row * a.out.ts + (uint64_t)head * a.out.hs + 32 * x + 2 * i + 4 * half,
             f32x4{acc[x][i], acc[x][i + 1], acc[x][i + 2], acc[x][i + 3]} * f);
}

// Joins the parts of split tile blockIdx.x, a wave for each row: first all parts' weights, then the weighted sums. Memory and the look
// for the tile bound it: 5 to 19 us (51200 rows of 128 in two or three parts).
template <int D>
__global__ __launch_bounds__(64 * kWaves) void k_extend_join(ExtendArgs a) {
  constexpr int L = D / 4, G = 64 / L;  // lanes of a row, parts at a time
  Unit u;
  if (!find_unit(a, true, u)) return;
  const Reach t = reach_of(a, u);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t hk = blockIdx.y;
  const uint64_t apart = (uint64_t)a.kv.n_heads << a.bits;  // rows from a part to the next
  for (int x = blockIdx.z * kWaves + wave; x < t.rows; x += gridDim.z * kWaves) {
    const uint32_t r = (uint32_t)(t.r0 + x), i = a.group.of(r), head = hk * a.group.d + (r - i * a.group.d);
    const uint64_t unit0 = (((uint64_t)u.slot * a.kv.n_heads + hk) << a.bits) + x;
    const float* stat = a.part + (uint64_t)kScratchRows * D + 2 * unit0;
    const float sink = sink_of(a.o.sinks, head);
    float top = sink;
    for (uint32_t p = lane; p < u.parts; p += 64) top = fmaxf(top, stat[2 * p * apart]);
    float base = wave_max(top);
    if (base == -INFINITY) base = 0.f;
    float l = 0.f;
    for (uint32_t p = lane; p < u.parts; p += 64) l += stat[2 * p * apart + 1] * __builtin_amdgcn_exp2f(stat[2 * p * apart] - base);
    l = wave_sum_fast(l) + __builtin_amdgcn_exp2f(sink - base);
    f32x4 acc = {};
    const float* src = a.part + unit0 * D + 4 * (lane % L);
#pragma unroll 4
    for (uint32_t p = lane / L; p < u.parts; p += G)
      acc += *reinterpret_cast<const f32x4*>(src + p * apart * D) * __builtin_amdgcn_exp2f(stat[2 * p * apart] - base);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (G >= 2) acc[j] = add_xor32(acc[j]);
      if (G >= 4) acc[j] = add_xor16(acc[j]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (lane < L)
      store4(a.out.p, a.out.dtype, (uint64_t)(u.sp.q0 + (int)i) * a.out.ts + (uint64_t)head * a.out.hs + 4 * lane, acc * inv);
  }
}

// Whether tiles of 17 to 32 rows are a wave's of its own chunks: where its operands, turned into f16 for two products of 16 rows,
// leave it registers. Else they are a tile of 64 rows of k_attn_extend_wide. 32 sequences of 3 new tokens behind up to 24000, 8 heads
// on each key head, D 64, 128, 256 (8, 4, 2 key heads), this : that (us): MXFP4 81 : 95, 95 : 86, 88 : 125; MXINT8 109 : 116,
// 150 : 106, 144 : 143 (a call: 150 : 139); F16 161 : 153, 184 : 152, 191 : 160.
template <int FMT, int D>
constexpr bool kTwo = FMT != MR_KV_F16 && (D == 64 || (D == 256 && FMT == MR_KV_MXFP4));

using ExtendKernel = void (*)(ExtendArgs);
template <int NT, int FMT, int D>
ExtendKernel pick(int& per_cu) {
  constexpr ExtendKernel kernel = [] {
    if constexpr (NT == 8) return k_attn_extend_wide<FMT, D, 2>;
    else if constexpr (NT == 4) return k_attn_extend_wide<FMT, D, 1>;
    else return k_attn_extend<NT, FMT, D>;
  }();
  static const int n = [] {
    int v = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, kernel, 64 * kWaves, 0) == hipSuccess && v > 0 ? v : 1;
  }();
  per_cu = n;
  return kernel;
}
template <int FMT, int D>
ExtendKernel pick(int& bits, int& per_cu) {
  if (bits == 4) return pick<1, FMT, D>(per_cu);
  if constexpr (kTwo<FMT, D>) {
    if (bits == 5) return pick<2, FMT, D>(per_cu);
  }
  bits = std::max(bits, 6);
  return bits == 6 ? pick<4, FMT, D>(per_cu) : pick<8, FMT, D>(per_cu);
}
template <int FMT>
ExtendKernel pick(uint32_t D, int& bits, int& per_cu) {
  return D == 64 ? pick<FMT, 64>(bits, per_cu) : D == 128 ? pick<FMT, 128>(bits, per_cu) : pick<FMT, 256>(bits, per_cu);
}

}  // namespace

uint64_t attn_extend_scratch_bytes() { return (uint64_t)kScratchRows * (256 + 2) * sizeof(float); }

hipError_t launch_attn_extend(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& q, uint32_t nq,
                              uint32_t n_seqs, const int32_t* cu, const int32_t* len, const int32_t* table,
                              uint32_t max_pages, const AttnOpts& o, const Heads& out, uint32_t* err, float* scratch,
                              int n_cu) {
  const uint32_t group = q.n / kv.n_heads;
  const uint64_t rows = (uint64_t)nq * group;
  int bits = rows <= 16ull * n_seqs ? 4 : rows <= 32ull * n_seqs ? 5 : rows <= 64ull * n_seqs ? 6 : 7;
  int per_cu = 1;
  const ExtendKernel kernel = format == MR_KV_F16      ? pick<MR_KV_F16>(D, bits, per_cu)
                              : format == MR_KV_MXINT8 ? pick<MR_KV_MXINT8>(D, bits, per_cu)
                                                       : pick<MR_KV_MXFP4>(D, bits, per_cu);
  ExtendArgs a{kv, q, out, cu, len, table, max_pages, n_seqs, (int)nq, Divisor(group), bits, rows <= 32ull * n_seqs ? kSlackFew : kSlackMany, 0, o, err, scratch};
  // chunks that a tile sees at most
  const uint64_t pages = (uint64_t)max_pages << (kv.page_shift - 6);
  const uint64_t cap = o.window ? std::min<uint64_t>(pages, (o.window + ((1ull << bits) / group + 1) + 62) / 64 + 1) : pages;
  const uint64_t tiles = (rows >> bits) + n_seqs;  // at most
  // chunks that a sequence's tiles see together, at most
  const uint64_t span = o.window ? std::min<uint64_t>(pages, ((uint64_t)o.window + nq + 62) / 64 + 1) : pages;
  const uint32_t room = std::min<uint32_t>(kScratchRows >> bits, per_cu * n_cu);
  // the chunks of all tiles are counted in 32 bits
  const bool whole = cap <= 2 * kWaves || n_seqs > kSplitSeqs || tiles * span >= 1ull << 31;
  a.parts = whole ? 1 : std::max<uint32_t>(1, room / kv.n_heads);
  hipError_t e;
  {
    ProfScope ps(K, "attn_extend");
    const uint64_t units = a.parts > 1 ? std::max<uint64_t>(a.parts, tiles + a.parts / 2) : tiles;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(units * kv.n_heads)), dim3(64 * kWaves), 0, K.s, a);
    e = hipGetLastError();
    if (e != hipSuccess || a.parts == 1) return e;
  }
  ProfScope ps(K, "extend_join");
  const dim3 j((unsigned)std::min<uint64_t>(tiles, a.parts / 2 + 1), kv.n_heads, bits <= 5 ? 4 : 1 << (bits - 3)), blk(64 * kWaves);
  if (D == 64) hipLaunchKernelGGL((k_extend_join<64>), j, blk, 0, K.s, a);
  if (D == 128) hipLaunchKernelGGL((k_extend_join<128>), j, blk, 0, K.s, a);
  if (D == 256) hipLaunchKernelGGL((k_extend_join<256>), j, blk, 0, K.s, a);
  return hipGetLastError();
}

}  // namespace mr
