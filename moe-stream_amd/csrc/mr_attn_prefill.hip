// mr_attn_prefill.hip -- causal attention over packed prompts.
//
// One pass over the keys with the running maximum m and sum l of each row's softmax:
//   S = K Q^T (keys down, rows across), p = 2^((S - m) c), O = 2^((m_old - m) c) O + V^T p,  c = scale log2 e.
// Both products are 32x32x16 matrix instructions. With the keys down, a lane holds the scores of one
// row, 16 of each 32 keys, so that maximum, sum and p need one exchange between two lanes; and p is
// already where the second product wants its right operand, if that product counts its keys in the
// order the first one left them in (16 c + 4 h + 0..3, then 16 c + 8 + 4 h + 0..3 for lane half h).
// V^T in that order is what the transposing LDS read returns: four adjacent keys of one column.
// p is rounded to the type of v for the second product, as the matrix instructions take it.
//
// Heads of 128: matrix instructions and the exponentials' vector instructions bound it in about equal parts (55% and 46%
// of the cycles), under the card's power limit (1.75 GHz): fewer cycles, as with the pipelined form below, came at a lower
// clock. Of 64: the vector instructions (50% and 73%). Of 256: one wave to a SIMD, whose instructions wait for each other (40% and
// 27%, 2.1 GHz). 8192 tokens, the card warm: heads of 128 (32 on 4) 497 to 515 us by card, 1067 to 1106 TFLOP/s; of 64 (64 on 8) 567
// to 580 us, 948 to 970; of 256 (16 on 2) 555 to 560 us, 982 to 991; the library's products reach 1430 to 1490. With a window of
// 128, 64 heads of 64, 57 us: 151 MB at 2.6 TB/s, the exponentials of steps that rows see in part; short prompts are
// latency, 6 us for 61 tokens.
#include <numeric>

#include "mr_attn_device.h"

namespace mr {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;   // keys of a step
// Up to so many sequences are looked through, 64 at a time, to find a tile's: each step costs about as much as one
// of a search among more, which takes their log2.
constexpr int kScan = 512;
constexpr float kSlack = 8.f;
// f16 weights are 2^kLift times as large: up to 2^15 with kSlack. Ones down to 2^-21 of the largest keep all of
// f16's bits, and what is lost of smaller ones is 2^-32 of it at most; not lifted, 20,000 keys 18 below a first one that has no
// value were lost. bf16 has the range of 32 bits.
template <bool BF>
constexpr float kLift = BF ? 0.f : 7.f;
constexpr float kFar = 0x1p22f;  // a base's last bit is half a power of two from here on, its rounding a quarter
constexpr float kLargest = 0x1.fffffep127f;

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  return BF ? pack_bf16(a, b) : pack_f16(a, b);
}

// Where 16-byte piece `c` of a tile's row lies in LDS, in pieces of the row. Rows are a multiple of the
// 64 banks or half of it: without the exclusive or, the 8 rows of a read's phase would share banks.
template <int D>
__device__ __forceinline__ int k_piece(int row, int c) {
  return D == 64 ? c ^ ((row >> 1) & 7) : c ^ (row & 15);
}
// The transposing read takes 4 adjacent rows and 64 adjacent bytes of each in a phase.
template <int D>
__device__ __forceinline__ int v_piece(int row, int c) {
  return D == 64 ? c ^ (((row >> 1) & 1) * 4) : c ^ ((row & 3) * 4);
}

// 16 bytes a lane from base + offset (a lane's own) straight to LDS, lane i's to dst + 16 i (the same dst for all
// lanes); zeros for lanes whose offset is `bytes` or more. Not the compiler's builtin: after that it waits for
// all of them before each LDS read that it cannot tell apart, here for the next step's tile in the middle of
// this one. The caller waits (vmcnt) and synchronises.
__device__ __forceinline__ void load_lds16(uint64_t base, uint32_t bytes, uint32_t offset, uint32_t dst) {
  const u32x4 rsrc = {(uint32_t)base, (uint32_t)(base >> 32), bytes, 0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(offset), "s"(rsrc)
               : "memory", "m0");
}

// Division of x < 2^24 by 1 <= d < 2^24: with 2^b <= d < 2^(b + 1), x ceil(2^(39 + b) / d) has 64 bits, and over
// 2^(39 + b) it is above x / d by less than x / 2^(39 + b) < 1 / d.
struct Divisor {
  uint64_t mul;
  uint32_t d, shift;
  explicit Divisor(uint32_t d) : d(d), shift(70 - __builtin_clz(d)) { mul = ((1ull << shift) + d - 1) / d; }
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return (uint32_t)((x * mul) >> shift); }
};

// x where bit `at` of `seen` is set, else -infinity.
__device__ __forceinline__ float seen_or_least(float x, uint32_t seen, int at) {
  const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)seen, (uint32_t)at, 1u);
  return bits_f32((keep & __float_as_uint(x)) | (~keep & 0xFF800000u));
}

struct PrefillArgs {
  Heads q, k, v, out;
  int nq, nk, n_seqs, n_tiles;
  int share;        // log2 of the heads side by side: 2, 1, 0, with tiles of 32, 64, 128 rows
  Divisor together;  // head sets (of 1 << share heads) whose tiles take turns
  Divisor turn;      // their tiles
  Divisor group;     // query heads that share a key head
  __device__ __forceinline__ int rows() const { return kPrefillRows >> share; }
  const int32_t *cu_q, *cu_k;
  AttnOpts o;
  uint32_t* err;
};

// The sequence and first row of row tile `tile`; false for a tile that there is not. Offsets are clamped into
// the rows; `report` also looks at all of them.
struct Place {
  int q0, q1, k0, k1;  // the sequence's rows
  int row;             // the tile's first row
};
__device__ __forceinline__ bool find_tile(const PrefillArgs& a, int tile, bool report, int lane, Place& p) {
  struct Seq {
    int q0, q1, k0, k1, tiles;
    bool bad;
  };
  const int row_bits = 7 - a.share;
  auto seq = [&](int s) {
    auto in = [](int x, int hi) { return min(max(x, 0), hi); };
    const int x = a.cu_q[s], y = a.cu_q[s + 1], kx = a.cu_k[s], ky = a.cu_k[s + 1];
    Seq r{in(x, a.nq), in(y, a.nq), in(kx, a.nk), in(ky, a.nk), 0, x < 0 || y < x || y > a.nq || kx < 0 || ky < kx || ky > a.nk};
    r.q1 = max(r.q0, r.q1), r.k1 = max(r.k0, r.k1), r.tiles = (r.q1 - r.q0 + a.rows() - 1) >> row_bits;
    return r;
  };
  const bool search = a.n_seqs > kScan;
  bool found = false;
  if (search) {
    // Sequence s has the tiles from cu_q[s] / rows + s on: room for one that is not full, some left out.
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((min(max(a.cu_q[mid], 0), a.nq) >> row_bits) + mid <= tile) lo = mid;
      else hi = mid - 1;
    }
    const Seq r = seq(lo);
    const int i = tile - ((r.q0 >> row_bits) + lo);
    found = i >= 0 && i < r.tiles;
    p.q0 = __builtin_amdgcn_readfirstlane(r.q0), p.q1 = __builtin_amdgcn_readfirstlane(r.q1);
    p.k0 = __builtin_amdgcn_readfirstlane(r.k0), p.k1 = __builtin_amdgcn_readfirstlane(r.k1);
    p.row = __builtin_amdgcn_readfirstlane(r.q0 + (r.tiles - 1 - i) * a.rows());
    if (!report) return __builtin_amdgcn_readfirstlane(found);
  }
  int before = 0;
  for (int s0 = 0; s0 < a.n_seqs && (report || !found); s0 += 64) {
    const Seq r = s0 + lane < a.n_seqs ? seq(s0 + lane) : Seq{};
    if (report && __any(r.bad) && lane == 0) note_error(a.err, kErrOffset);
    if (search) continue;
    const int sum = (int)wave_prefix((uint32_t)r.tiles);
    const uint64_t past = __ballot(before + sum > tile);
    if (past && !found) {
      const int l = __ffsll((unsigned long long)past) - 1;
      p.q0 = __builtin_amdgcn_readlane(r.q0, l), p.q1 = __builtin_amdgcn_readlane(r.q1, l);
      p.k0 = __builtin_amdgcn_readlane(r.k0, l), p.k1 = __builtin_amdgcn_readlane(r.k1, l);
      // the longest rows first
      p.row = p.q0 + (before + __builtin_amdgcn_readlane(sum, l) - 1 - tile) * a.rows();
      found = true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return found;
}

// One tile of rows and one head. p is 0 where a row does not see a key, but 0 * inf and 0 * NaN are NaN: a tile
// that ends with such a sum returns false and is done over with `careful`, where values that are not finite
// are taken out of the steps that some row sees in part, and added at the end to the rows that see them.
//
// p is 2^((S - m) c + kLift). For heads of 64 and 128 it is worked out as 2^(S c - base), base = m c - kLift, an instruction
// less: the base's rounding is then the same factor on all of a row's weights. Where a base is so large (kFar) that this
// factor could leave the range of 16 bits, the tile is done over `careful` too, with the differences taken first.
template <int D, bool BF>
__device__ __forceinline__ bool attend_tile(const PrefillArgs& a, uint16_t* lds, int unit, bool careful) {
  constexpr int P = D / 8, ND = D / 32;  // 16-byte pieces of a row; 32-wide tiles of a head
  constexpr int kTile = kKeys * D;       // elements of a key or value tile
  constexpr uint32_t kTop = BF ? 0x7F80u : 0x7C00u;  // the exponent of infinities and NaN
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // nothing is kept in registers for the second time over
  const int wave = __builtin_amdgcn_readfirstlane(thread >> 6), lane = thread & 63, n = lane & 31, half = lane >> 5;

  const uint32_t set = a.turn.of(unit), in_set = unit - set * a.turn.d, tile = a.together.of(in_set);
  const int h0 = (int)(set * a.together.d + in_set - tile * a.together.d) << a.share, h = h0 + (wave & ((1 << a.share) - 1));
  const int hk = (int)a.group.of(h0), wave_row = (wave >> a.share) * 32;
  Place pl;
  if (!find_tile(a, (int)tile, unit == 0 && !careful, lane, pl)) return true;

  // keys [first, last] of the tile's rows; a row r sees those up to r + diff, from r + diff - window + 1 on
  const int diff = pl.k1 - pl.q1;
  const int row = pl.row + wave_row + n;  // this lane's query row
  const int last_row = min(pl.row + a.rows(), pl.q1) - 1;
  const int last = last_row + diff;  // < k1
  int first = pl.k0;
  if (a.o.window) first = (int)max((int64_t)first, (int64_t)pl.row + diff + 1 - (int64_t)a.o.window);
  const int see_last = row + diff;
  const int64_t w = a.o.window ? (int64_t)a.o.window : (int64_t)1 << 32;
  const int see_first = (int)max((int64_t)pl.k0, (int64_t)see_last + 1 - w);
  const int wave_least = (int)max((int64_t)pl.k0, (int64_t)pl.row + wave_row + diff + 1 - w);  // first key of its first row
  const int wave_first = (int)max((int64_t)pl.k0, (int64_t)pl.row + wave_row + 31 + diff + 1 - w);  // of its last row

  // above zero and finite: a masked score times c stays -inf, a score of zero zero
  const float c = fminf(fmaxf(fabsf(a.o.scale) * 1.44269504088896340736f, 0x1p-126f), kLargest);
  u32x4 qf[D / 16];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q.p) + (uint64_t)min(row, pl.q1 - 1) * a.q.ts + (uint64_t)h * a.q.hs;
    const uint32_t flip = a.o.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = *reinterpret_cast<const u32x4*>(qp + 16 * i + 8 * half) ^ flip;
  }

  const uint16_t* kp = static_cast<const uint16_t*>(a.k.p) + (uint64_t)hk * a.k.hs;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v.p) + (uint64_t)hk * a.v.hs;
  // Copies the 64 keys from k0 on into buffer b, zeros for rows behind the last key. A wave's load is kStep / 4
  // rows; the pieces' order within a row is the same every 16 rows.
  constexpr int kLoads = kTile / 8 / 256, kStep = kKeys / kLoads, kOff = kStep < 16 ? 16 / kStep : 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t*)lds;
  uint32_t k_off[kOff], v_off;
  {
    const int r = (wave * 64 + lane) / P, cp = lane % P;
#pragma unroll
    for (int i = 0; i < kOff; ++i) k_off[i] = (uint32_t)(r * a.k.ts + 8 * k_piece<D>(r + i * kStep, cp)) * 2;
    v_off = (uint32_t)(r * a.v.ts + 8 * v_piece<D>(r, cp)) * 2;
  }
  // One base and bound for a tile, with the rows in the lanes' offsets: worked out for each load it was 90 scalar instructions
  // a step (8192 tokens, heads of 128 504 -> 496 us, of 256 577 -> 541).
  const uint32_t k_step = (uint32_t)(kStep * a.k.ts) * 2, v_step = (uint32_t)(kStep * a.v.ts) * 2;
  auto fetch_k = [&](int k0, int b) {
    const uint64_t base = (uint64_t)kp + (uint64_t)k0 * a.k.ts * 2;
    const uint32_t bytes = (uint32_t)(min(last - k0, kKeys - 1) * a.k.ts + D) * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_lds16(base, bytes, k_off[i % kOff] + i * k_step, lds0 + b * 4 * kTile + (i * 4 + wave) * 1024);
  };
  auto fetch_v = [&](int k0, int b) {
    const uint64_t base = (uint64_t)vp + (uint64_t)k0 * a.v.ts * 2;
    const uint32_t bytes = (uint32_t)(min(last - k0, kKeys - 1) * a.v.ts + D) * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_lds16(base, bytes, v_off + i * v_step, lds0 + b * 4 * kTile + 2 * kTile + (i * 4 + wave) * 1024);
  };

  // whether some row of the workgroup does not see some key of the step
  const int64_t all_first = a.o.window ? (int64_t)last + 1 - (int64_t)a.o.window : pl.k0;
  auto edge = [&](int k0) { return k0 < all_first || k0 + kKeys - 1 > pl.row + diff; };

  f32x16 acc[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) acc[t] = f32x16{};
  // Heads of 256 take differences always, mostly beside the matrix instructions (8192 tokens: 550 us without, 560 so): with both
  // forms in the loop the compiler has no registers left for it.
  constexpr bool kDiff = D == 256;
  float m = -INFINITY, l = 0.f;
  const float c_base = careful ? 0.f : c;
  // finite where no key has been seen (-inf, or 0 * -inf): a masked score stays -inf
  auto base_of = [&] { return fmaxf(kDiff ? m : fmaf(m, c_base, -kLift<BF>), -kLargest); };
  // A sink joins at the end: as the first maximum, one far above the scores left their weights no bits in f16.
  const float sink = sink_of(a.o.sinks, h);

  constexpr int NI = D / 16, NV = 4 * ND;
  // Operand of the scores: 8 elements of key 32 t + n; of the values: V^T of 16 keys and 32 elements, where lane
  // 16 g + i of a transposing read takes row (i >> 2), elements 4 (i & 3).. and gets column i of four rows.
  // Pieces are exclusive-ored into place, and so are the parts' addresses from the first one's.
  const int vr = 4 * half + ((lane & 15) >> 2), ve = (lane & 16) + 4 * (lane & 3);
  const uint32_t k_at = lds0 + 2 * (n * D + 8 * k_piece<D>(n, half));
  const uint32_t v_at = lds0 + 2 * (kTile + vr * D + 8 * v_piece<D>(vr, ve >> 3) + (ve & 7));
  auto key_part = [&](uint32_t k_at, int t, int i) {
    const uint32_t at = (k_at ^ (32 * i)) + t * 64 * D;
    return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
  };
  auto value_part = [&](uint32_t v_at, int q) {
    const uint32_t at = (v_at ^ (64 * (q % ND))) + (q / ND) * 32 * D;
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)at));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)(at + 16 * D)));
    return u32x4{x.x, x.y, y.x, y.y};
  };
  // Masks the scores of the keys from k0 on and moves the maximum m, with the sums, if theirs has left it
  // kSlack behind: p is at most 2^(kSlack + kLift), and nearly no step rescales.
  auto settle = [&](int k0, f32x16& s0, f32x16& s1) {
    if (k0 + kKeys - 1 > pl.row + wave_row + diff || k0 < wave_first) {
      // Bit i: the row sees the i-th key from its half's first on. A bit and a select a score; a comparison and a select for
      // each end have waits between them (8192 tokens, heads of 128, with the maxima below: 496 -> 492 us).
      int most = see_last - k0 - 4 * half, least = see_first - k0 - 4 * half;
      asm volatile("" : "+v"(most));  // a branch: the compiler would do this in every step
      const uint64_t seen = (most < 0 ? 0 : ~0ull >> (63 - min(most, 63))) & (least > 63 ? 0 : ~0ull << max(least, 0));
      const uint32_t seen0 = (uint32_t)seen, seen1 = (uint32_t)(seen >> 32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = 8 * (i >> 2) + (i & 3);
        s0[i] = seen_or_least(s0[i], seen0, at);
        s1[i] = seen_or_least(s1[i], seen1, at);
      }
    }
    float top = s0[0];
#pragma unroll
    for (int i = 0; i < 16; ++i) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s0[i]), s1[i]);
    top = max_xor32(top);
    if (__any((top - m) * c > kSlack)) {
      const float m1 = fmaxf(m, top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m1) * c);
      l *= f;
#pragma unroll
      for (int t = 0; t < ND; ++t) acc[t] *= f;
      m = m1;
    }
    if (!kDiff && careful) {
      const float first = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[i] -= first, s1[i] -= first;
    }
  };
  // Two of a step's 32 weights (pair i): rounded into the operand of the second product.
  auto weigh = [&](const f32x16& s0, const f32x16& s1, int i, float base, u32x4 (&pf)[4]) {
    const f32x16& s = i < 8 ? s0 : s1;
    const float x0 = s[2 * (i & 7)], x1 = s[2 * (i & 7) + 1];
    const float p0 = __builtin_amdgcn_exp2f(kDiff ? fmaf(x0 - base, c, kLift<BF>) : fmaf(x0, c, -base));
    const float p1 = __builtin_amdgcn_exp2f(kDiff ? fmaf(x1 - base, c, kLift<BF>) : fmaf(x1, c, -base));
    const uint32_t w = pack16<BF>(p0, p1);
    pf[i >> 2][i & 3] = w;
    l = BF ? add_bf16(w, l) : add_f16(w, l);
  };
  // Takes the values that are not finite out of buffer b.
  auto clean = [&](int b) {
    uint16_t* vt = lds + b * 2 * kTile + kTile;
    for (int i = threadIdx.x; i < kTile; i += 256)
      if ((vt[i] & kTop) == kTop) vt[i] = 0;
    __syncthreads();
  };

  if constexpr (D != 256) {
    // Two waves or more to a SIMD: one's matrix instructions run beside another's exponentials.
    if (first <= last) {
      fetch_k(first, 0), fetch_v(first, 0);
      for (int k0 = first, b = 0; k0 <= last; k0 += kKeys, b ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (k0 + kKeys <= last) fetch_k(k0 + kKeys, b ^ 1), fetch_v(k0 + kKeys, b ^ 1);
        if (careful && edge(k0)) clean(b);
        // keys behind all of the wave's rows, or in front of all their windows
        if (k0 > pl.row + wave_row + 31 + diff || k0 + kKeys <= wave_least) continue;
        uint32_t kb = k_at + b * 4 * kTile, vb = v_at + b * 4 * kTile;
        asm("" : "+v"(kb), "+v"(vb));  // the parts' addresses are worked out from here, not kept
        f32x16 s0 = {}, s1 = {};
        // Key operands are read so many pairs of products ahead: for heads of 128 one 512 us, two 505; for heads of 64 the second
        // pair has no registers left.
        constexpr int kAhead = D == 128 ? 2 : 1;
        u32x4 pf[4], kf[kAhead + 1][2], vf[3];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) kf[i][0] = key_part(kb, 0, i), kf[i][1] = key_part(kb, 1, i);
        // Waves between their matrix instructions give way to those at them: the two of a SIMD then take turns
        // (8192 tokens, heads of 128: 675 -> 649 us, before the later steps).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (i + kAhead < NI) {
            kf[(i + kAhead) % (kAhead + 1)][0] = key_part(kb, 0, i + kAhead);
            kf[(i + kAhead) % (kAhead + 1)][1] = key_part(kb, 1, i + kAhead);
          }
          if (i >= NI - 2) vf[i - (NI - 2)] = value_part(vb, i - (NI - 2));
          s0 = mfma32<BF>(kf[i % (kAhead + 1)][0], qf[i], s0);
          s1 = mfma32<BF>(kf[i % (kAhead + 1)][1], qf[i], s1);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        settle(k0, s0, s1);
        const float base = base_of();
#pragma unroll
        for (int x = 0; x < 4; ++x) weigh(s0, s1, x, base, pf);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int q = 0; q < NV; ++q) {
          if (q + 2 < NV) vf[(q + 2) % 3] = value_part(vb, q + 2);
          acc[q % ND] = mfma32<BF>(vf[q % 3], pf[q / ND], acc[q % ND]);
          // the next 16 keys' weights
          if (q / ND < 3) {
#pragma unroll
            for (int x = 4 * (q / ND + 1) + q % ND * 4 / ND; x < 4 * (q / ND + 1) + (q % ND + 1) * 4 / ND; ++x) weigh(s0, s1, x, base, pf);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
  } else {
    // One wave to a SIMD: the scores run a step ahead of the values, so that a wave's matrix instructions have its own
    // exponentials between them (8192 tokens, heads of 256: 742 -> 655 us; of 128, where two waves do the same
    // for each other, 619 -> 647).
    //
    // Scores (p, q) of one step, their first and second 32 keys; the next ones go to x and, once p's weights are
    // taken, to p.
    constexpr int kAhead = 3;  // products between an operand's read and its use: 2 618 us, 3 604, 4 and 5 no better
    auto step = [&](int k0, int b, f32x16& p, f32x16& q, f32x16& x) {
      const float base = base_of();
      u32x4 pf[4], kf[kAhead + 1], vf[kAhead + 1];
      uint32_t kb = k_at + (b ^ 1) * 4 * kTile, vb = v_at + b * 4 * kTile;
      asm("" : "+v"(kb), "+v"(vb));  // the parts' addresses are worked out from here, not kept
#pragma unroll
      for (int i = 0; i < kAhead; ++i) kf[i] = key_part(kb, 0, i);
      f32x16 n0 = {};
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        kf[(i + kAhead) % (kAhead + 1)] = key_part(kb, (i + kAhead) / NI, (i + kAhead) % NI);
        n0 = mfma32<BF>(kf[i % (kAhead + 1)], qf[i], n0);
#pragma unroll
        for (int y = i * 8 / NI; y < (i + 1) * 8 / NI; ++y) weigh(p, p, y, base, pf);
        __builtin_amdgcn_sched_barrier(0);
      }
      x = n0;
      f32x16 n1 = {};
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (i + kAhead < NI) kf[(NI + i + kAhead) % (kAhead + 1)] = key_part(kb, 1, i + kAhead);
        else vf[i + kAhead - NI] = value_part(vb, i + kAhead - NI);
        n1 = mfma32<BF>(kf[(NI + i) % (kAhead + 1)], qf[i], n1);
#pragma unroll
        for (int y = 8 + i * 8 / NI; y < 8 + (i + 1) * 8 / NI; ++y) weigh(q, q, y, base, pf);
        __builtin_amdgcn_sched_barrier(0);
      }
      p = n1;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i + kAhead < NV) vf[(i + kAhead) % (kAhead + 1)] = value_part(vb, i + kAhead);
        acc[i % ND] = mfma32<BF>(vf[i % (kAhead + 1)], pf[i / ND], acc[i % ND]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      settle(k0 + kKeys, x, p);
    };
    // Between steps: the other buffer's tiles have come in, and this one's keys are no longer needed.
    auto turn = [&](int k0, int b) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (k0 + kKeys <= last) fetch_v(k0 + kKeys, b ^ 1);
      if (k0 + 2 * kKeys <= last) fetch_k(k0 + 2 * kKeys, b);
      if (careful && edge(k0)) clean(b);
    };
    if (first <= last) {
      fetch_k(first, 0), fetch_v(first, 0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (first + kKeys <= last) fetch_k(first + kKeys, 1);
      f32x16 s0 = {}, s1 = {}, s2 = {};
      uint32_t kb = k_at;
      asm("" : "+v"(kb));
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        s0 = mfma32<BF>(key_part(kb, 0, i), qf[i], s0);
        s1 = mfma32<BF>(key_part(kb, 1, i), qf[i], s1);
        __builtin_amdgcn_sched_barrier(0);
      }
      settle(first, s0, s1);
      int b = 0;
      for (int k0 = first;;) {
        turn(k0, b);
        if (k0 + kKeys > last) break;
        step(k0, b, s0, s1, s2);
        k0 += kKeys, b ^= 1;
        turn(k0, b);
        if (k0 + kKeys > last) {
          s1 = s0, s0 = s2;
          break;
        }
        step(k0, b, s2, s0, s1);
        k0 += kKeys, b ^= 1;
        turn(k0, b);
        if (k0 + kKeys > last) {
          s0 = s1, s1 = s2;
          break;
        }
        step(k0, b, s1, s2, s0);
        k0 += kKeys, b ^= 1;
      }
      const float base = base_of();
      u32x4 pf[4];
      uint32_t vb = v_at + b * 4 * kTile;
      asm("" : "+v"(vb));
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
#pragma unroll
        for (int x = 4 * cc; x < 4 * cc + 4; ++x) weigh(s0, s1, x, base, pf);
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          acc[t] = mfma32<BF>(value_part(vb, cc * ND + t), pf[cc], acc[t]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  if (!careful) {
    float most = 0.f;  // NaN if any sum is
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = __builtin_elementwise_maximum(most, fabsf(acc[t][i]));
    const bool far = !kDiff && m != -INFINITY && !(fabsf(m) * c < kFar);
    if (__syncthreads_or(far || !(most < INFINITY))) return false;
  }

  l = add_xor32(l);
  float own = 1.f;
  if (sink != -INFINITY) {
    const float top = m == -INFINITY ? m : fminf(fmaxf(m * c, -kLargest), kLargest) - kLift<BF>, m1 = fmaxf(top, sink);
    own = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m1);
    l = l * own + __builtin_amdgcn_exp2f(sink - m1);  // NaN for a sink that is infinite or NaN
  }
  const float inv = l > 0.f ? own / l : l == 0.f ? 0.f : NAN;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // the row's address is worked out here, not kept through the steps
  const int out_row = pl.row + wave_row + (tid & 31);
  if (out_row < pl.q1) {
    uint16_t* dst = static_cast<uint16_t*>(a.out.p) + (uint64_t)out_row * a.out.ts + (uint64_t)h * a.out.hs;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const u32x2 w = {pack16<BF>(acc[t][i] * inv, acc[t][i + 1] * inv), pack16<BF>(acc[t][i + 2] * inv, acc[t][i + 3] * inv)};
        *reinterpret_cast<u32x2*>(dst + 32 * t + 8 * (i >> 2) + 4 * (tid >> 5 & 1)) = w;
      }
  }
  if (careful) {
    __syncthreads();  // the rows are written
    const int d = threadIdx.x % D;
    for (int k0 = first; k0 <= last; k0 += kKeys) {
      if (!edge(k0)) continue;
      for (int key = k0; key < min(k0 + kKeys, last + 1); ++key) {
        const uint16_t x = vp[(uint64_t)key * a.v.ts + d];
        if ((x & kTop) != kTop) continue;
        for (int i = threadIdx.x / D; i < (last_row + 1 - pl.row) << a.share; i += 256 / D) {
          const int r = pl.row + (i >> a.share), head = h0 + (i & ((1 << a.share) - 1));
          if (key > r + diff || (a.o.window && key <= (int64_t)r + diff - (int64_t)a.o.window)) continue;
          uint16_t* dst = static_cast<uint16_t*>(a.out.p) + (uint64_t)r * a.out.ts + (uint64_t)head * a.out.hs + d;
          const float y = BF ? bits_f32((uint32_t)*dst << 16) + bits_f32((uint32_t)x << 16) : h2f(*dst) + h2f(x);
          *dst = (uint16_t)pack16<BF>(y, 0.f);
        }
      }
    }
  }
  return true;
}

// Waves of a SIMD, and so workgroups of a CU.
template <int D>
constexpr int kLayers = D == 256 ? 1 : D == 128 ? 2 : 4;

template <int D, bool BF>
__global__ __launch_bounds__(256, kLayers<D>) void k_attn_prefill(PrefillArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[4 * kKeys * D];  // rows at multiples of their length
  // Workgroups go to the 8 XCDs in turn. Each XCD gets an eighth of the head sets, so that the query heads that share
  // keys find them in one L2; sets that are not a multiple of 8 are spread over all.
  const int sets = (int)a.q.n >> a.share, units = a.n_tiles * sets;
  // An XCD's 32 CUs hold so many workgroups each at once, the first 32 one each, and so on: every second of these layers goes
  // the other way round, so that a CU's tiles are long and short ones (2048 tokens, 32 heads of 128: 50.7 us without,
  // 46.2 so; 4096, 12 heads: 83.4 and 75.7; 64 heads of 64: 158.5 and 153.8; three prompts behind 2000 tokens, heads
  // of 128: 185 and 188).
  const int per = (units + 7) / 8, xcd = blockIdx.x & 7;
  int at = blockIdx.x >> 3;
  const int layer = at / 32;
  if (layer < kLayers<D> && (layer & 1)) at = 32 * layer + min(32, per - 32 * layer) - 1 - at % 32;
  const int unit = sets % 8 ? at * 8 + xcd : xcd * per + at;
  if (unit >= units) return;
  for (bool careful = false; !attend_tile<D, BF>(a, lds, unit, careful); careful = true) {
  }
}

}  // namespace

hipError_t launch_attn_prefill(const Launch& K, uint32_t D, const Heads& q, uint32_t nq, const Heads& k, const Heads& v,
                               uint32_t nk, uint32_t n_seqs, const int32_t* cu_q, const int32_t* cu_k, const AttnOpts& o,
                               const Heads& out, uint32_t* err) {
  ProfScope ps(K, "attn_prefill");
  // A tile is of 4, 2 or 1 heads that share their keys and of 32, 64 or 128 rows. With the 4 waves at the same rows all take
  // all of the tile's steps: with a window of 128 they are 3, not 4 of which each wave needs 3 (8192 tokens, 64 heads
  // of 64: 63.2 us by 128 rows, 58.4 by 32 and 4 heads; 2000 earlier tokens, 16 heads of 256: 229 and 221; 20 prompts
  // of 17 tokens: 10.7 and 7.6; but one of 61 tokens 5.8 and 6.5, in half as many workgroups).
  const uint32_t group = q.n / k.n, share = group % 4 == 0 ? 2 : group % 2 == 0 ? 1 : 0, rows = kPrefillRows >> share;
  // every sequence ends with at most one tile that is not full
  const uint64_t most = (uint64_t)nq / rows + n_seqs, tiles = n_seqs > kScan ? most : std::min<uint64_t>(most, nq);
  const uint32_t sets = q.n >> share, per_xcd = sets / 8;
  const uint64_t units = tiles * sets;  // below 2^24, checked by the caller
  // Workgroups start in the order of their units, the longest rows first: with that for all of an XCD's heads at once the
  // last to start are short (4096 tokens, 32 heads of 128 on 4: 177 us head by head, 142 so; on 32: 179 and 144; 28 on
  // 4, over all XCDs: 170 and 130). More than 16 heads that share no keys lose more by it in the L2s than they gain
  // (256 heads on 256, 32 of them to an XCD: 349 and 362).
  const uint32_t together = sets % 8 ? sets : per_xcd <= 16 ? per_xcd : std::gcd(per_xcd, 16u);
  PrefillArgs a{q, k, v, out, (int)nq, (int)nk, (int)n_seqs, (int)tiles, (int)share, Divisor(together),
                Divisor(together * (uint32_t)tiles), Divisor(group), cu_q, cu_k, o, err};
  const dim3 g((unsigned)((units + 7) / 8 * 8)), blk(256);
  const bool bf = q.dtype == MR_BF16;
  if (D == 64) hipLaunchKernelGGL((bf ? k_attn_prefill<64, true> : k_attn_prefill<64, false>), g, blk, 0, K.s, a);
  if (D == 128) hipLaunchKernelGGL((bf ? k_attn_prefill<128, true> : k_attn_prefill<128, false>), g, blk, 0, K.s, a);
  if (D == 256) hipLaunchKernelGGL((bf ? k_attn_prefill<256, true> : k_attn_prefill<256, false>), g, blk, 0, K.s, a);
  return hipGetLastError();
}

}  // namespace mr
