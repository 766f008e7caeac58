// mr_kv.hip -- the paged cache of keys and values: quantising what is written, and reading it back.
//
// A block of 32 elements is stored as codes * 2^e. e comes from the bits of the largest magnitude and
// x * 2^-e is exact, so the codes are the nearest ones, with no rounding before the last. Memory bounds large calls
// (100001 tokens of 2 heads of 256, f32 to 8 bits: 516 MB in 126 us, 4.1 TB/s), latency small ones: 5 us.
#include "mr_attn_device.h"

namespace mr {

namespace {

__device__ __forceinline__ float finite_or_inf(float x) { return x == x ? x : 0.f; }

// Value of the MXINT8 code in the low byte of c; +0 for a slot that was never written (scale 0).
__device__ __forceinline__ float int8_value(uint32_t c, float scale) { return fmaf((float)((int)(c & 0xFFu) - 128), scale, 0.f); }

// The block exponent for the largest magnitude `top`.
template <int FMT>
__device__ __forceinline__ int block_exp(float top) {
  const uint32_t b = __float_as_uint(top), man = b & 0x7FFFFFu;
  const int E = (int)(b >> 23) - 127;
  const int e = FMT == MR_KV_MXFP4 ? E - 2 + (man > 0x600000u) : E - 6 + (man >= 0x7F0000u);
  return min(max(e, -16), FMT == MR_KV_MXFP4 ? 13 : 9);
}
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(int e) {
  if (FMT == MR_KV_MXFP4) return (uint32_t)(e + 127);
  return e >= -14 ? (uint32_t)(e + 15) << 2 : e == -15 ? 2u : 1u;
}
template <int FMT>
__device__ __forceinline__ uint32_t code(float y) {
  if (FMT == MR_KV_MXINT8) return (uint32_t)((int)rintf(fminf(fmaxf(y, -127.f), 127.f)) + 128);
  const float a = fabsf(y);
  const uint32_t c = (uint32_t)(a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
  return y < 0.f && c ? c | 8u : c;
}

// Token s of the chunk that slot `slot` lies in; nullptr (and the error word) for a slot out of range.
__device__ __forceinline__ uint8_t* find(const KvPages& kv, int slot, uint32_t head, uint32_t* err, int& s) {
  const uint32_t page = (uint32_t)slot >> kv.page_shift;
  if (slot < 0) return nullptr;
  if (page >= kv.n_pages) {
    note_error(err, kErrSlot);
    return nullptr;
  }
  s = slot & 63;
  return kv.at(page, head, ((uint32_t)slot & ((1u << kv.page_shift) - 1u)) >> 6);
}

constexpr int kWindow = 64;  // tokens of a workgroup

// Runs of tokens that fill a chunk. The values' bytes of a token lie 16 bytes apart in its chunk; where 64 tokens
// in a row go to (come from) the 64 slots of a chunk in order, as most of a prompt's do, they are put together
// in LDS and the chunk is moved whole (8192 tokens, 4 heads of 128, 8 bits, the same again: 8.3 us written, 8.0 read; 100001 tokens,
// 2 heads of 256: written in 232 us one by one, in 126 so). The workgroup in whose
// window of 64 tokens such a run begins does all of it. Of the others, kPiece tokens or more in a row in a chunk (a
// prompt's first and last) go four at a time to words of the chunk: 8191 tokens were written in 12.4 us and read in 12.9 with
// the last 63 one by one, each byte an access of its own in one workgroup, and are in 10.7 and 8.9. The rest go one by one.
struct Runs {
  // bit i: token i of the window begins a run; begins a piece; ends a row of tokens in a chunk; is in none, and has a slot
  uint64_t start, piece, end, single;
};
constexpr int kPiece = 8;
__device__ __forceinline__ int piece_length(uint64_t end, int b) { return __ffsll((unsigned long long)(end >> b)); }
// slots[i] is the slot of token i - 63 of the window, -1 outside the call. All threads call.
__device__ __forceinline__ Runs find_runs(const KvPages& kv, const int32_t* __restrict__ slots, int T, int t0, int (&sl)[192],
                                          uint64_t (&breaks)[3]) {
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < 192) {
    const int t = t0 - 63 + tid;
    sl[tid] = tid < 191 && t >= 0 && t < T ? slots[t] : -1;
  }
  __syncthreads();
  if (tid < 192) {
    const bool b = tid == 191 || sl[tid] < 0 || (uint32_t)sl[tid + 1] != (uint32_t)sl[tid] + 1u;
    const uint64_t m = __ballot(b);
    if (lane == 0) breaks[tid >> 6] = m;
  }
  __syncthreads();
  const int slot = sl[63 + lane], first = 63 + lane - (slot & 63);  // where this token's run would begin
  bool in_run = false;
  if (slot >= 0 && first >= 0 && ((uint32_t)slot >> kv.page_shift) < kv.n_pages) {
    const int w = first >> 6, o = first & 63;
    const uint64_t lo = breaks[w] >> o, hi = o && w < 2 ? breaks[w + 1] << (64 - o) : 0;
    in_run = ((lo | hi) & 0x7FFFFFFFFFFFFFFFull) == 0;
  }
  Runs r;
  r.start = __ballot(in_run && (slot & 63) == 0);
  const uint64_t rest = __ballot(!in_run && slot >= 0);
  r.end = __ballot(lane == 63 || (breaks[(63 + lane) >> 6] >> ((63 + lane) & 63) & 1) || (slot & 63) == 63);
  // a piece: begins behind an end, is long enough, and lies in the cache
  const bool first_in = (lane == 0 || (r.end >> (lane - 1) & 1)) && (rest >> lane & 1);
  r.piece = __ballot(first_in && ((uint32_t)slot >> kv.page_shift) < kv.n_pages && piece_length(r.end, lane) >= kPiece);
  r.single = rest;
  for (uint64_t todo = r.piece; todo; todo &= todo - 1) {
    const int b = __ffsll((unsigned long long)todo) - 1;
    r.single &= ~((~0ull >> (64 - piece_length(r.end, b))) << b);
  }
  return r;
}

// Two quads of a token: 8 adjacent elements for keys, 32 b + 4 w and 32 b + 16 + 4 w for values (the two
// nibbles of a byte).
struct Quads {
  int e0, e1;
};
__device__ __forceinline__ Quads quads(bool key, int u) {
  const int e0 = key ? 8 * u : 32 * (u >> 2) + 4 * (u & 3);
  return Quads{e0, key ? e0 + 4 : e0 + 16};
}

// Codes of 8 elements (for F16 the f16 bits), and the block's exponent. The 4 lanes of a block call together.
template <int FMT>
__device__ __forceinline__ int quantise(f32x4 x, f32x4 y, uint32_t (&c)[8]) {
  float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = finite_or_inf(v[i]), top = fmaxf(top, fabsf(v[i]));
  if constexpr (FMT == MR_KV_F16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = pack_f16(fminf(fmaxf(v[i], -65504.f), 65504.f), 0.f);
    return 0;
  }
  top = fmaxf(top, __shfl_xor(top, 1, kWave));
  top = fmaxf(top, __shfl_xor(top, 2, kWave));
  const int ex = block_exp<FMT>(top);
  const float inv = bits_f32((uint32_t)(127 - ex) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = code<FMT>(v[i] * inv);
  return ex;
}

// Quantises 8 elements of token s and stores them in the chunk. The 4 lanes of a block call together.
template <int FMT, int D, bool KEY>
__device__ __forceinline__ void put(uint8_t* chunk, int s, int u, f32x4 x, f32x4 y) {
  using L = KvLayout<FMT, D>;
  const Quads e = quads(KEY, u);
  uint32_t c[8];
  const int ex = quantise<FMT>(x, y, c);
  if (FMT != MR_KV_F16 && (u & 3) == 0) chunk[KEY ? L::ks_off(s, u >> 2) : L::vs_off(s, u >> 2)] = (uint8_t)scale_byte<FMT>(ex);
  if constexpr (KEY) {
    uint8_t* p = chunk + L::k_off(s, e.e0);
    if constexpr (FMT == MR_KV_F16) {
      *reinterpret_cast<u32x4*>(p) = u32x4{c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16};
    } else if constexpr (FMT == MR_KV_MXINT8) {
      *reinterpret_cast<u32x2*>(p) = u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= c[i] << (4 * i);
      *reinterpret_cast<uint32_t*>(p) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint8_t *lo = chunk + L::v_off(s, e.e0 + i), *hi = chunk + L::v_off(s, e.e1 + i);
      if constexpr (FMT == MR_KV_MXFP4) {
        *lo = (uint8_t)(c[i] | c[i + 4] << 4);
      } else if constexpr (FMT == MR_KV_MXINT8) {
        *lo = (uint8_t)c[i], *hi = (uint8_t)c[i + 4];
      } else {
        *reinterpret_cast<uint16_t*>(lo) = (uint16_t)c[i], *reinterpret_cast<uint16_t*>(hi) = (uint16_t)c[i + 4];
      }
    }
  }
}

// The same elements back.
template <int FMT, int D, bool KEY>
__device__ __forceinline__ void get(const uint8_t* chunk, int s, int u, f32x4& x, f32x4& y) {
  using L = KvLayout<FMT, D>;
  const Quads e = quads(KEY, u);
  float v[8];
  if constexpr (FMT == MR_KV_F16) {
    if constexpr (KEY) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(chunk + L::k_off(s, e.e0));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 p = unpack_f16(w[i]);
        v[2 * i] = p.x, v[2 * i + 1] = p.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = (float)*reinterpret_cast<const _Float16*>(chunk + L::v_off(s, e.e0 + i));
        v[i + 4] = (float)*reinterpret_cast<const _Float16*>(chunk + L::v_off(s, e.e1 + i));
      }
    }
  } else {
    const float sc = scale_value<FMT>(chunk[KEY ? L::ks_off(s, u >> 2) : L::vs_off(s, u >> 2)]);
    if constexpr (KEY && FMT == MR_KV_MXFP4) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(chunk + L::k_off(s, e.e0));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = sc * fp4_value(w >> (4 * i) & 15u);
    } else if constexpr (KEY) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(chunk + L::k_off(s, e.e0));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = int8_value(w[i >> 2] >> (8 * (i & 3)), sc);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FMT == MR_KV_MXFP4) {
          const uint32_t b = chunk[L::v_off(s, e.e0 + i)];
          v[i] = sc * fp4_value(b & 15u), v[i + 4] = sc * fp4_value(b >> 4);
        } else {
          v[i] = int8_value(chunk[L::v_off(s, e.e0 + i)], sc), v[i + 4] = int8_value(chunk[L::v_off(s, e.e1 + i)], sc);
        }
      }
    }
  }
  x = f32x4{v[0], v[1], v[2], v[3]}, y = f32x4{v[4], v[5], v[6], v[7]};
}

__device__ __forceinline__ uint64_t at(const Heads& h, int t, int head) { return (uint64_t)t * h.ts + (uint64_t)head * h.hs; }

// The values of tokens t + lo .. t + hi - 1 to slots lo .. hi - 1 of an LDS image of a chunk's values (codes, then
// scales); other slots get something. A thread has 4 adjacent slots: their codes of an element are adjacent too, a
// word (F16: two) of the image.
template <int FMT, int D>
__device__ __forceinline__ void put_run(uint8_t* image, const Heads& in, int t, int head, int lo, int hi) {
  using L = KvLayout<FMT, D>;
  constexpr int U = D / 8;
  for (int i = threadIdx.x; i < U * 16; i += 256) {
    const int u = i % U, s = 4 * (i / U);
    if (s + 4 <= lo || s >= hi) continue;  // the same for the lanes of a token
    const Quads e = quads(false, u);
    f32x4 x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t o = at(in, t + min(max(s + j, lo), hi - 1), head);
      x[j] = load4(in.p, in.dtype, o + e.e0), y[j] = load4(in.p, in.dtype, o + e.e1);
    }
    uint32_t w[8] = {}, w2[8] = {}, sc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t c[8];
      const int ex = quantise<FMT>(x[j], y[j], c);
      if (FMT != MR_KV_F16) sc |= scale_byte<FMT>(ex) << (8 * j);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (FMT == MR_KV_F16) (j < 2 ? w : w2)[k] |= c[k] << (16 * (j & 1));
        else if (FMT == MR_KV_MXFP4) w[k & 3] |= c[k] << (8 * j + (k & 4));
        else w[k] |= c[k] << (8 * j);
      }
    }
#pragma unroll
    for (int k = 0; k < (FMT == MR_KV_MXFP4 ? 4 : 8); ++k) {
      uint8_t* p = image + L::v_off(s, (k < 4 ? e.e0 : e.e1 - 4) + k) - L::kV;
      if (FMT == MR_KV_F16) *reinterpret_cast<u32x2*>(p) = u32x2{w[k], w2[k]};
      else *reinterpret_cast<uint32_t*>(p) = w[k];
    }
    if (FMT != MR_KV_F16 && (u & 3) == 0) *reinterpret_cast<uint32_t*>(image + L::vs_off(s, u >> 2) - L::kVs + L::kCodes) = sc;
  }
}
// Slots lo .. hi - 1 of the image to the chunk, by 4 adjacent slots; the ends, which share those bytes with tokens
// that others may be writing, one by one.
template <int FMT, int D>
__device__ __forceinline__ void store_piece(uint8_t* chunk, const uint8_t* image, int lo, int hi) {
  using L = KvLayout<FMT, D>;
  constexpr int E = FMT == MR_KV_F16 ? 2 : 1;  // bytes of a token's code
  for (int i = threadIdx.x * 4 * E; i < L::kCodes + L::kScales; i += 256 * 4 * E) {
    // v_off and vs_off the other way round: j, and the slot's bits 5 and 2 to 3
    const bool codes = i < L::kCodes;
    const int n = codes ? ((i >> 10) * 16 + (i & 15)) / E : i - L::kCodes, q = (n >> 3) / (codes && FMT != MR_KV_MXFP4 ? D / 16 : D / 32);
    const int s = 4 * (n & 4) + (codes ? 32 * q + 4 * (i >> 8 & 3) : 32 * (q & 1) + 4 * (q >> 1));
    if (s + 4 <= lo || s >= hi) continue;
    uint8_t* g = chunk + (codes ? L::kV + i : L::kVs + i - L::kCodes);
    const uint8_t* l = image + i;
    if (s >= lo && s + 4 <= hi) {
      if (FMT == MR_KV_F16) *reinterpret_cast<u32x2*>(g) = *reinterpret_cast<const u32x2*>(l);
      else *reinterpret_cast<uint32_t*>(g) = *reinterpret_cast<const uint32_t*>(l);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (s + j < lo || s + j >= hi) continue;
        if (FMT == MR_KV_F16) reinterpret_cast<uint16_t*>(g)[j] = reinterpret_cast<const uint16_t*>(l)[j];
        else g[j] = l[j];
      }
    }
  }
}
// And back: all 64 tokens, or tokens t + lo .. t + hi - 1, of the image or of the chunk itself.
template <int FMT, int D, bool WHOLE>
__device__ __forceinline__ void get_run(const uint8_t* codes, const uint8_t* scales, const Heads& out, int t, int head, int lo = 0,
                                        int hi = 64) {
  using L = KvLayout<FMT, D>;
  constexpr int U = D / 8;
  for (int i = threadIdx.x; i < U * 16; i += 256) {
    const int u = i % U, s = 4 * (i / U);
    if (!WHOLE && (s + 4 <= lo || s >= hi)) continue;
    const Quads e = quads(false, u);
    uint32_t w[8] = {}, w2[8] = {}, sc = 0;
#pragma unroll
    for (int k = 0; k < (FMT == MR_KV_MXFP4 ? 4 : 8); ++k) {
      const uint8_t* p = codes + L::v_off(s, (k < 4 ? e.e0 : e.e1 - 4) + k) - L::kV;
      if (FMT == MR_KV_F16) {
        const u32x2 a = *reinterpret_cast<const u32x2*>(p);
        w[k] = a.x, w2[k] = a.y;
      } else {
        w[k] = *reinterpret_cast<const uint32_t*>(p);
      }
    }
    if (FMT != MR_KV_F16) sc = *reinterpret_cast<const uint32_t*>(scales + L::vs_off(s, u >> 2) - L::kVs);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!WHOLE && (s + j < lo || s + j >= hi)) continue;
      const float f = FMT == MR_KV_F16 ? 1.f : scale_value<FMT>(sc >> (8 * j) & 0xFFu);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (FMT == MR_KV_F16) v[k] = h2f((j < 2 ? w : w2)[k] >> (16 * (j & 1)) & 0xFFFFu);
        else if (FMT == MR_KV_MXFP4) v[k] = f * fp4_value(w[k & 3] >> (8 * j + (k & 4)) & 15u);
        else v[k] = int8_value(w[k] >> (8 * j), f);
      }
      const uint64_t o = at(out, t + s + j, head);
      store4(out.p, out.dtype, o + e.e0, f32x4{v[0], v[1], v[2], v[3]});
      store4(out.p, out.dtype, o + e.e1, f32x4{v[4], v[5], v[6], v[7]});
    }
  }
}
// Moves 16 bytes a thread; the scales lie behind the keys' scales in the chunk, behind the codes in the image.
template <int FMT, int D, bool STORE>
__device__ __forceinline__ void move_image(uint8_t* chunk, uint8_t* image) {
  using L = KvLayout<FMT, D>;
  for (int i = threadIdx.x * 16; i < L::kCodes + L::kScales; i += 256 * 16) {
    u32x4* g = reinterpret_cast<u32x4*>(chunk + (i < L::kCodes ? L::kV + i : L::kVs + i - L::kCodes));
    u32x4* l = reinterpret_cast<u32x4*>(image + i);
    if (STORE) *g = *l;
    else *l = *g;
  }
}

// blockIdx: 64 tokens, head, keys or values. D / 8 lanes to a token.
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_kv_write(KvPages kv, Heads kin, Heads vin, int T, const int32_t* __restrict__ slots,
                                                  uint32_t* err) {
  using L = KvLayout<FMT, D>;
  constexpr int U = D / 8, N = 256 / U;  // lanes of a token, tokens at a time
  const int u = threadIdx.x % U, i0 = threadIdx.x / U, h = blockIdx.y, t0 = blockIdx.x * kWindow;
  if (blockIdx.z == 0) {
    const Quads e = quads(true, u);
#pragma unroll 4
    for (int i = i0; i < kWindow; i += N) {
      if (t0 + i >= T) break;
      int s = 0;
      uint8_t* chunk = find(kv, slots[t0 + i], h, err, s);
      if (!chunk) continue;  // the same for the lanes of a token
      const uint64_t o = at(kin, t0 + i, h);
      put<FMT, D, true>(chunk, s, u, load4(kin.p, kin.dtype, o + e.e0), load4(kin.p, kin.dtype, o + e.e1));
    }
    return;
  }
  __shared__ int sl[192];
  __shared__ uint64_t breaks[3];
  __shared__ __attribute__((aligned(16))) uint8_t image[L::kCodes + L::kScales];
  const Quads e = quads(false, u);
  const Runs r = find_runs(kv, slots, T, t0, sl, breaks);
  for (uint64_t todo = r.start | r.piece; todo; todo &= todo - 1) {
    const int b = __ffsll((unsigned long long)todo) - 1;
    const bool whole = r.start >> b & 1;
    int lo;
    uint8_t* chunk = find(kv, sl[63 + b], h, err, lo);
    const int hi = whole ? 64 : lo + piece_length(r.end, b);
    put_run<FMT, D>(image, vin, t0 + b - lo, h, lo, hi);
    __syncthreads();
    if (whole) move_image<FMT, D, true>(chunk, image);
    else store_piece<FMT, D>(chunk, image, lo, hi);
    __syncthreads();
  }
  for (int i = i0; i < kWindow; i += N) {
    if (!(r.single >> i & 1)) continue;
    int s = 0;
    uint8_t* chunk = find(kv, sl[63 + i], h, err, s);
    if (!chunk) continue;
    const uint64_t o = at(vin, t0 + i, h);
    put<FMT, D, false>(chunk, s, u, load4(vin.p, vin.dtype, o + e.e0), load4(vin.p, vin.dtype, o + e.e1));
  }
}

template <int FMT, int D>
__global__ __launch_bounds__(256) void k_kv_read(KvPages kv, int T, const int32_t* __restrict__ slots, Heads kout, Heads vout,
                                                 uint32_t* err) {
  using L = KvLayout<FMT, D>;
  constexpr int U = D / 8, N = 256 / U;
  const int u = threadIdx.x % U, i0 = threadIdx.x / U, h = blockIdx.y, t0 = blockIdx.x * kWindow;
  if (blockIdx.z == 0) {
    if (!kout.p) return;
    const Quads e = quads(true, u);
#pragma unroll 4
    for (int i = i0; i < kWindow; i += N) {
      if (t0 + i >= T) break;
      int s = 0;
      const uint8_t* chunk = find(kv, slots[t0 + i], h, err, s);
      f32x4 x = {0, 0, 0, 0}, y = x;
      if (chunk) get<FMT, D, true>(chunk, s, u, x, y);
      const uint64_t o = at(kout, t0 + i, h);
      store4(kout.p, kout.dtype, o + e.e0, x), store4(kout.p, kout.dtype, o + e.e1, y);
    }
    return;
  }
  if (!vout.p) return;
  __shared__ int sl[192];
  __shared__ uint64_t breaks[3];
  __shared__ __attribute__((aligned(16))) uint8_t image[L::kCodes + L::kScales];
  const Quads e = quads(false, u);
  const Runs r = find_runs(kv, slots, T, t0, sl, breaks);
  for (uint64_t todo = r.start; todo; todo &= todo - 1) {
    const int b = __ffsll((unsigned long long)todo) - 1;
    int s;
    move_image<FMT, D, false>(find(kv, sl[63 + b], h, err, s), image);
    __syncthreads();
    get_run<FMT, D, true>(image, image + L::kCodes, vout, t0 + b, h);
    __syncthreads();
  }
  for (uint64_t todo = r.piece; todo; todo &= todo - 1) {
    const int b = __ffsll((unsigned long long)todo) - 1;
    int lo;
    const uint8_t* chunk = find(kv, sl[63 + b], h, err, lo);
    get_run<FMT, D, false>(chunk + L::kV, chunk + L::kVs, vout, t0 + b - lo, h, lo, lo + piece_length(r.end, b));
  }
  // the others, and zeros for tokens without a slot
  for (int i = i0; i < kWindow; i += N) {
    if (t0 + i >= T) break;
    const int slot = sl[63 + i];
    if (slot >= 0 && !(r.single >> i & 1)) continue;
    int s = 0;
    const uint8_t* chunk = find(kv, slot, h, err, s);
    f32x4 x = {0, 0, 0, 0}, y = x;
    if (chunk) get<FMT, D, false>(chunk, s, u, x, y);
    const uint64_t o = at(vout, t0 + i, h);
    store4(vout.p, vout.dtype, o + e.e0, x), store4(vout.p, vout.dtype, o + e.e1, y);
  }
}

template <int FMT>
hipError_t write_fmt(const Launch& K, const KvPages& kv, uint32_t D, const Heads& k, const Heads& v, uint32_t T,
                     const int32_t* slots, uint32_t* err) {
  const dim3 g((T + kWindow - 1) / kWindow, kv.n_heads, 2);
  if (D == 64) hipLaunchKernelGGL((k_kv_write<FMT, 64>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  if (D == 128) hipLaunchKernelGGL((k_kv_write<FMT, 128>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  if (D == 256) hipLaunchKernelGGL((k_kv_write<FMT, 256>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  return hipGetLastError();
}

template <int FMT>
hipError_t read_fmt(const Launch& K, const KvPages& kv, uint32_t D, uint32_t T, const int32_t* slots, const Heads& k,
                    const Heads& v, uint32_t* err) {
  const dim3 g((T + kWindow - 1) / kWindow, kv.n_heads, 2);
  if (D == 64) hipLaunchKernelGGL((k_kv_read<FMT, 64>), g, dim3(256), 0, K.s, kv, (int)T, slots, k, v, err);
  if (D == 128) hipLaunchKernelGGL((k_kv_read<FMT, 128>), g, dim3(256), 0, K.s, kv, (int)T, slots, k, v, err);
  if (D == 256) hipLaunchKernelGGL((k_kv_read<FMT, 256>), g, dim3(256), 0, K.s, kv, (int)T, slots, k, v, err);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& k, const Heads& v,
                           uint32_t T, const int32_t* slots, uint32_t* err) {
  ProfScope ps(K, "kv_write");
  if (format == MR_KV_F16) return write_fmt<MR_KV_F16>(K, kv, D, k, v, T, slots, err);
  if (format == MR_KV_MXINT8) return write_fmt<MR_KV_MXINT8>(K, kv, D, k, v, T, slots, err);
  return write_fmt<MR_KV_MXFP4>(K, kv, D, k, v, T, slots, err);
}

hipError_t launch_kv_read(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, uint32_t T,
                          const int32_t* slots, const Heads& k, const Heads& v, uint32_t* err) {
  ProfScope ps(K, "kv_read");
  if (format == MR_KV_F16) return read_fmt<MR_KV_F16>(K, kv, D, T, slots, k, v, err);
  if (format == MR_KV_MXINT8) return read_fmt<MR_KV_MXINT8>(K, kv, D, T, slots, k, v, err);
  return read_fmt<MR_KV_MXFP4>(K, kv, D, T, slots, k, v, err);
}

}  // namespace mr
