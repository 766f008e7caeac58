// mr_kv_operand.h -- a chunk of the paged cache as operands of 16x16x32 matrix instructions, for the kernels that
// attend over the cache.
#pragma once

#include "mr_attn_device.h"

namespace mr {

namespace {

constexpr float kLargest = 0x1.fffffep127f;
// The largest weight is 2^kLift. Weights are rounded to f16 for the second product: ones down to 2^-28 of the largest keep
// all of its bits, and what is lost of smaller ones is 2^-39 of it at most. With the largest at one, a tail of keys
// 18 below a first one that has no value was lost (1000 keys: 96% off).
constexpr float kLift = 14.f;

// The sum over the wave in every lane, by the lane swaps and row moves of wave_sum_fast.
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = a[0] + a[1];
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = b[0] + b[1];
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false);  // row_ror:8
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false);  // row_ror:4
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);   // l ^ 2
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);  // l ^ 1
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two of an MXFP4 word's codes (byte `sel`) as f16, times the power of two in the exponent field of sc.
template <int SEL>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, uint32_t sc) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, bits_f32(sc), SEL));
}
// Byte `sel` of w in the exponent field; the conversion takes no notice of the other bits.
__device__ __forceinline__ uint32_t exp_bits(uint32_t w, int sel) { return sel == 3 ? w >> 1 : w << (23 - 8 * sel); }

// Two MXINT8 codes as f16: 0x6400 | u is 1024 + u.
__device__ __forceinline__ f16x2 int8_pair(uint32_t codes, int pair) {
  const uint32_t w = __builtin_amdgcn_perm(0x64646464u, codes, pair ? 0x07030602u : 0x05010400u);
  return __builtin_bit_cast(f16x2, w) - f16x2{(_Float16)1152.f, (_Float16)1152.f};
}

// Two tiles of 16 elements of 8 tokens from their codes (MXFP4: a word for 4 tokens of both; MXINT8: two words for each tile) and the
// tokens' scale bytes.
template <int FMT>
__device__ __forceinline__ void value_pair(const uint32_t (&c)[FMT / 2], uint32_t s0, uint32_t s1, u32x4& lo, u32x4& hi) {
  if constexpr (FMT == MR_KV_MXFP4) {
    const uint32_t p[8] = {fp4_pair<0>(c[0], exp_bits(s0, 0)), fp4_pair<1>(c[0], exp_bits(s0, 1)),
                           fp4_pair<2>(c[0], exp_bits(s0, 2)), fp4_pair<3>(c[0], exp_bits(s0, 3)),
                           fp4_pair<0>(c[1], exp_bits(s1, 0)), fp4_pair<1>(c[1], exp_bits(s1, 1)),
                           fp4_pair<2>(c[1], exp_bits(s1, 2)), fp4_pair<3>(c[1], exp_bits(s1, 3))};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = __builtin_amdgcn_perm(p[2 * j + 1], p[2 * j], 0x05040100u);
      hi[j] = __builtin_amdgcn_perm(p[2 * j + 1], p[2 * j], 0x07060302u);
    }
  } else if constexpr (FMT == MR_KV_MXINT8) {
    // scale bytes j, j + 1 as the high bytes of two f16
    const f16x2 e[4] = {__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0u, s0, 0x010C000Cu)),
                        __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0u, s0, 0x030C020Cu)),
                        __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0u, s1, 0x010C000Cu)),
                        __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0u, s1, 0x030C020Cu))};
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        (x ? hi : lo)[j] = __builtin_bit_cast(uint32_t, int8_pair(c[2 * x + (j >> 1)], j & 1) * e[j]);
  }
}

template <int FMT, int D>
struct Chunk {
  static constexpr int NP = D * FMT / 128;  // 16-byte pieces a lane has of the keys, and of the values
  static constexpr int NKS = FMT == MR_KV_F16 ? 0 : D == 256 ? 2 : 1, NVS = FMT == MR_KV_F16 ? 0 : D / 32;
  u32x4 k[NP], v[NP];
  uint32_t ks[NKS ? NKS : 1];
  u32x4 vs[NVS ? NVS : 1];  // [G][block][j] bytes: D / 2 in all

  __device__ __forceinline__ void load_k(const uint8_t* p, int lane) {
    using L = KvLayout<FMT, D>;
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = *reinterpret_cast<const u32x4*>(p + i * 1024 + lane * 16);
    if constexpr (FMT != MR_KV_F16) {
      const int m = lane & 15, g = lane >> 4;
#pragma unroll
      for (int i = 0; i < NKS; ++i) {
        const int blk = D == 64 ? g >> 1 : D == 128 ? g : 2 * g + i;
        ks[i] = *reinterpret_cast<const uint32_t*>(p + L::kKs + (blk * 16 + m) * 4);
      }
    }
  }
  // The values of group G (32 tokens).
  __device__ __forceinline__ void load_v(const uint8_t* p, int lane, int G) {
    using L = KvLayout<FMT, D>;
#pragma unroll
    for (int i = G * NP / 2; i < (G + 1) * NP / 2; ++i) v[i] = *reinterpret_cast<const u32x4*>(p + L::kV + i * 1024 + lane * 16);
    if constexpr (FMT != MR_KV_F16) {
#pragma unroll
      for (int i = G * NVS / 2; i < (G + 1) * NVS / 2; ++i) vs[i] = *reinterpret_cast<const u32x4*>(p + L::kVs + (lane >> 4) * (D / 2) + 16 * i);
    }
  }
  // Elements 8 i .. 8 i + 7 of the lane's quarter of key 16 t + m.
  __device__ __forceinline__ u32x4 key(int t, int i) const {
    if constexpr (FMT == MR_KV_F16) return k[t * (D / 32) + i];
    const uint32_t s = ks[D == 256 ? i >> 2 : 0];
    if constexpr (FMT == MR_KV_MXFP4) {
      const int w = t * (D / 32) + i;
      const uint32_t c = k[w >> 2][w & 3], e = exp_bits(s, t);
      return u32x4{fp4_pair<0>(c, e), fp4_pair<1>(c, e), fp4_pair<2>(c, e), fp4_pair<3>(c, e)};
    } else {
      const int w = 2 * (t * (D / 32) + i);
      const uint32_t c0 = k[w >> 2][w & 3], c1 = k[w >> 2][(w & 3) + 1];
      const uint32_t b = s >> (8 * t) & 0xFFu;
      const f16x2 e = __builtin_bit_cast(f16x2, b << 8 | b << 24);
      return u32x4{__builtin_bit_cast(uint32_t, int8_pair(c0, 0) * e), __builtin_bit_cast(uint32_t, int8_pair(c0, 1) * e),
                   __builtin_bit_cast(uint32_t, int8_pair(c1, 0) * e), __builtin_bit_cast(uint32_t, int8_pair(c1, 1) * e)};
    }
  }
  // Element m of tiles 2 b and 2 b + 1 (of 16) for the 8 tokens of the lane in group G.
  __device__ __forceinline__ void value(int G, int b, u32x4& lo, u32x4& hi) const {
    if constexpr (FMT == MR_KV_F16) {
      lo = v[G * (D / 16) + 2 * b], hi = v[G * (D / 16) + 2 * b + 1];
      return;
    }
    const int sw = 2 * (G * (D / 32) + b), w = FMT == MR_KV_MXFP4 ? sw : 2 * sw;
    uint32_t codes[FMT / 2];
#pragma unroll
    for (int i = 0; i < FMT / 2; ++i) codes[i] = v[(w + i) >> 2][(w + i) & 3];
    value_pair<FMT>(codes, vs[sw >> 2][sw & 3], vs[sw >> 2][(sw & 3) + 1], lo, hi);
  }
};

}  // namespace

}  // namespace mr
