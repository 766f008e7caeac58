// mr_attn_device.h -- device helpers of the attention-side kernels.
#pragma once

#include "mr_attn.h"
#include "mr_device.h"

namespace mr {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Two f32 to adjacent f16 (bf16), rounded to nearest even.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f16x2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ f32x2 unpack_f16(uint32_t w) {
  const f16x2 v = __builtin_bit_cast(f16x2, w);
  return f32x2{(float)v.x, (float)v.y};
}
__device__ __forceinline__ f32x2 unpack_bf16(uint32_t w) { return f32x2{bits_f32(w << 16), bits_f32(w & 0xFFFF0000u)}; }

// s + the two f16 (bf16) of w: subnormal ones count too. The weights' sum is taken of the rounded weights, so that
// what rounding one does to the sum of values it does to the divisor as well: a row on one key is exact.
__device__ __forceinline__ float add_f16(uint32_t w, float s) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.f, (_Float16)1.f}, s, false);
}
__device__ __forceinline__ float add_bf16(uint32_t w, float s) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)1.f, (__bf16)1.f}, s, false);
}

// Four adjacent elements at element offset i of an array of type `dtype` (the same for all lanes).
__device__ __forceinline__ f32x4 load4(const void* p, uint32_t dtype, uint64_t i) {
  if (dtype == MR_F32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + i);
  const f32x2 a = dtype == MR_F16 ? unpack_f16(w.x) : unpack_bf16(w.x);
  const f32x2 b = dtype == MR_F16 ? unpack_f16(w.y) : unpack_bf16(w.y);
  return f32x4{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ void store4(void* p, uint32_t dtype, uint64_t i, f32x4 v) {
  if (dtype == MR_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
    return;
  }
  const u32x2 w = dtype == MR_F16 ? u32x2{pack_f16(v.x, v.y), pack_f16(v.z, v.w)}
                                  : u32x2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + i) = w;
}

// A head's sink in powers of two; a finite one stays finite. No sinks: -infinity.
__device__ __forceinline__ float sink_of(const float* sinks, uint32_t h) {
  const float s = sinks ? sinks[h] : -INFINITY;
  return (s > 0x1p127f && s < INFINITY ? 0x1p127f : s) * 1.44269504088896340736f;
}

// Sets the error word of a kind; it is the host's memory.
__device__ __forceinline__ void note_error(uint32_t* err, uint32_t kind) {
  __hip_atomic_store(err + kind, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// The sum of lanes 0 .. l in lane l: shifts inside the rows of 16 lanes, then row ends broadcast to the rows after
// them. All 64 lanes active.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1 and 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2 and 3
  return v;
}

// Value of a doubled e2m1 code (0..15), halved on use: {0,1,2,3,4,6,8,12}.
__device__ __forceinline__ float fp4_value(uint32_t c) {
  const uint32_t m = c & 7u;
  const float a = m < 5u ? 0.5f * (float)m : (m == 5u ? 3.f : m == 6u ? 4.f : 6.f);
  return c & 8u ? -a : a;
}
// 2^e of a scale byte.
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t b) {
  return FMT == MR_KV_MXFP4 ? bits_f32(b << 23) : h2f(b << 8);
}

}  // namespace mr
