// mr_kv.hip -- the paged cache of keys and values: quantising what is written, and reading it back.
//
// A block of 32 elements is stored as codes * 2^e. e comes from the bits of the largest magnitude and
// x * 2^-e is exact, so the codes are the nearest ones, with no rounding before the last.
#include "mr_attn_device.h"

namespace mr {

namespace {

__device__ __forceinline__ float finite_or_inf(float x) { return x == x ? x : 0.f; }

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
  if (FMT == MR_KV_MXINT8) return (uint32_t)(int)rintf(fminf(fmaxf(y, -127.f), 127.f)) & 0xFFu;
  const float a = fabsf(y);
  const uint32_t c = (uint32_t)(a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
  return y < 0.f && c ? c | 8u : c;
}

// Token s of the chunk that slot `slot` lies in; nullptr (and the error bit) for a slot out of range.
__device__ __forceinline__ uint8_t* find(const KvPages& kv, int slot, uint32_t head, uint32_t* err, int& s) {
  const uint32_t page = (uint32_t)slot >> kv.page_shift;
  if (slot < 0) return nullptr;
  if (page >= kv.n_pages) {
    atomicOr(err, kErrSlot);
    return nullptr;
  }
  s = slot & 63;
  return kv.at(page, head, ((uint32_t)slot & ((1u << kv.page_shift) - 1u)) >> 6);
}

constexpr int kWriteTokens = 64;  // tokens of a workgroup

// blockIdx: 64 tokens, head, keys or values. D/8 lanes to a token; a lane has 8 elements as two quads:
// adjacent ones for keys, 32 b + 4 w and 32 b + 16 + 4 w for values (the halves of a byte).
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_kv_write(KvPages kv, Heads kin, Heads vin, int T, const int32_t* __restrict__ slots,
                                                  uint32_t* err) {
  using L = KvLayout<FMT, D>;
  constexpr int U = D / 8;
  const bool key = blockIdx.z == 0;
  const Heads in = key ? kin : vin;
  const int u = threadIdx.x % U, h = blockIdx.y;
  const int e0 = key ? 8 * u : 32 * (u >> 2) + 4 * (u & 3), e1 = key ? e0 + 4 : e0 + 16;
  const int t1 = min(T, (int)(blockIdx.x + 1) * kWriteTokens);
  for (int t = blockIdx.x * kWriteTokens + threadIdx.x / U; t < t1; t += 256 / U) {
    int s = 0;
    uint8_t* chunk = find(kv, slots[t], h, err, s);
    if (!chunk) continue;  // the same for the U lanes of a token
    const uint64_t o = (uint64_t)t * in.ts + (uint64_t)h * in.hs;
    const f32x4 x = load4(in.p, in.dtype, o + e0), y = load4(in.p, in.dtype, o + e1);
    float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite_or_inf(v[i]), top = fmaxf(top, fabsf(v[i]));
    if (FMT == MR_KV_F16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -65504.f), 65504.f);
      if (key) {
        *reinterpret_cast<u32x4*>(chunk + L::k_off(s, e0)) =
            u32x4{pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7])};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<_Float16*>(chunk + L::v_off(s, (i < 4 ? e0 : e1 - 4) + i)) = (_Float16)v[i];
      }
      continue;
    }
    top = fmaxf(top, __shfl_xor(top, 1, kWave));
    top = fmaxf(top, __shfl_xor(top, 2, kWave));
    const int e = block_exp<FMT>(top);
    const float inv = bits_f32((uint32_t)(127 - e) << 23);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code<FMT>(v[i] * inv);
    if ((u & 3) == 0) chunk[key ? L::ks_off(s, u >> 2) : L::vs_off(s, u >> 2)] = (uint8_t)scale_byte<FMT>(e);
    if (key) {
      if (FMT == MR_KV_MXFP4) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= c[i] << (4 * i);
        *reinterpret_cast<uint32_t*>(chunk + L::k_off(s, e0)) = w;
      } else {
        *reinterpret_cast<u32x2*>(chunk + L::k_off(s, e0)) =
            u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (FMT == MR_KV_MXFP4) {
          chunk[L::v_off(s, e0 + i)] = (uint8_t)(c[i] | c[i + 4] << 4);
        } else {
          chunk[L::v_off(s, e0 + i)] = (uint8_t)c[i];
          chunk[L::v_off(s, e1 + i)] = (uint8_t)c[i + 4];
        }
      }
    }
  }
}

template <int FMT, int D>
__global__ __launch_bounds__(256) void k_kv_read(KvPages kv, int T, const int32_t* __restrict__ slots, Heads kout, Heads vout,
                                                 uint32_t* err) {
  constexpr int U = D / 8;
  const bool key = blockIdx.z == 0;
  const Heads out = key ? kout : vout;
  if (!out.p) return;
  const int u = threadIdx.x % U, h = blockIdx.y;
  const int e0 = key ? 8 * u : 32 * (u >> 2) + 4 * (u & 3), e1 = key ? e0 + 4 : e0 + 16;
  const int t1 = min(T, (int)(blockIdx.x + 1) * kWriteTokens);
  for (int t = blockIdx.x * kWriteTokens + threadIdx.x / U; t < t1; t += 256 / U) {
    int s = 0;
    const uint8_t* chunk = find(kv, slots[t], h, err, s);
    f32x4 x = {0, 0, 0, 0}, y = x;
    if (chunk) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = kv_value<FMT, D>(chunk, key, s, e0 + i);
        y[i] = kv_value<FMT, D>(chunk, key, s, e1 + i);
      }
    }
    const uint64_t o = (uint64_t)t * out.ts + (uint64_t)h * out.hs;
    store4(out.p, out.dtype, o + e0, x);
    store4(out.p, out.dtype, o + e1, y);
  }
}

template <int FMT>
hipError_t write_fmt(const Launch& K, const KvPages& kv, uint32_t D, const Heads& k, const Heads& v, uint32_t T,
                     const int32_t* slots, uint32_t* err) {
  const dim3 g((T + kWriteTokens - 1) / kWriteTokens, kv.n_heads, 2);
  if (D == 64) hipLaunchKernelGGL((k_kv_write<FMT, 64>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  if (D == 128) hipLaunchKernelGGL((k_kv_write<FMT, 128>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  if (D == 256) hipLaunchKernelGGL((k_kv_write<FMT, 256>), g, dim3(256), 0, K.s, kv, k, v, (int)T, slots, err);
  return hipGetLastError();
}

template <int FMT>
hipError_t read_fmt(const Launch& K, const KvPages& kv, uint32_t D, uint32_t T, const int32_t* slots, const Heads& k,
                    const Heads& v, uint32_t* err) {
  const dim3 g((T + kWriteTokens - 1) / kWriteTokens, kv.n_heads, 2);
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
