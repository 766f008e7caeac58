// mr_attn.h -- objects and launchers behind include/moe_rocm_attn.h, and the cache's layout.
#pragma once

#include <vector>

#include "../../include/moe_rocm_attn.h"
#include "mr_internal.h"

struct mr_rope {
  mr_ctx* ctx = nullptr;
  mr_rope_desc d{};
  std::vector<double> freq;  // radians per position
  double* d_turns = nullptr; // device: freq / (2 pi)
  float mul = 1.f;
};

struct mr_kv {
  mr_ctx* ctx = nullptr;
  mr_kv_desc d{};
  uint8_t* base = nullptr;
  uint64_t bytes = 0;
};

namespace mr {

// Of the context's attention error words: which kind of device index was out of range.
constexpr uint32_t kErrSlot = 0, kErrLength = 1, kErrPage = 2, kErrOffset = 3;
static_assert(kErrOffset + 1 == kAttnErrWords, "a word for each kind");

// mr_heads with its defaults filled in.
struct Heads {
  void* p;
  uint32_t dtype, n;
  uint64_t ts, hs;
};

// Cache layout. A page holds, for each head in turn, page_size / 64 chunks of 64 tokens; a chunk is
// laid out for the lanes of the attention kernel (lane = 16 g + m), so that each reads 16 adjacent
// bytes at a time, 1 KiB per wave, and no element has to change its lane:
//   keys    [piece][lane][16 B]: lane (m, g) has, of the keys 16 t + m for t = 0..3 in turn, the
//           elements g * D/4 .. (g + 1) * D/4 - 1 (MXFP4: two to a byte, the even one low)
//   values  [piece][lane][16 B]: slot j = 0..7 of lane (m, g) stands for token 32 G + 4 g + j (j < 4) or
//           32 G + 16 + 4 g + j - 4, for G = 0, 1 in turn; the elements are, in turn,
//             MXFP4   blocks of 32: a byte for each j, element 32 b + m low, 32 b + 16 + m high
//             others  tiles of 16: element 16 t + m for each j
//   An MXINT8 code is stored with 128 added, the form that turns into f16 in the fewest instructions.
//   key scales    [block][m][t], value scales [g][G][block][j]; a byte each, none for F16. The byte is
//           e + 127 for MXFP4 (the scale operand of the conversion), the high byte of 2^e in f16 for
//           MXINT8 (the factor of the packed f16 product).
template <int FMT, int D>
struct KvLayout {
  static constexpr int kCodes = 64 * D * FMT / 8;
  static constexpr int kScales = FMT == MR_KV_F16 ? 0 : 64 * (D / 32);
  static constexpr int kV = kCodes, kKs = 2 * kCodes, kVs = 2 * kCodes + kScales;
  static constexpr int kChunk = 2 * kCodes + 2 * kScales;
  // Byte of element d of the chunk's token s.
  static __host__ __device__ __forceinline__ int k_off(int s, int d) {
    const int lane = 16 * (d / (D / 4)) + (s & 15), in = ((s >> 4) * (D / 4) + d % (D / 4)) * FMT / 8;
    return (in >> 4) * 1024 + lane * 16 + (in & 15);
  }
  static __host__ __device__ __forceinline__ int v_off(int s, int d) {
    const int lane = 16 * ((s >> 2) & 3) + (d & 15), G = s >> 5, j = ((s >> 2) & 4) + (s & 3);
    const int in = FMT == MR_KV_MXFP4 ? (G * (D / 32) + (d >> 5)) * 8 + j : ((G * (D / 16) + (d >> 4)) * 8 + j) * (FMT / 8);
    return kV + (in >> 4) * 1024 + lane * 16 + (in & 15);
  }
  static __host__ __device__ __forceinline__ int ks_off(int s, int b) { return kKs + (b * 16 + (s & 15)) * 4 + (s >> 4); }
  static __host__ __device__ __forceinline__ int vs_off(int s, int b) {
    return kVs + ((((s >> 2) & 3) * 2 + (s >> 5)) * (D / 32) + b) * 8 + ((s >> 2) & 4) + (s & 3);
  }
};

inline uint64_t kv_chunk_bytes(uint32_t format, uint32_t D) {
  return 64ull * D * format / 8 * 2 + (format == MR_KV_F16 ? 0 : 2 * 64ull * (D / 32));
}

// The pages as the kernels see them.
struct KvPages {
  uint8_t* base;
  uint32_t n_pages, page_shift, n_heads;
  uint64_t chunk;  // bytes of a chunk
  // Chunk (page, head, c).
  __host__ __device__ __forceinline__ uint8_t* at(uint32_t page, uint32_t head, uint32_t c) const {
    return base + ((((uint64_t)page * n_heads + head) << (page_shift - 6)) + c) * chunk;
  }
};

struct AttnOpts {
  float scale;
  uint32_t window;  // 0: none
  const float* sinks;
};

constexpr int kPrefillRows = 128;  // query rows of a prefill tile, times the heads side by side

hipError_t launch_qk_norm_rope(const Launch& K, const mr_rope& r, const Heads& q, const Heads& k, const float* qn,
                               const float* kn, float eps, const int32_t* pos, uint32_t T, const Heads& qo,
                               const Heads& ko);
hipError_t launch_kv_write(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& k, const Heads& v,
                           uint32_t T, const int32_t* slots, uint32_t* err);
hipError_t launch_kv_read(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, uint32_t T,
                          const int32_t* slots, const Heads& k, const Heads& v, uint32_t* err);
hipError_t launch_attn_decode(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& q, uint32_t B,
                              const int32_t* len, const int32_t* table, uint32_t max_pages, const AttnOpts& o,
                              const Heads& out, uint32_t* err, float* scratch, int n_cu);
// Scratch of launch_attn_decode, at any size.
uint64_t attn_decode_scratch_bytes();
hipError_t launch_attn_prefill(const Launch& K, uint32_t D, const Heads& q, uint32_t nq, const Heads& k, const Heads& v,
                               uint32_t nk, uint32_t n_seqs, const int32_t* cu_q, const int32_t* cu_k, const AttnOpts& o,
                               const Heads& out, uint32_t* err);

}  // namespace mr
