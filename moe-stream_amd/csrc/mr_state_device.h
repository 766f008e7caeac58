// mr_state_device.h -- where packed sequences lie and which states are theirs, for the kernels over kept states.
#pragma once

#include "mr_attn_device.h"
#include "mr_state.h"

namespace mr {

// Tiles of 1 << bits rows (mul rows to a token) are numbered so that sequence s has those from
// (cu[s] mul >> bits) + s on: room for its rows wherever they begin, and for one tile of a sequence without
// rows. The last sequence whose tiles begin at `tile` or before, 64 candidates at a time; all 64 lanes active.
__device__ __forceinline__ uint32_t first_tile(const int32_t* cu, int n_rows, uint32_t s, uint32_t mul, int bits) {
  return (uint32_t)((uint64_t)min(max(cu[s], 0), n_rows) * mul >> bits) + s;
}
__device__ __forceinline__ uint32_t find_seq(const int32_t* cu, uint32_t n_seqs, int n_rows, uint32_t mul, int bits,
                                             uint32_t tile) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = 0, n = n_seqs;
  for (;;) {
    const uint32_t step = (n + 63) / 64, at = lane * step;
    const int c = __popcll(__ballot(at < n && first_tile(cu, n_rows, lo + at, mul, bits) <= tile));
    const uint32_t past = c > 0 ? (uint32_t)(c - 1) * step : 0;
    lo += past, n = min(step, n - past);
    if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
  }
}

// Rows [q0, q1) of sequence s, clamped into the call's.
__device__ __forceinline__ void rows_of(const int32_t* cu, int n_rows, uint32_t s, int& q0, int& q1) {
  q0 = min(max(cu[s], 0), n_rows);
  q1 = max(q0, min(max(cu[s + 1], 0), n_rows));
}

// Reports offsets out of order or range; by every thread of one workgroup.
__device__ __forceinline__ void check_offsets(const int32_t* cu, uint32_t n_seqs, int n_rows, uint32_t* err, uint32_t kind) {
  for (uint32_t s = threadIdx.x; s < n_seqs; s += blockDim.x) {
    const int x = cu[s], y = cu[s + 1];
    if (x < 0 || y < x || y > n_rows) note_error(err, kind);
  }
}

// The slot in array `slots` for sequence s, -1 for none.
__device__ __forceinline__ int slot_of(const Sequences& q, const int32_t* slots, uint32_t s) {
  if (!slots) return -1;
  const int x = slots[s];
  if (x >= 0 && (uint32_t)x < q.n_slots) return x;
  if (x >= 0) note_error(q.err, kErrState);
  return -1;
}

}  // namespace mr
