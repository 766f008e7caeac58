// mr_state.h -- objects and launchers behind include/moe_rocm_state.h.
#pragma once

#include "../../include/moe_rocm_state.h"
#include "mr_attn.h"

struct mr_delta {
  mr_ctx* ctx = nullptr;
  mr_delta_desc d{};
};

namespace mr {

// mr_rows with its default filled in.
struct RowsOf {
  void* p;
  uint32_t dtype, width;
  uint64_t stride;
};

// Packed sequences over states: offsets, and where each state comes from and goes to.
struct Sequences {
  const int32_t* cu;
  uint32_t n_seqs;
  int n_rows;
  float* states;
  uint32_t n_slots;
  const int32_t *source, *target;
  uint32_t* err;
};

struct DeltaShape {
  uint32_t key_heads, value_heads, key_dim, value_dim;
  float scale, unit_eps;
  uint64_t gate_stride;
  const float *a_log, *dt_bias;
};

hipError_t launch_attn_extend(const Launch& K, const KvPages& kv, uint32_t format, uint32_t D, const Heads& q, uint32_t nq,
                              uint32_t n_seqs, const int32_t* cu, const int32_t* len, const int32_t* table,
                              uint32_t max_pages, const AttnOpts& o, const Heads& out, uint32_t* err, float* scratch,
                              int n_cu);
// Scratch of launch_attn_extend, at any size.
uint64_t attn_extend_scratch_bytes();
hipError_t launch_causal_conv(const Launch& K, const RowsOf& x, const float* w, uint32_t taps, const float* bias, bool silu,
                              const Sequences& s, const RowsOf& out);
hipError_t launch_delta_rule(const Launch& K, const DeltaShape& d, const Heads& q, const Heads& k, const Heads& v,
                             const float* decay, const float* beta, const Sequences& s, const Heads& out, void* scratch);
// Workspace of launch_delta_rule, at any size.
uint64_t delta_scratch_bytes();

}  // namespace mr
