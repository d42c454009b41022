// The consumer of the q|k|v projection with head norms and several position axes.
#pragma once

#include "fi_common.h"
#include "fi_device.h"

namespace fi {

struct QkvNormArgs {
  const float* parts;  // [splits][tokens][(hq + 2 hkv) * D]
  int splits;
  const float* bias_q;  // each may be null
  const float* bias_k;
  const float* bias_v;
  const float* q_norm;  // [D], or null: no norm
  const float* k_norm;
  float eps;
  const int* positions;  // [num_axes][tokens]
  int num_axes;
  // two bits a rotary pair, sixteen pairs a word: the axis whose position turns it.  Four names, not an
  // array: indexed by a lane it would be copied to scratch memory
  uint32_t pair_axes0, pair_axes1, pair_axes2, pair_axes3;
  const float* cos_t;     // [max_positions][rotary_dims / 2]
  const float* sin_t;
  int rotary_dims;
  int max_positions;
  const int64_t* slots;
  void* k_cache;
  void* v_cache;
  int64_t pool_slots;
  size_t code_bytes;  // 4-bit pools: where an array's scales begin
  int block_size;
  int tokens;
  FastDiv chunks;  // workgroups a token
  int hq, hkv;
  float* q_out;
  uint32_t* faults;
};

// Checks the arguments and launches the consumer; `name` is the entry point's.  pair_axes (host,
// rotary_dims / 2 entries) may be null with one axis.
int32_t qkv_norm_rope_append(fi_context* ctx, const char* name, QkvNormArgs a, int32_t head_dim, int32_t kv_dtype,
                             int32_t num_blocks, const int32_t* pair_axes);

}  // namespace fi
