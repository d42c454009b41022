// Launches over 4-bit KV pools, called by the pool entry points once their arguments are checked.
#pragma once

#include "fi_common.h"

namespace fi {

struct DecodeArgs;
struct PrefillArgs;

// What every entry point requires of a 4-bit pool beyond a pool's own checks: head_dim 32, 64 or
// 128 (whole groups, and the head dims of the attention kernels) and 16-byte aligned arrays.
inline int32_t check_fp4_pool(const char* name, const void* k_cache, const void* v_cache, int32_t head_dim) {
  FI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, FI_ERR_UNSUPPORTED,
             std::string(name) + ": a 4-bit pool needs head_dim 32, 64 or 128");
  FI_REQUIRE(((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0,
             FI_ERR_INVALID_LAYOUT, std::string(name) + ": a 4-bit pool must be 16-byte aligned (vector accesses)");
  return FI_OK;
}

int32_t kv_append_fp4(fi_context* ctx, const float* key, const float* value, const int64_t* slots, int32_t num_tokens,
                      void* k_cache, void* v_cache, int32_t num_blocks, int32_t block_size, int32_t hkv, int32_t d);

int32_t kv_copy_blocks_fp4(fi_context* ctx, void* k_cache, void* v_cache, const int32_t* src, const int32_t* dst,
                           const int32_t* counts, int32_t num_pairs, int32_t num_blocks, int32_t block_size,
                           int32_t hkv, int32_t d);

int32_t kv_gather_fp4(fi_context* ctx, const void* k_cache, const void* v_cache, const int32_t* table, int32_t length,
                      int32_t num_blocks, int32_t block_size, int32_t hkv, int32_t d, float* k_out, float* v_out);

// Tokens of a sequence that decode serves over a 4-bit pool: 256 partitions of 512 tokens, or 512 of 256 where
// the rows are narrow (wave_tokens_for).
constexpr int kFp4MaxContext = 131072;

// Whether a decode launch of several partitions (up to `heads` heads a workgroup) merges them by itself:
// the workgroup that ends a sequence's last partition does, instead of a launch of its own.  One
// strand of the merge holds a sequence's weights, up to 16 partitions.  Up to 8 that is the faster way
// (us merging by itself against by a launch: 64 sequences of 128 to 2048 tokens over 8 heads of 128 24.2
// against 26.0, 64 of 4000 66.2 against 68.7, one of 700 over 2 heads of 64 7.4 against 10.0).  Of 9 to 16 it is
// for large launches with few heads a workgroup (128 of 512 to 8192 142.5 against 145.0, 16 of 5500 26.5 against
// 27.4), not for small ones, which end in the merge of a few workgroups (one of 8000 11.6 against 10.8), nor
// for more heads a workgroup (14/2 heads of 64, 8 of 4000 13.0 against 9.9, 64 of 4000 22.9 against 22.1).
bool decode_fp4_merges(int64_t workgroups, int parts, int heads, int64_t cus);

// Decode attention: the partition launch and, where the launch does not merge by itself, the merge.
int32_t decode_fp4(fi_context* ctx, const DecodeArgs& args, int32_t head_dim, dim3 grid, int wave_tokens);

// Prefill attention, its arguments checked as the other pools'.
int32_t prefill_fp4(fi_context* ctx, const PrefillArgs& args, int32_t head_dim);

}  // namespace fi
