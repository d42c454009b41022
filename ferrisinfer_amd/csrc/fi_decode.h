// Paged decode attention: what the kernels over every pool type share (launch arguments, partitions,
// head shares).
#pragma once

#include "fi_common.h"
#include "fi_device.h"

namespace fi {

struct DecodeArgs {
  const float* q;
  const void* k_cache;
  const void* v_cache;
  const int* block_tables;
  const int* context_lens;
  float* part_acc;  // [num_seqs * Hq * parts_per_seq, D]
  float* part_ml;   // [num_seqs * Hq * parts_per_seq, 2]
  // Merge in the partition kernel: one arrival counter per (sequence, kv head), zero between
  // launches (the last arriver resets it).  Null: decode_merge_kernel merges.
  unsigned* counters;
  // Fused q|k|v consumer (decode ticks, one new token per sequence), when qkv_parts is set:
  // every workgroup forms its group's query rows from the q|k|v projection's split-K partials
  // (+ bias, RoPE) instead of reading q, and the last partition's workgroup of each
  // (sequence, kv head) first writes the new token's K/V row into the pool at slots[seq].
  const float* qkv_parts;  // [qkv_splits][num_seqs][Hq D + 2 Hkv D]
  int qkv_splits;
  const float* bias_q;
  const float* bias_k;
  const float* bias_v;
  const int* positions;  // [num_seqs] RoPE positions
  const float* cos_t;    // [max_positions][rotary_dims / 2]
  const float* sin_t;
  int rotary_dims;
  int max_positions;
  const int64_t* slots;  // [num_seqs] pool slots of the new tokens
  float* out;
  uint32_t* faults;
  int num_seqs;
  int max_blocks;
  int parts_per_seq;
  int hq;
  int hkv;
  int group;       // query heads per kv head
  int heads_per;   // of them, the heads of one workgroup (gridDim.y workgroups share the group)
  int block_size;
  int num_blocks;
  float scale;
  FastDiv blocks;  // 4-bit pools: by block_size
};

}  // namespace fi

namespace {

using fi::DecodeArgs;

// Tunables (compile-time).  The wave chunk fixes the reduction order for a given context
// length and model shape, so it is a constant of the library, not of a launch.
#ifndef FI_DECODE_WIDE_WAVE_TOKENS
#define FI_DECODE_WIDE_WAVE_TOKENS 128  // context tokens per wave when Hkv * D >= 512
#endif
#ifndef FI_DECODE_NARROW_WAVE_TOKENS
#define FI_DECODE_NARROW_WAVE_TOKENS 64  // narrow KV rows (few, small heads): more workgroups
#endif

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxParts = 256;  // merge weights live in LDS

// Tokens per wave for a model shape (never a batch property: outputs stay batch-invariant).
constexpr int wave_tokens_for(int hkv, int d) {
  return hkv * d >= 512 ? FI_DECODE_WIDE_WAVE_TOKENS : FI_DECODE_NARROW_WAVE_TOKENS;
}

// The query heads of one workgroup: `pair` numbers (sequence, kv head), `share` the part of its
// group (gridDim.y shares, so that a pair's workgroups lie gridDim.x apart: where that is a
// multiple of 8 they run on one XCD and its L2 serves the second read of their K/V).
struct HeadUnit {
  int seq, kvh;
  int first;     // first query head of the share, within the sequence
  int heads;     // <= 0: the group has no heads left for this share
  size_t head0;  // first query head of the share over the batch
};

template <bool SHARES>
__device__ __forceinline__ HeadUnit head_unit(const DecodeArgs& a, int pair) {
  HeadUnit u;
  u.seq = pair / a.hkv;
  u.kvh = pair - u.seq * a.hkv;
  u.first = u.kvh * a.group;
  u.heads = a.group;
  if constexpr (SHARES) {
    const int skip = static_cast<int>(blockIdx.y) * a.heads_per;
    u.first += skip;
    u.heads = min(a.heads_per, a.group - skip);
  }
  u.head0 = (size_t)u.seq * a.hq + u.first;
  return u;
}

// Keeps the instruction scheduler from moving code across this point, so loads issued
// before it stay ahead of the arithmetic after it (the ring's depth is what stays in flight).
__device__ __forceinline__ void sched_fence() { __builtin_amdgcn_sched_barrier(0); }

// A partial of another workgroup: a plain load after a kernel boundary, a device-coherent
// load (past the XCDs' private L2s) inside the partition kernel.
template <bool COHERENT>
__device__ __forceinline__ float load_partial(float* p) {
  if constexpr (COHERENT) return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return *p;
}

}  // namespace
