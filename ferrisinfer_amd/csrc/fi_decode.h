// Paged decode attention: what the kernels over every pool type share (launch arguments, head
// shares, the split-KV merge).
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

// Orders this wave's LDS stores before its later LDS loads by other lanes (a compiler
// barrier only: a wave's LDS operations execute in order).
__device__ __forceinline__ void wave_lds_sync() { __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); }

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

// Combines the partitions of one (sequence, kv_head) group: M = max m_p,
// L = sum l_p e^(m_p-M), out = sum acc_p e^(m_p-M) / L per query head.  The first
// partitions' partials are fetched before the weights are known so the loads overlap.  The
// same arithmetic, in the same order, runs in decode_merge_kernel and in the partition
// kernel's last-arriving workgroup, so both give identical outputs.
template <int D, int MAXG, bool COHERENT>
__device__ __forceinline__ void merge_unit(const DecodeArgs& a, size_t head0, int group, int nparts,
                                           float (*s_w)[kMaxParts], float* s_inv) {
  constexpr int kPrefetch = 8;
  constexpr int kPerThread = (MAXG * D + kThreads - 1) / kThreads;
  const int tid = threadIdx.x;
  const int w = tid >> 6;
  const int lane = tid & 63;
  const int P = a.parts_per_seq;

  float pre[kPerThread][kPrefetch];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = tid + k * kThreads;
    const int g = i / D, d = i % D;
#pragma unroll
    for (int p = 0; p < kPrefetch; ++p)
      pre[k][p] = (g < group && p < nparts) ? load_partial<COHERENT>(&a.part_acc[((head0 + g) * P + p) * D + d]) : 0.0f;
  }
  for (int g = w; g < group; g += 4) {
    // each lane's (max, sum) pairs are read once and kept for the weights
    constexpr int kPartsPerLane = kMaxParts / 64;
    float* ml = a.part_ml + (head0 + g) * P * 2;
    float2 mlv[kPartsPerLane];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPartsPerLane; ++j) {
      const int p = lane + 64 * j;
      if constexpr (COHERENT)
        mlv[j] = p < nparts ? make_float2(load_partial<true>(&ml[2 * p]), load_partial<true>(&ml[2 * p + 1]))
                            : make_float2(-INFINITY, 0.0f);
      else
        mlv[j] = p < nparts ? reinterpret_cast<const float2*>(ml)[p] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, mlv[j].x);
    }
    m = fi::wave_max(m);
    float l = 0.0f;
#pragma unroll
    for (int j = 0; j < kPartsPerLane; ++j) {
      const int p = lane + 64 * j;
      if (p < nparts) {
        const float wgt = __expf(mlv[j].x - m);
        s_w[g][p] = wgt;
        l += mlv[j].y * wgt;
      }
    }
    l = fi::wave_sum(l);
    if (lane == 0) s_inv[g] = 1.0f / l;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = tid + k * kThreads;
    const int g = i / D, d = i % D;
    if (g >= group) continue;
    float acc = 0.0f;
#pragma unroll
    for (int p = 0; p < kPrefetch; ++p) acc += pre[k][p] * (p < nparts ? s_w[g][p] : 0.0f);
    for (int p = kPrefetch; p < nparts; ++p)
      acc += load_partial<COHERENT>(&a.part_acc[((head0 + g) * P + p) * D + d]) * s_w[g][p];
    a.out[(head0 + g) * D + d] = acc * s_inv[g];
  }
}

// The end of a partition workgroup: the waves' (max, sum, acc) in LDS are combined in wave order.
// A sequence with one partition writes its normalised output; otherwise the partition's partial is
// stored, and where the launch merges by itself the last of the group's partitions merges them.
template <int D, int G, int WT, bool SHARES>
__device__ __forceinline__ void combine_waves(const DecodeArgs& a, const HeadUnit& hu, int pairs, int pair, int part,
                                              int nparts, int n_part, const float (*s_ml)[G][2],
                                              const float (*s_acc)[G][D]) {
  constexpr int kWaveTokens = WT;
  const int tid = threadIdx.x, group = hu.heads;
  const size_t head0 = hu.head0;
  const int nw = (n_part + kWaveTokens - 1) / kWaveTokens;
  for (int i = tid; i < group * D; i += kThreads) {
    const int g = i / D, d = i - (i / D) * D;
    float mx = s_ml[0][g][0];
    for (int v = 1; v < nw; ++v) mx = fmaxf(mx, s_ml[v][g][0]);
    float l = 0.0f, sum = 0.0f;
    for (int v = 0; v < nw; ++v) {
      const float wgt = __expf(s_ml[v][g][0] - mx);
      l += s_ml[v][g][1] * wgt;
      sum += s_acc[v][g][d] * wgt;
    }
    if (nparts == 1) {
      a.out[(head0 + g) * D + d] = sum * (1.0f / l);
    } else if (a.counters) {  // read by another workgroup of this launch: device-coherent stores
      const size_t slot = (head0 + g) * a.parts_per_seq + part;
      __hip_atomic_store(&a.part_acc[slot * D + d], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0) {
        __hip_atomic_store(&a.part_ml[slot * 2], mx, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&a.part_ml[slot * 2 + 1], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    } else {
      const size_t slot = (head0 + g) * a.parts_per_seq + part;
      a.part_acc[slot * D + d] = sum;
      if (d == 0) {
        a.part_ml[slot * 2] = mx;
        a.part_ml[slot * 2 + 1] = l;
      }
    }
  }
  if (nparts <= 1 || a.counters == nullptr) return;  // workgroup-uniform

  // ---- the last of the group's partitions to finish merges them ----
  // Each thread waits until its coherent stores have completed, so when the counter shows
  // every partition arrived, every partial is readable at the coherence point.  No cache-wide
  // fence is used (a device-scope fence writes back the whole L2 of the XCD).  The last
  // arriver resets the counter for the next launch or graph replay.
  __shared__ float s_w[G][kMaxParts];
  __shared__ float s_inv[G];
  __shared__ int s_last;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const int unit = (SHARES ? blockIdx.y * pairs : 0) + pair;
    const unsigned arrived =
        __hip_atomic_fetch_add(&a.counters[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    s_last = arrived == static_cast<unsigned>(nparts);
    if (s_last) __hip_atomic_store(&a.counters[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  merge_unit<D, G, true>(a, head0, group, nparts, s_w, s_inv);
}

// The separate merge launch (used where the partition kernel does not merge): one workgroup
// per (sequence, kv_head) group; sequences with a single partition were finished by the
// partition kernel, and the launch boundary orders the partials' stores before these loads.
template <int D, int MAXG, int WT>
__global__ __launch_bounds__(kThreads) void decode_merge_kernel(DecodeArgs a) {
  constexpr int kPartTokens = kWaves * WT;
  __shared__ float s_w[MAXG][kMaxParts];
  __shared__ float s_inv[MAXG];
  const HeadUnit u = head_unit<true>(a, blockIdx.x);
  if (u.heads <= 0) return;
  const int ctx = min(a.context_lens[u.seq], a.parts_per_seq * kPartTokens);  // clamped as in the partitions
  const int nparts = (ctx + kPartTokens - 1) / kPartTokens;
  if (nparts <= 1) return;
  merge_unit<D, MAXG, false>(a, u.head0, u.heads, nparts, s_w, s_inv);
}

}  // namespace
