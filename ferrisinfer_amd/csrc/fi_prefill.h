// Varlen causal prefill attention over the paged pool: what the kernels of every pool type share
// (launch arguments, tile order, grid, three-piece operands).
#pragma once

#include <algorithm>

#include "fi_common.h"
#include "fi_device.h"

namespace fi {

struct PrefillArgs {
  const float* q;            // [T, Hq, D]
  const void* k_cache;       // [blocks, Hkv, bs, D]
  const void* v_cache;
  const int* cu_seqlens;     // [B+1]
  const int* context_lens;   // [B]
  const int* block_tables;   // [B, max_blocks]
  float* out;                // [T, Hq, D]
  uint32_t* faults;
  int max_blocks;
  int hq, hkv, group;
  int block_size, num_blocks;
  float scale;
  int num_seqs;
  int max_query_len;
  const int* order;          // (sequence, query tile) pairs, largest first; null: tile_of's own order
  int fold;                  // that order pairs long and short tiles (see prefill_plan_kernel)
  // prefill_x3_kernel and prefill_fp4_kernel with key splits: each (tile, kv head) runs as kv_splits
  // workgroups over consecutive ranges of its key chunks, writing partials (unnormalised O, reference
  // point and row sum per row) that prefill_split_merge_kernel (prefill_merge_fp4_kernel) combines in
  // split order
  int kv_splits;
  float* part;
  int split_chunks;  // 4-bit pools: a tile is cut into kv_splits ranges, or as many of this many chunks as it has
};

}  // namespace fi

namespace {

using fi::PrefillArgs;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// ds_read_b64_tr_b16 at an LDS address (8-byte aligned)
__device__ __forceinline__ v4s lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
}

constexpr int kThreads = 256;
constexpr int kRows = 64;     // (head, token) rows per workgroup

// One workgroup sorts the (sequence, query tile) pairs by the number of kb-key chunks they
// attend, largest first (counting sort over 1024 buckets; order within a bucket arbitrary,
// which no result depends on; tiles past a sequence's end sort last).
__global__ __launch_bounds__(1024) void prefill_plan_kernel(const int* __restrict__ cu, const int* __restrict__ ctxl,
                                                            int num_seqs, int ntiles, int qt_rows, int kb, int fold,
                                                            int* __restrict__ order, uint32_t* __restrict__ faults) {
  __shared__ int hist[1024];
  __shared__ int part[1024];
  __shared__ int s_live;
  const int tid = threadIdx.x;
  const int total = num_seqs * ntiles;
  hist[tid] = 0;
  // a query length beyond the tiles that max_query_len sized: its tail rows get no workgroup
  for (int s = tid; s < num_seqs; s += 1024) {
    if (cu[s + 1] - cu[s] > ntiles * qt_rows) atomicOr(faults, FI_FAULT_QUERY_RANGE);
  }
  __syncthreads();
  auto bucket = [&](int t) {  // 0 = past the sequence's end, else chunks + 1 (capped)
    const int seq = t / ntiles, qt = t - (t / ntiles) * ntiles;
    const int qs = cu[seq], qlen = cu[seq + 1] - qs;
    const int q0 = qt * qt_rows;
    if (q0 >= qlen) return 0;
    const int kend = ctxl[seq] - qlen + min(qlen, q0 + qt_rows);
    return min(max((kend + kb - 1) / kb, 0) + 1, 1023);
  };
  for (int t = tid; t < total; t += 1024) atomicAdd(&hist[1023 - bucket(t)], 1);
  __syncthreads();
  if (tid == 0) s_live = total - hist[1023];  // tiles with rows (bucket 0 sorts last)
  const int v = hist[tid];  // exclusive scan of the bucket counts (Hillis-Steele)
  part[tid] = v;
  __syncthreads();
  for (int off = 1; off < 1024; off <<= 1) {
    const int x = tid >= off ? part[tid - off] : 0;
    __syncthreads();
    part[tid] += x;
    __syncthreads();
  }
  hist[tid] = part[tid] - v;
  __syncthreads();
  // fold (a launch that fits the device in one round, two workgroups per CU): sorted position
  // p of the n live tiles goes to rank p in the first half and to rank half + (n - 1 - p) in
  // the second, so ranks r and r + half, which the dispatcher places on the same CU, pair a
  // long tile with a short one
  const int n = s_live, half = (n + 1) / 2;
  for (int t = tid; t < total; t += 1024) {
    const int p = atomicAdd(&hist[1023 - bucket(t)], 1);
    order[fold && p < n && p >= half ? half + (n - 1 - p) : p] = t;
  }
}

// The tile (seq * ntiles + query tile) of a rank.  Without a planned order: one sequence's tiles
// from its last to its first, which is largest first, folded as the plan folds them; several
// sequences' last tiles, then the ones before, and so on (launches of at most one workgroup a CU).
__device__ __forceinline__ int tile_of(const PrefillArgs& a, int rank, int ntiles, int qt_tokens) {
  if (a.order) return a.order[rank];
  if (a.num_seqs > 1) {
    const int t = rank / a.num_seqs;
    return (rank - t * a.num_seqs) * ntiles + ntiles - 1 - t;
  }
  const int n = min(ntiles, (a.cu_seqlens[1] - a.cu_seqlens[0] + qt_tokens - 1) / qt_tokens);
  if (rank >= n) return rank;  // past the sequence's end
  const int half = (n + 1) / 2;
  return a.fold && rank >= half ? rank - half : n - 1 - rank;
}

// What the plan reports, where there is none: a query length beyond the tiles that max_query_len
// sized (its tail rows get no workgroup).
__device__ __forceinline__ void check_query_length(const PrefillArgs& a, int qt, int qlen, int rows) {
  if (!a.order && qt == 0 && qlen > rows && threadIdx.x == 0) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
}

// Sizes the grid (one workgroup per tile and kv head, and split) and sorts the tiles largest first
// into the context workspace, one small launch before the attention kernel (4.7 us).  No plan
// where the kernels know as good an order: a single sequence, and several whose workgroups
// have a CU each (13 prompts of 20-70 tokens, 14/2 heads: 12.1 -> 8.2 us; a 2048-token chunk
// after 2048, bf16: 130.6 -> 126.5 us; 700 tokens after 300, f32 pool: 71.5 -> 67.5 us).  At two to
// four a CU the unplanned order cost more than the launch (3 sequences of 20-150 tokens after up
// to 2000, 32/8 heads, f32 pool: 104 planned, 118 us without).
#ifndef FI_PREFILL_FOLD
#define FI_PREFILL_FOLD 1
#endif

int32_t plan_tiles(fi_context* ctx, PrefillArgs& args, int qt, int kb, const char* name, dim3* grid, int splits = 1,
                   size_t part_floats = 0) {
  const int ntiles = (args.max_query_len + qt - 1) / qt;
  const long pairs = (long)ntiles * args.num_seqs;
  const long wgs = pairs * args.hkv * splits;
  FI_REQUIRE(wgs <= 0x7fffffffL, FI_ERR_INVALID_SHAPE, std::string(name) + ": grid too large");
  const long cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const bool plan = args.num_seqs > 1 && wgs > cus;
  // the tile order, then (split launches) each workgroup's partials
  const size_t order_bytes = plan ? ((size_t)pairs * sizeof(int) + 255) & ~static_cast<size_t>(255) : 0;
  const size_t part_bytes = splits > 1 ? (size_t)wgs * part_floats * sizeof(float) : 0;
  if (order_bytes + part_bytes > 0) FI_TRY(fi::ensure_workspace(ctx, order_bytes + part_bytes));
  args.kv_splits = splits;
  args.part = splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(ctx->workspace) + order_bytes) : nullptr;
  // one round of workgroups (two per CU): pair long and short tiles on each CU
  args.fold = FI_PREFILL_FOLD && splits == 1 && wgs <= 2 * cus;
  args.order = nullptr;
  if (plan) {
    int* order = static_cast<int*>(ctx->workspace);
    hipLaunchKernelGGL(prefill_plan_kernel, dim3(1), dim3(1024), 0, ctx->stream, args.cu_seqlens, args.context_lens,
                       args.num_seqs, ntiles, qt, kb, args.fold, order, ctx->d_faults);
    FI_CHECK_LAUNCH("prefill_plan_kernel");
    args.order = order;
  }
  *grid = dim3(static_cast<unsigned>(wgs));
  return FI_OK;
}

// An f32 operand as its three bf16 pieces (fi::split3_pk).
__device__ __forceinline__ void split3(const f32x8& x, bf16x8 (&p)[3]) {
  uint4 h, m, l;
  fi::split3_pk(x[0], x[1], h.x, m.x, l.x);
  fi::split3_pk(x[2], x[3], h.y, m.y, l.y);
  fi::split3_pk(x[4], x[5], h.z, m.z, l.z);
  fi::split3_pk(x[6], x[7], h.w, m.w, l.w);
  p[0] = __builtin_bit_cast(bf16x8, h);
  p[1] = __builtin_bit_cast(bf16x8, m);
  p[2] = __builtin_bit_cast(bf16x8, l);
}

}  // namespace
