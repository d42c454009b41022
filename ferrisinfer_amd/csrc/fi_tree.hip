// Trees of drafted tokens: masks and positions from the nodes' parents, and the accepted path's K/V rows
// moved to their places behind the prefix.  No counterpart in the reference, whose sessions feed one sampled
// token a step (crates/ferrisinfer-runtime/src/session.rs:246-262).
#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "fi_common.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"
#include "fi_tree.h"

namespace {

// One workgroup a tree, its parents in LDS.  A thread walks from its node upwards: ancestors come in falling
// order, so a word of the mask is complete, and stored, when the walk leaves it.  mask[i] = mask[parent] | 1 << i
// and depth[i] = depth[parent] + 1 without waiting for the parent's thread.  256 trees of 17 to 100 nodes take 3.2 us, one
// of eight 2.2: the launch, two dependent loads, and a walk of LDS reads.
__global__ __launch_bounds__(256) void tree_plan_kernel(const int* __restrict__ parents, const int* __restrict__ cu,
                                                        const int* __restrict__ lens, int max_query_len, int words,
                                                        uint64_t* __restrict__ mask, int* __restrict__ positions,
                                                        uint32_t* __restrict__ faults) {
  __shared__ int s_parent[fi::kMaxTreeNodes];
  const fi::TreeSpan t = fi::tree_span(cu, lens, blockIdx.x);
  const int n = min(t.nodes, max_query_len);
  if (t.nodes > max_query_len && threadIdx.x == 0) atomicOr(faults, FI_FAULT_QUERY_RANGE);
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int p = parents[t.first + i];
    if (p < -1 || p >= i) {  // also what keeps the walks below finite
      atomicOr(faults, FI_FAULT_TREE_RANGE);
      p = -1;
    }
    s_parent[i] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    uint64_t* row = mask + (size_t)(t.first + i) * words;
    int word = words - 1, depth = -1;
    uint64_t bits = 0;
    for (int a = i; a >= 0; a = s_parent[a]) {
      for (; word > a >> 6; --word) {
        row[word] = bits;
        bits = 0;
      }
      bits |= 1ull << (a & 63);
      ++depth;
    }
    for (; word >= 0; --word) {
      row[word] = bits;
      bits = 0;
    }
    positions[t.first + i] = t.prefix + depth;
  }
}

// ---- the accepted path's rows ----

typedef uint32_t quad __attribute__((ext_vector_type(4)));  // 16 bytes

constexpr int kLayersPerLaunch = 64;
constexpr int kBatch = 8;  // rows of a path that are loaded before any of them is stored

struct KeepArgs {
  void* pools[2 * kLayersPerLaunch];  // K and V arrays, each once
  const int* block_tables;
  const int* cu_seqlens;
  const int* context_lens;
  const int* path;  // [num_seqs, max_path]
  uint32_t* faults;
  int max_blocks, max_path, num_blocks, block_size, hkv;
  int pools_in_launch;
  size_t second;  // 4-bit pools: bytes of the codes, behind which the scales lie
  fi::FastDiv blocks;
};

// Rows of `units` T's, one thread a T: row prefix + path[i] to row prefix + 1 + i, in path order.  path rises
// strictly, so path[i] >= i + 1: a store into row 1 + i can only overwrite a row whose own turn has been
// (a thread loads kBatch rows before it stores them, and later rows lie behind all of these places), and each
// thread moves its own column, so the rows may overlap.
template <typename T>
__device__ __forceinline__ void move_rows(const KeepArgs& a, T* pool, int units, const fi::TreeSpan& t, const int* table,
                                          const int* path, int from, int step, bool report) {
  for (int u = from; u < a.hkv * units; u += step) {
    const int head = u / units, col = u - head * units;
    // element of a row at `position`, or null: no block there
    auto at = [&](int position) -> T* {
      const int lb = position < 0 ? -1 : static_cast<int>(a.blocks.div(position));
      const int id = lb >= 0 && lb < a.max_blocks ? table[lb] : -1;
      if (id < 0 || id >= a.num_blocks) {
        if (report) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
        return nullptr;
      }
      return pool + (((size_t)id * a.hkv + head) * a.block_size + (position - lb * a.block_size)) * units + col;
    };
    int last = 0;
    bool more = true;
    for (int i0 = 0; more && i0 < a.max_path; i0 += kBatch) {
      T held[kBatch];
      T* to[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        to[j] = nullptr;
        const int node = more && i0 + j < a.max_path ? path[i0 + j] : -1;
        if (node <= last || node >= t.nodes) {  // the path's end, or an entry that is none
          if (report && more && node >= 0) atomicOr(a.faults, FI_FAULT_TREE_RANGE);
          more = false;
          continue;
        }
        last = node;
        if (node == 1 + i0 + j) continue;  // in its place
        const T* src = at(t.prefix + node);
        T* dst = at(t.prefix + 1 + i0 + j);
        if (src && dst) {
          held[j] = *src;
          to[j] = dst;
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (to[j]) *to[j] = held[j];
    }
  }
}

// One workgroup a (sequence, pool array): row_units T's a head's row; 4-bit pools' scale bytes (an S a row) lie
// behind the codes.  32 sequences, up to six rows of 8 heads of 128 bf16 each in 32 layers: 10.2 us for 25 MB read and
// written; one sequence in 24 layers 4.8.  A chain of latencies (the path, the block ids, the rows) in 2048 workgroups.
template <typename T, typename S>
__global__ __launch_bounds__(256) void keep_path_kernel(KeepArgs a, int row_units) {
  const int seq = blockIdx.x / a.pools_in_launch, which = blockIdx.x - seq * a.pools_in_launch;
  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, seq);
  const int* table = a.block_tables + (size_t)seq * a.max_blocks;
  const int* path = a.path + (size_t)seq * a.max_path;
  uint8_t* pool = static_cast<uint8_t*>(a.pools[which]);
  const bool report = threadIdx.x == 0;
  move_rows(a, reinterpret_cast<T*>(pool), row_units, t, table, path, threadIdx.x, blockDim.x, report);
  if constexpr (!std::is_void_v<S>)
    move_rows(a, reinterpret_cast<S*>(pool + a.second), 1, t, table, path, threadIdx.x, blockDim.x, false);
}

template <typename T, typename S>
void launch_keep(fi_context* ctx, const KeepArgs& args, int num_seqs, int row_units) {
  const int threads = std::min(256, (args.hkv * row_units + 63) / 64 * 64);
  hipLaunchKernelGGL((keep_path_kernel<T, S>), dim3(static_cast<unsigned>(num_seqs) * args.pools_in_launch), dim3(threads), 0,
                     ctx->stream, args, row_units);
}

}  // namespace

extern "C" {

int32_t fi_tree_plan(fi_context* ctx, const int32_t* d_parents, const int32_t* d_cu_seqlens, const int32_t* d_context_lens,
                     int32_t num_seqs, int32_t max_query_len, int32_t mask_words, uint64_t* d_tree_mask,
                     int32_t* d_positions) {
  FI_TRY(fi::enter(ctx));
  FI_REQUIRE(num_seqs >= 0 && max_query_len >= 0 && mask_words >= 0, FI_ERR_INVALID_SHAPE, "fi_tree_plan: negative sizes");
  FI_REQUIRE(max_query_len <= fi::kMaxTreeNodes, FI_ERR_UNSUPPORTED,
             "fi_tree_plan: trees of more than " + std::to_string(fi::kMaxTreeNodes) + " nodes");
  FI_REQUIRE(mask_words <= (1 << 20) && max_query_len <= 64 * mask_words, FI_ERR_INVALID_SHAPE,
             "fi_tree_plan: mask_words must hold a bit for each of max_query_len nodes");
  if (num_seqs == 0 || max_query_len == 0) return FI_OK;
  FI_REQUIRE(d_parents && d_cu_seqlens && d_context_lens && d_tree_mask && d_positions, FI_ERR_INVALID_CONFIG,
             "fi_tree_plan: null pointer");
  const int threads = std::min(256, (max_query_len + 63) / 64 * 64);
  hipLaunchKernelGGL(tree_plan_kernel, dim3(num_seqs), dim3(threads), 0, ctx->stream, d_parents, d_cu_seqlens, d_context_lens,
                     max_query_len, mask_words, d_tree_mask, d_positions, ctx->d_faults);
  FI_CHECK_LAUNCH("tree_plan_kernel");
  return FI_OK;
}

int32_t fi_kv_keep_path(fi_context* ctx, void* const* k_caches, void* const* v_caches, int32_t num_layers, int32_t kv_dtype,
                        const int32_t* d_block_tables, int32_t max_blocks_per_seq, const int32_t* d_cu_seqlens,
                        const int32_t* d_context_lens, const int32_t* d_path, int32_t max_path, int32_t num_seqs,
                        int32_t num_blocks, int32_t block_size, int32_t num_kv_heads, int32_t head_dim) {
  FI_TRY(fi::enter(ctx));
  FI_REQUIRE(num_seqs >= 0 && num_layers >= 0 && max_path >= 0, FI_ERR_INVALID_SHAPE, "fi_kv_keep_path: negative sizes");
  FI_REQUIRE(kv_dtype == FI_DTYPE_F32 || kv_dtype == FI_DTYPE_BF16 || kv_dtype == FI_DTYPE_MXFP4, FI_ERR_INVALID_TYPE,
             "fi_kv_keep_path: KV dtype must be f32, bf16 or mxfp4");
  FI_REQUIRE(num_blocks > 0 && block_size > 0 && max_blocks_per_seq > 0 && num_kv_heads > 0 && head_dim > 0,
             FI_ERR_INVALID_CONFIG, "fi_kv_keep_path: pool dimensions must be greater than zero");
  FI_REQUIRE(static_cast<int64_t>(num_kv_heads) * head_dim <= (1 << 24), FI_ERR_UNSUPPORTED,
             "fi_kv_keep_path: rows of more than 2^24 elements");
  FI_REQUIRE(num_seqs <= INT32_MAX / (2 * kLayersPerLaunch), FI_ERR_INVALID_SHAPE, "fi_kv_keep_path: too many sequences");
  if (num_seqs == 0 || num_layers == 0 || max_path == 0) return FI_OK;
  FI_REQUIRE(k_caches && v_caches && d_block_tables && d_cu_seqlens && d_context_lens && d_path, FI_ERR_INVALID_CONFIG,
             "fi_kv_keep_path: null pointer");
  uintptr_t bits = 0;  // every layer is checked before any layer's rows move
  std::vector<void*> pools;  // each array once: rows that have moved must not move again, nor two workgroups move the same
  try {
    for (int32_t l = 0; l < num_layers; ++l) {
      FI_REQUIRE(k_caches[l] && v_caches[l], FI_ERR_INVALID_CONFIG, "fi_kv_keep_path: null pointer");
      if (kv_dtype == FI_DTYPE_MXFP4) FI_TRY(fi::check_fp4_pool("fi_kv_keep_path", k_caches[l], v_caches[l], head_dim));
      bits |= reinterpret_cast<uintptr_t>(k_caches[l]) | reinterpret_cast<uintptr_t>(v_caches[l]);
      pools.push_back(k_caches[l]);
      pools.push_back(v_caches[l]);
    }
    std::sort(pools.begin(), pools.end());
    pools.erase(std::unique(pools.begin(), pools.end()), pools.end());
  } catch (const std::exception& e) {
    return fi::set_error(FI_ERR_RUNTIME, std::string("fi_kv_keep_path: ") + e.what());
  }
  KeepArgs a{};
  a.block_tables = d_block_tables;
  a.cu_seqlens = d_cu_seqlens;
  a.context_lens = d_context_lens;
  a.path = d_path;
  a.faults = ctx->d_faults;
  a.max_blocks = max_blocks_per_seq;
  a.max_path = max_path;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.hkv = num_kv_heads;
  a.second = kv_dtype == FI_DTYPE_MXFP4 ? fi::fp4_code_bytes(num_blocks, num_kv_heads, block_size, head_dim) : 0;
  a.blocks = fi::FastDiv(static_cast<uint32_t>(block_size));
  const int cell = kv_dtype == FI_DTYPE_F32 ? 4 : 2;
  for (size_t at = 0; at < pools.size(); at += 2 * kLayersPerLaunch) {
    a.pools_in_launch = static_cast<int>(std::min<size_t>(pools.size() - at, 2 * kLayersPerLaunch));
    std::copy_n(pools.begin() + at, a.pools_in_launch, a.pools);
    if (kv_dtype == FI_DTYPE_MXFP4) {
      if (head_dim == 32)
        launch_keep<quad, uint8_t>(ctx, a, num_seqs, 1);
      else if (head_dim == 64)
        launch_keep<quad, uint16_t>(ctx, a, num_seqs, 2);
      else
        launch_keep<quad, uint32_t>(ctx, a, num_seqs, 4);
    } else if (head_dim * cell % 16 == 0 && bits % 16 == 0) {
      launch_keep<quad, void>(ctx, a, num_seqs, head_dim * cell / 16);
    } else if (cell == 4) {
      launch_keep<uint32_t, void>(ctx, a, num_seqs, head_dim);
    } else {
      launch_keep<uint16_t, void>(ctx, a, num_seqs, head_dim);
    }
    FI_CHECK_LAUNCH("keep_path_kernel");
  }
  return FI_OK;
}

}  // extern "C"
