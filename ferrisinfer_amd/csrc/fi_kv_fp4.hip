// Append to, copy within and read back from a 4-bit KV pool (fi_fp4.h): fi_kv_append,
// fi_kv_copy_blocks and fi_kv_gather with FI_DTYPE_MXFP4.
#include <algorithm>
#include <type_traits>

#include "fi_common.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"

namespace {

// Eight consecutive elements of one head row per thread over the flat (token, element) range; the
// four lanes of a group exchange their largest magnitude in registers, so the row is read once and
// its codes (4 bytes a lane) and scale (the first lane) are written once.  A group's lanes are
// always the four lanes of an aligned quad: rows are multiples of 32 elements.  Bound by the bytes
// of the f32 rows: 6001 tokens of 8 heads of 128, 55.7 MB, in 15.2 us (3.7 TB/s); 64 tokens, one round of
// dependent loads, 3.2 us.
template <bool VEC>
__global__ __launch_bounds__(256) void kv_append_fp4_kernel(const float* __restrict__ key,
                                                            const float* __restrict__ value,
                                                            const int64_t* __restrict__ slots,
                                                            uint8_t* __restrict__ k_cache,
                                                            uint8_t* __restrict__ v_cache, int64_t pool_slots,
                                                            int block_size, int hkv, int d, size_t code_bytes,
                                                            uint32_t total8, fi::FastDiv row8,
                                                            uint32_t* __restrict__ faults) {
  const uint32_t idx = blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= total8) return;
  const uint32_t t = row8.div(idx);
  const int i = static_cast<int>(idx - t * row8.d) * 8;
  const int64_t slot = slots[t];
  if (slot < 0) return;
  if (slot >= pool_slots) {
    if (i == 0) atomicOr(faults, FI_FAULT_SLOT_RANGE);
    return;
  }
  // slots past 32 bits take the long division
  const int64_t blk = slot <= 0xffffffffLL ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(block_size))
                                           : slot / block_size;
  const int off = static_cast<int>(slot - blk * block_size);
  const int h = i >> (31 - __clz(d)), e = i & (d - 1);  // d is 32, 64 or 128
  const size_t row = ((size_t)blk * hkv + h) * block_size + off;
  const size_t src = (size_t)t * hkv * d + i;
  auto load = [&](const float* p) {
    if constexpr (VEC) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
  };
  auto put = [&](const float* from, uint8_t* cache) {
    uint32_t scale;
    const uint32_t codes = fi::fp4_quantise8(load(from + src), load(from + src + 4), scale);
    *reinterpret_cast<uint32_t*>(cache + row * (d / 2) + e / 2) = codes;
    if ((threadIdx.x & 3) == 0) cache[code_bytes + row * (d / fi::kFp4Group) + e / fi::kFp4Group] = scale;
  };
  put(key, k_cache);
  put(value, v_cache);
}

// One workgroup per (pair, kv_head): copies the first n token rows of a block, codes and scales, a dword
// and a byte a thread at a time.  64 blocks of 16 rows of 8 heads of 128, 2.2 MB moved, 3.1 us, one block 2.9: the
// launch and the chain of its loads.
__global__ __launch_bounds__(256) void kv_copy_blocks_fp4_kernel(uint8_t* __restrict__ k_cache,
                                                                 uint8_t* __restrict__ v_cache,
                                                                 const int* __restrict__ src,
                                                                 const int* __restrict__ dst,
                                                                 const int* __restrict__ counts, int num_blocks,
                                                                 int block_size, int hkv, int d, size_t code_bytes,
                                                                 uint32_t* __restrict__ faults) {
  const int pair = blockIdx.x / hkv;
  const int h = blockIdx.x % hkv;
  const int s = src[pair], t = dst[pair];
  const int n = min(max(counts[pair], 0), block_size);
  if (s < 0 || s >= num_blocks || t < 0 || t >= num_blocks) {
    if (threadIdx.x == 0) atomicOr(faults, FI_FAULT_BLOCK_RANGE);
    return;
  }
  const size_t so = ((size_t)s * hkv + h) * block_size, to = ((size_t)t * hkv + h) * block_size;
  const int words = d / 8;  // dwords of a row's codes
  const int groups = d / fi::kFp4Group;
  for (uint8_t* cache : {k_cache, v_cache}) {
    uint32_t* codes = reinterpret_cast<uint32_t*>(cache);
    for (int i = threadIdx.x; i < n * words; i += blockDim.x) codes[to * words + i] = codes[so * words + i];
    uint8_t* scales = cache + code_bytes;
    for (int i = threadIdx.x; i < n * groups; i += blockDim.x) scales[to * groups + i] = scales[so * groups + i];
  }
}

// One thread per 8 consecutive elements of an output row [t][h][d .. d + 7].  Bound by the bytes of the
// f32 rows that it writes: 6001 tokens of 8 heads of 128, 55.7 MB, in 13.6 us (4.1 TB/s).
__global__ __launch_bounds__(256) void kv_gather_fp4_kernel(const uint8_t* __restrict__ k_cache,
                                                            const uint8_t* __restrict__ v_cache,
                                                            const int* __restrict__ table, int64_t total8,
                                                            int num_blocks, fi::FastDiv bs, fi::FastDiv heads, int d,
                                                            size_t code_bytes, float* __restrict__ k_out,
                                                            float* __restrict__ v_out, uint32_t* __restrict__ faults) {
  const int d8_shift = 28 - __clz(d);  // d / 8; d is 32, 64 or 128
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total8; i += stride) {
    const int e = (static_cast<int>(i) & ((1 << d8_shift) - 1)) * 8;
    const uint32_t r = static_cast<uint32_t>(i >> d8_shift);
    const uint32_t t = heads.div(r), h = r - t * heads.d;
    const uint32_t lb = bs.div(t);
    const int b = table[lb];
    const bool bad = b < 0 || b >= num_blocks;
    if (bad) atomicOr(faults, FI_FAULT_BLOCK_RANGE);
    const size_t row = ((size_t)(bad ? 0 : b) * heads.d + h) * bs.d + (t - lb * bs.d);
    auto widen = [&](const uint8_t* cache, float* out) {
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(cache + row * (d / 2) + e / 2);
      const uint32_t scale = cache[code_bytes + row * (d / fi::kFp4Group) + e / fi::kFp4Group];
      const uint4 w = fi::fp4_widen8(codes, fi::fp4_scale_f32(scale));
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      float4* p = reinterpret_cast<float4*>(out + i * 8);
      p[0] = bad ? zero : fi::bf16x4_to_f32(w.x, w.y);
      p[1] = bad ? zero : fi::bf16x4_to_f32(w.z, w.w);
    };
    widen(k_cache, k_out);
    widen(v_cache, v_out);
  }
}

}  // namespace

namespace fi {

int32_t kv_append_fp4(fi_context* ctx, const float* key, const float* value, const int64_t* slots, int32_t num_tokens,
                      void* k_cache, void* v_cache, int32_t num_blocks, int32_t block_size, int32_t hkv, int32_t d) {
  const int64_t pool_slots = static_cast<int64_t>(num_blocks) * block_size;
  const int64_t total8 = static_cast<int64_t>(num_tokens) * hkv * d / 8;
  FI_REQUIRE(total8 < 0x7fffffffLL && static_cast<int64_t>(hkv) * d <= 0x7fffffffLL, FI_ERR_INVALID_SHAPE,
             "fi_kv_append: too many tokens for one launch");
  const bool vec = ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) == 0;
  const dim3 grid(static_cast<unsigned>((total8 + 255) / 256));
  const size_t code_bytes = fp4_code_bytes(num_blocks, hkv, block_size, d);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, key, value, slots, static_cast<uint8_t*>(k_cache),
                       static_cast<uint8_t*>(v_cache), pool_slots, block_size, hkv, d, code_bytes,
                       static_cast<uint32_t>(total8), FastDiv(static_cast<uint32_t>(hkv * d / 8)), ctx->d_faults);
  };
  if (vec) {
    launch(kv_append_fp4_kernel<true>);
  } else {
    launch(kv_append_fp4_kernel<false>);
  }
  FI_CHECK_LAUNCH("kv_append_fp4_kernel");
  return FI_OK;
}

int32_t kv_copy_blocks_fp4(fi_context* ctx, void* k_cache, void* v_cache, const int32_t* src, const int32_t* dst,
                           const int32_t* counts, int32_t num_pairs, int32_t num_blocks, int32_t block_size,
                           int32_t hkv, int32_t d) {
  hipLaunchKernelGGL(kv_copy_blocks_fp4_kernel, dim3(static_cast<unsigned>(num_pairs) * hkv), dim3(256), 0, ctx->stream,
                     static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), src, dst, counts, num_blocks,
                     block_size, hkv, d, fp4_code_bytes(num_blocks, hkv, block_size, d), ctx->d_faults);
  FI_CHECK_LAUNCH("kv_copy_blocks_fp4_kernel");
  return FI_OK;
}

int32_t kv_gather_fp4(fi_context* ctx, const void* k_cache, const void* v_cache, const int32_t* table, int32_t length,
                      int32_t num_blocks, int32_t block_size, int32_t hkv, int32_t d, float* k_out, float* v_out) {
  const int64_t total8 = static_cast<int64_t>(length) * hkv * (d / 8);
  FI_REQUIRE(static_cast<int64_t>(length) * hkv < 0x7fffffffLL, FI_ERR_INVALID_SHAPE, "fi_kv_gather: too many rows for one launch");
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((total8 + 255) / 256, 4096));
  hipLaunchKernelGGL(kv_gather_fp4_kernel, dim3(grid), dim3(256), 0, ctx->stream, static_cast<const uint8_t*>(k_cache),
                     static_cast<const uint8_t*>(v_cache), table, total8, num_blocks,
                     FastDiv(static_cast<uint32_t>(block_size)), FastDiv(static_cast<uint32_t>(hkv)), d,
                     fp4_code_bytes(num_blocks, hkv, block_size, d), k_out, v_out, ctx->d_faults);
  FI_CHECK_LAUNCH("kv_gather_fp4_kernel");
  return FI_OK;
}

}  // namespace fi
