// The q|k|v projection's consumer with RMS norms of the query and key heads and rotary positions
// of one or several axes (fi_qkv_norm_rope_append), and the consumer of 4-bit pools
// (fi_qkv_rope_append with FI_DTYPE_MXFP4, whose groups need a head row's neighbours).
//
//   x = sum_z parts[z] + bias                                     (splits added in order)
//   y = x / sqrt(mean(x^2) + eps) * w      per query / key head   (where weights are given)
//   pair i of a head, i < rotary_dims / 2, at angle row positions[axis(i)][t] of the cos / sin tables:
//     z[i] = y[i] cos - y[i + half] sin,  z[i + half] = y[i + half] cos + y[i] sin
//   q -> q_out, k and v -> the pool (f32; bf16, nearest even; 4-bit groups of 32)
//
// D / 4 consecutive lanes hold one head row, four elements each, so that the row is read once, the
// sum of squares, the rotary partner and a group's largest magnitude are exchanged in registers, and
// every store is as wide as its row allows.  Bound by the bytes of the partials and outputs.
#include "fi_common.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"
#include "fi_qkv_norm.h"

namespace {

constexpr int kThreads = 256;

struct Fp4Pool {};  // pool type tag

// Sum over the D / 4 lanes of a row.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, int lane) {
  v = fi::group_sum < LPR<16 ? LPR : 16>(v);
  if constexpr (LPR == 32) v += fi::lane_xor16(v, lane);
  return v;
}

template <int D, typename Pool>
__global__ __launch_bounds__(kThreads) void qkv_norm_rope_append_kernel(fi::QkvNormArgs a) {
  constexpr int LPR = D / 4;  // lanes per head row
  const int lane = threadIdx.x & 63;
  const int c = lane % LPR;  // this lane's elements are 4 c .. 4 c + 3
  const int heads = a.hq + 2 * a.hkv;
  const int64_t row = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LPR;
  if (row >= (int64_t)a.tokens * heads) return;  // whole rows leave
  const int t = static_cast<int>(row / heads);
  const int head = static_cast<int>(row - (int64_t)t * heads);
  const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
  const int local = is_q ? head : (is_v ? head - a.hq - a.hkv : head - a.hq);  // within its projection

  const int64_t slot = a.slots[t];
  const bool write_kv = slot >= 0 && slot < a.pool_slots;
  if (head == 0 && c == 0 && slot >= a.pool_slots) atomicOr(a.faults, FI_FAULT_SLOT_RANGE);
  if (!is_q && !write_kv) return;

  const size_t plane = (size_t)a.tokens * heads * D;
  const float* bias = is_q ? a.bias_q : (is_v ? a.bias_v : a.bias_k);
  float4 x = fi::qkv_value4(a.parts + (size_t)t * heads * D, plane, a.splits, bias, local * D + 4 * c,
                            head * D + 4 * c);
  const float* weight = is_q ? a.q_norm : a.k_norm;
  if (!is_v && weight) {
    const float ms = row_sum<LPR>(x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w, lane) * (1.0f / D);
    const float inv = 1.0f / sqrtf(ms + a.eps);
    const float4 w = *reinterpret_cast<const float4*>(weight + 4 * c);
    x = make_float4(x.x * inv * w.x, x.y * inv * w.y, x.z * inv * w.z, x.w * inv * w.w);
  }
  const int half = a.rotary_dims / 2;
  if (!is_v && half > 0) {
    // the partner's elements: half / 4 lanes up for the first half of the rotary dims, down for the second
    const bool rotary = 4 * c < 2 * half, low = 4 * c < half;
    const int from = lane + (rotary ? (low ? half / 4 : -(half / 4)) : 0);
    const float4 o = make_float4(__shfl(x.x, from, 64), __shfl(x.y, from, 64), __shfl(x.z, from, 64),
                                 __shfl(x.w, from, 64));
    if (rotary) {
      const int pair = low ? 4 * c : 4 * c - half;
      float4 cs, sn;
      auto position = [&](int axis) {
        int pos = a.positions[(size_t)axis * a.tokens + t];
        if (pos < 0 || pos >= a.max_positions) {
          atomicOr(a.faults, FI_FAULT_POSITION_RANGE);
          pos = 0;
        }
        return (size_t)pos * half;
      };
      if (a.num_axes == 1) {
        const size_t at = position(0) + pair;
        cs = *reinterpret_cast<const float4*>(a.cos_t + at);
        sn = *reinterpret_cast<const float4*>(a.sin_t + at);
      } else {
        // two bits a pair; four consecutive pairs lie in one word (pair is a multiple of 4)
        const uint32_t axes = a.pair_axes[pair / 16] >> (2 * (pair % 16));
        const size_t p0 = position(axes & 3) + pair, p1 = position((axes >> 2) & 3) + pair + 1,
                     p2 = position((axes >> 4) & 3) + pair + 2, p3 = position((axes >> 6) & 3) + pair + 3;
        cs = make_float4(a.cos_t[p0], a.cos_t[p1], a.cos_t[p2], a.cos_t[p3]);
        sn = make_float4(a.sin_t[p0], a.sin_t[p1], a.sin_t[p2], a.sin_t[p3]);
      }
      float4 y0, y1;
      fi::rope4(low ? x : o, low ? o : x, cs, sn, y0, y1);
      x = low ? y0 : y1;
    }
  }
  if (is_q) {
    *reinterpret_cast<float4*>(a.q_out + ((size_t)t * a.hq + local) * D + 4 * c) = x;
    return;
  }
  const int64_t blk = slot / a.block_size;
  const int off = static_cast<int>(slot - blk * a.block_size);
  const size_t dst = ((size_t)blk * a.hkv + local) * a.block_size + off;  // pool row
  void* cache = is_v ? a.v_cache : a.k_cache;
  if constexpr (std::is_same_v<Pool, Fp4Pool>) {
    uint8_t* pool = static_cast<uint8_t*>(cache);
    // eight lanes hold a group
    const uint32_t top = fi::group_max<8>(max(max(fi::magnitude_bits(x.x), fi::magnitude_bits(x.y)),
                                              max(fi::magnitude_bits(x.z), fi::magnitude_bits(x.w))));
    const uint32_t scale = fi::fp4_scale(top);
    uint32_t codes = 0;
    if (scale != 255u) {
      codes = fi::fp4_pack2<0>(codes, x.x, x.y, fi::fp4_scale_f32(scale));
      codes = fi::fp4_pack2<1>(codes, x.z, x.w, fi::fp4_scale_f32(scale));
    }
    *reinterpret_cast<uint16_t*>(pool + dst * (D / 2) + 2 * c) = static_cast<uint16_t>(codes);
    if (c % 8 == 0) pool[a.code_bytes + dst * (D / fi::kFp4Group) + c / 8] = static_cast<uint8_t>(scale);
  } else {
    fi::put_kv4(static_cast<Pool*>(cache), dst * D + 4 * c, x);
  }
}

template <int D>
void launch(fi_context* ctx, const fi::QkvNormArgs& a, int32_t kv_dtype, dim3 grid) {
  if (kv_dtype == FI_DTYPE_F32) {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, float>), grid, dim3(kThreads), 0, ctx->stream, a);
  } else if (kv_dtype == FI_DTYPE_BF16) {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, uint16_t>), grid, dim3(kThreads), 0, ctx->stream, a);
  } else {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, Fp4Pool>), grid, dim3(kThreads), 0, ctx->stream, a);
  }
}

}  // namespace

namespace fi {

int32_t qkv_norm_rope_append(fi_context* ctx, const char* name, QkvNormArgs a, int32_t head_dim, int32_t kv_dtype,
                             int32_t num_blocks, const int32_t* pair_axes) {
  const std::string n(name);
  FI_REQUIRE(a.tokens >= 0 && a.splits >= 1, FI_ERR_INVALID_SHAPE, n + ": bad shape");
  FI_REQUIRE(a.hq > 0 && a.hkv > 0 && a.hq % a.hkv == 0, FI_ERR_INVALID_SHAPE,
             "number of query heads must be divisible by number of KV heads");
  FI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, FI_ERR_UNSUPPORTED,
             n + ": head_dim must be 32, 64 or 128");
  FI_REQUIRE(a.rotary_dims >= 0 && a.rotary_dims <= head_dim && a.rotary_dims % 2 == 0, FI_ERR_INVALID_CONFIG,
             "rope.rotary_dims must be even and at most the head dimension");
  FI_REQUIRE(a.rotary_dims % 8 == 0, FI_ERR_UNSUPPORTED, n + ": rotary_dims / 2 must be a multiple of 4");
  FI_REQUIRE(num_blocks > 0 && a.block_size > 0, FI_ERR_INVALID_CONFIG, n + ": pool dimensions must be positive");
  FI_REQUIRE(kv_dtype == FI_DTYPE_F32 || kv_dtype == FI_DTYPE_BF16 || kv_dtype == FI_DTYPE_MXFP4, FI_ERR_INVALID_TYPE,
             n + ": KV dtype must be f32, bf16 or mxfp4");
  FI_REQUIRE(a.num_axes >= 1 && a.num_axes <= 4, FI_ERR_INVALID_CONFIG, n + ": one to four position axes");
  FI_REQUIRE(a.num_axes == 1 || a.rotary_dims == 0 || pair_axes != nullptr, FI_ERR_INVALID_CONFIG,
             n + ": several position axes need each pair's axis");
  FI_REQUIRE((!a.q_norm && !a.k_norm) || (a.eps >= 0.0f && a.eps < INFINITY), FI_ERR_INVALID_CONFIG,
             n + ": eps must be finite and not negative");
  for (uint32_t& word : a.pair_axes) word = 0;
  if (pair_axes) {
    for (int32_t i = 0; i < a.rotary_dims / 2; ++i) {
      FI_REQUIRE(pair_axes[i] >= 0 && pair_axes[i] < a.num_axes, FI_ERR_INVALID_CONFIG,
                 n + ": pair " + std::to_string(i) + " names an axis beyond the positions'");
      a.pair_axes[i / 16] |= static_cast<uint32_t>(pair_axes[i]) << (2 * (i % 16));
    }
  }
  const int64_t threads = static_cast<int64_t>(a.tokens) * (a.hq + 2 * a.hkv) * (head_dim / 4);
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  FI_REQUIRE(blocks <= 0x7fffffffLL, FI_ERR_INVALID_SHAPE, n + ": too many tokens for one launch");
  FI_TRY(enter(ctx));
  if (a.tokens == 0) return FI_OK;
  FI_REQUIRE(a.parts && a.slots && a.k_cache && a.v_cache && a.q_out, FI_ERR_INVALID_CONFIG, n + ": null pointer");
  FI_REQUIRE(a.rotary_dims == 0 || (a.positions && a.cos_t && a.sin_t && a.max_positions > 0), FI_ERR_INVALID_CONFIG,
             n + ": rope tables required");
  uintptr_t bits = 0;
  for (const void* p : {static_cast<const void*>(a.parts), static_cast<const void*>(a.bias_q),
                        static_cast<const void*>(a.bias_k), static_cast<const void*>(a.bias_v),
                        static_cast<const void*>(a.q_norm), static_cast<const void*>(a.k_norm),
                        static_cast<const void*>(a.cos_t), static_cast<const void*>(a.sin_t),
                        static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_cache),
                        static_cast<const void*>(a.v_cache)})
    bits |= reinterpret_cast<uintptr_t>(p);
  FI_REQUIRE((bits & 15) == 0, FI_ERR_INVALID_LAYOUT,
             n + ": partials, biases, weights, tables, q_out and pools must be 16-byte aligned (vector accesses)");
  a.pool_slots = static_cast<int64_t>(num_blocks) * a.block_size;
  a.code_bytes = fp4_code_bytes(num_blocks, a.hkv, a.block_size, head_dim);
  a.faults = ctx->d_faults;
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (head_dim) {
    case 32:
      launch<32>(ctx, a, kv_dtype, grid);
      break;
    case 64:
      launch<64>(ctx, a, kv_dtype, grid);
      break;
    default:
      launch<128>(ctx, a, kv_dtype, grid);
      break;
  }
  FI_CHECK_LAUNCH("qkv_norm_rope_append_kernel");
  return FI_OK;
}

}  // namespace fi

extern "C" {

int32_t fi_qkv_norm_rope_append(fi_context* ctx, const float* d_parts, int32_t splits, const float* d_bias_q,
                                const float* d_bias_k, const float* d_bias_v, const float* d_q_norm,
                                const float* d_k_norm, float eps, const int32_t* d_positions, int32_t num_axes,
                                const int32_t* pair_axes, const float* d_cos, const float* d_sin, int32_t rotary_dims,
                                int32_t max_positions, const int64_t* d_slot_mapping, void* d_k_cache, void* d_v_cache,
                                int32_t kv_dtype, int32_t num_blocks, int32_t block_size, int32_t num_tokens,
                                int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float* d_q_out) {
  fi::QkvNormArgs a{};
  a.parts = d_parts;
  a.splits = splits;
  a.bias_q = d_bias_q;
  a.bias_k = d_bias_k;
  a.bias_v = d_bias_v;
  a.q_norm = d_q_norm;
  a.k_norm = d_k_norm;
  a.eps = eps;
  a.positions = d_positions;
  a.num_axes = num_axes;
  a.cos_t = d_cos;
  a.sin_t = d_sin;
  a.rotary_dims = rotary_dims;
  a.max_positions = max_positions;
  a.slots = d_slot_mapping;
  a.k_cache = d_k_cache;
  a.v_cache = d_v_cache;
  a.block_size = block_size;
  a.tokens = num_tokens;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.q_out = d_q_out;
  return fi::qkv_norm_rope_append(ctx, "fi_qkv_norm_rope_append", a, head_dim, kv_dtype, num_blocks, pair_axes);
}

}  // extern "C"
