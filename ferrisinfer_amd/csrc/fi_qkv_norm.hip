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

// y cos + o sin of four elements, each product rounded before the add as in fi::rope4 (the first
// half's minus sign is in sin: -(o sin) = o (-sin) exactly).
__device__ __forceinline__ float4 turn(const float4& y, const float4& o, const float4& cs, const float4& sn) {
#pragma clang fp contract(off)
  return make_float4(y.x * cs.x + o.x * sn.x, y.y * cs.y + o.y * sn.y, y.z * cs.z + o.z * sn.z,
                     y.w * cs.w + o.w * sn.w);
}

// The table row of a token's position on one axis.
__device__ __forceinline__ size_t table_row(const fi::QkvNormArgs& a, int t, uint32_t axis, int half) {
  int pos = a.positions[(size_t)axis * a.tokens + t];
  if (pos < 0 || pos >= a.max_positions) {
    atomicOr(a.faults, FI_FAULT_POSITION_RANGE);
    pos = 0;
  }
  return (size_t)pos * half;
}

// One workgroup = ROWS * kThreads / LPR head rows of one token: the token's slot, block and positions are
// uniform, and a thread's ROWS rows (the same elements of heads kThreads / LPR apart) share its
// weights, cosines and sines.  With one split every load is issued before the first is waited for, but for the
// table rows, which wait for the positions; several splits are loaded after the table rows, eight at a time
// (fi::sum_splits), one latency more.  The chain of dependent loads, not the arithmetic, bounds this.
// 2048 tokens of 32 + 16 heads of 128 (one split, three axes, norms, bf16 pool; 92 MB) 25.7 us, 3.6 TB/s (80
// registers with six rows: 1536 of its 2048 workgroups run at a time), into a 4-bit pool (86 MB) 26.3;
// 64 tokens of four splits 4.9 us (4-bit pool: 4.8, without norms 4.5), one token of 14 + 4 heads of 64 and seven
// splits 3.2 us (4-bit pool 3.8).
template <int D, typename Pool, int ROWS>
__global__ __launch_bounds__(kThreads) void qkv_norm_rope_append_kernel(fi::QkvNormArgs a) {
  constexpr int LPR = D / 4;            // lanes per head row
  constexpr int STEP = kThreads / LPR;  // heads between a thread's rows
  const int lane = threadIdx.x & 63;
  const int c = lane % LPR;  // this lane's elements are 4 c .. 4 c + 3
  const int heads = a.hq + 2 * a.hkv;
  const int t = static_cast<int>(a.chunks.div(blockIdx.x));
  const int chunk = static_cast<int>(blockIdx.x - t * a.chunks.d);
  const int head0 = chunk * (ROWS * STEP) + static_cast<int>(threadIdx.x) / LPR;
  const int64_t slot = a.slots[t];
  const int half = a.rotary_dims / 2;
  const size_t plane = (size_t)a.tokens * heads * D;
  const float* p0 = a.parts + (size_t)t * heads * D;

  float4 x[ROWS];
  if (a.splits == 1) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {  // rows past the last head read head 0 and are dropped
      const int head = head0 + i * STEP < heads ? head0 + i * STEP : 0;
      x[i] = *reinterpret_cast<const float4*>(p0 + head * D + 4 * c);
    }
  }
  // this lane's rotary pairs (of the first or the second half) and their cosines and sines
  const bool rotary = 4 * c < 2 * half, low = 4 * c < half;
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  if (rotary && head0 < a.hq + a.hkv) {
    const int pair = low ? 4 * c : 4 * c - half;
    // two bits a pair; four consecutive pairs lie in one word (pair is a multiple of 4)
    const uint32_t word = pair < 32 ? (pair < 16 ? a.pair_axes0 : a.pair_axes1) : (pair < 48 ? a.pair_axes2 : a.pair_axes3);
    const uint32_t axes = (word >> (2 * (pair % 16))) & 0xffu;
    const size_t r0 = table_row(a, t, axes & 3, half) + pair;
    if (axes == (axes & 3) * 0x55u) {  // one axis turns the four pairs, as all but a few lanes find
      cs = *reinterpret_cast<const float4*>(a.cos_t + r0);
      sn = *reinterpret_cast<const float4*>(a.sin_t + r0);
    } else {
      const size_t r1 = table_row(a, t, (axes >> 2) & 3, half) + pair + 1, r2 = table_row(a, t, (axes >> 4) & 3, half) + pair + 2,
                   r3 = table_row(a, t, axes >> 6, half) + pair + 3;
      cs = make_float4(a.cos_t[r0], a.cos_t[r1], a.cos_t[r2], a.cos_t[r3]);
      sn = make_float4(a.sin_t[r0], a.sin_t[r1], a.sin_t[r2], a.sin_t[r3]);
    }
    if (low) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
  }
  // the pool row of the token's kv head 0; slots past 32 bits take the long division
  const bool write_kv = slot >= 0 && slot < a.pool_slots;
  if (chunk == 0 && threadIdx.x == 0 && slot >= a.pool_slots) atomicOr(a.faults, FI_FAULT_SLOT_RANGE);
  const int64_t blk = !write_kv ? 0
                      : slot <= 0xffffffffLL
                          ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.block_size))
                          : slot / a.block_size;
  const size_t pool_row0 = (size_t)blk * a.hkv * a.block_size + (write_kv ? slot - blk * a.block_size : 0);

#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int head = head0 + i * STEP;
    if (head >= heads) return;  // whole rows leave
    const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
    const int local = is_q ? head : (is_v ? head - a.hq - a.hkv : head - a.hq);  // within its projection
    const float* bias = is_q ? a.bias_q : (is_v ? a.bias_v : a.bias_k);
    float4 y;
    if (a.splits == 1) {
      y = bias ? fi::add(x[i], *reinterpret_cast<const float4*>(bias + local * D + 4 * c)) : x[i];
    } else {
      y = fi::qkv_value4(p0, plane, a.splits, bias, local * D + 4 * c, head * D + 4 * c);
    }
    if (!is_v) {
      const float* weight = is_q ? a.q_norm : a.k_norm;
      if (weight) {
        const float ms = row_sum<LPR>(y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w, lane) * (1.0f / D);
        const float inv = 1.0f / sqrtf(ms + a.eps);
        const float4 w = *reinterpret_cast<const float4*>(weight + 4 * c);
        y = make_float4(y.x * inv * w.x, y.y * inv * w.y, y.z * inv * w.z, y.w * inv * w.w);
      }
      if (half > 0) {
        // the partner's elements: half / 4 lanes up for the first half of the rotary dims, down for the second
        const int from = lane + (rotary ? (low ? half / 4 : -(half / 4)) : 0);
        const float4 o = make_float4(__shfl(y.x, from, 64), __shfl(y.y, from, 64), __shfl(y.z, from, 64),
                                     __shfl(y.w, from, 64));
        const float4 z = turn(y, o, cs, sn);
        y = make_float4(rotary ? z.x : y.x, rotary ? z.y : y.y, rotary ? z.z : y.z, rotary ? z.w : y.w);
      }
    }
    if (is_q) {
      *reinterpret_cast<float4*>(a.q_out + ((size_t)t * a.hq + local) * D + 4 * c) = y;
      continue;
    }
    if (!write_kv) continue;
    const size_t dst = pool_row0 + (size_t)local * a.block_size;
    void* cache = is_v ? a.v_cache : a.k_cache;
    if constexpr (std::is_same_v<Pool, Fp4Pool>) {
      uint8_t* pool = static_cast<uint8_t*>(cache);
      // eight lanes hold a group
      const uint32_t top = fi::group_max<8>(max(max(fi::magnitude_bits(y.x), fi::magnitude_bits(y.y)),
                                                max(fi::magnitude_bits(y.z), fi::magnitude_bits(y.w))));
      const uint32_t scale = fi::fp4_scale(top);
      uint32_t codes = 0;
      if (scale != 255u) {
        codes = fi::fp4_pack2<0>(codes, y.x, y.y, fi::fp4_scale_f32(scale));
        codes = fi::fp4_pack2<1>(codes, y.z, y.w, fi::fp4_scale_f32(scale));
      }
      *reinterpret_cast<uint16_t*>(pool + dst * (D / 2) + 2 * c) = static_cast<uint16_t>(codes);
      if (c % 8 == 0) pool[a.code_bytes + dst * (D / fi::kFp4Group) + c / 8] = static_cast<uint8_t>(scale);
    } else {
      fi::put_kv4(static_cast<Pool*>(cache), dst * D + 4 * c, y);
    }
  }
}

template <int D, int ROWS>
void launch_rows(fi_context* ctx, fi::QkvNormArgs& a, int32_t kv_dtype) {
  const int rows = ROWS * kThreads / (D / 4);  // head rows of a workgroup
  a.chunks = fi::FastDiv(static_cast<uint32_t>((a.hq + 2 * a.hkv + rows - 1) / rows));
  const dim3 grid(static_cast<unsigned>(a.tokens) * a.chunks.d);
  if (kv_dtype == FI_DTYPE_F32) {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, float, ROWS>), grid, dim3(kThreads), 0, ctx->stream, a);
  } else if (kv_dtype == FI_DTYPE_BF16) {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, uint16_t, ROWS>), grid, dim3(kThreads), 0, ctx->stream, a);
  } else {
    hipLaunchKernelGGL((qkv_norm_rope_append_kernel<D, Fp4Pool, ROWS>), grid, dim3(kThreads), 0, ctx->stream, a);
  }
}

// Where one row a thread would make more workgroups than the device holds at once (eight a CU) and at
// most two splits are summed, as few workgroups a token as six rows a thread allow (2048 tokens of 48 heads
// of 128, six rows to a thread fill a workgroup: 46.6 us with one row, 31.3 with two, 28.2 with three,
// 32.4 with four, whose second workgroup is half empty, 26.2 with six; two splits 46.9 against 50.9 with one
// row).  Smaller launches end sooner with more workgroups, and a thread's rows wait for each other's
// splits (four splits 61.6 against 59.0).
template <int D>
void launch(fi_context* ctx, fi::QkvNormArgs& a, int32_t kv_dtype) {
  constexpr int STEP = kThreads / (D / 4);
  const int64_t cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int heads = a.hq + 2 * a.hkv;
  const int passes = a.splits <= 2 && static_cast<int64_t>(a.tokens) * heads > 8 * cus * STEP ? (heads + STEP - 1) / STEP : 1;
  switch (passes) {
    case 1:
      return launch_rows<D, 1>(ctx, a, kv_dtype);
    case 2:
      return launch_rows<D, 2>(ctx, a, kv_dtype);
    case 3:
      return launch_rows<D, 3>(ctx, a, kv_dtype);
    case 4:
      return launch_rows<D, 4>(ctx, a, kv_dtype);
    default:
      return launch_rows<D, 6>(ctx, a, kv_dtype);
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
  uint32_t words[4] = {0, 0, 0, 0};
  if (pair_axes) {
    for (int32_t i = 0; i < a.rotary_dims / 2; ++i) {
      FI_REQUIRE(pair_axes[i] >= 0 && pair_axes[i] < a.num_axes, FI_ERR_INVALID_CONFIG,
                 n + ": pair " + std::to_string(i) + " names an axis beyond the positions'");
      words[i / 16] |= static_cast<uint32_t>(pair_axes[i]) << (2 * (i % 16));
    }
  }
  a.pair_axes0 = words[0];
  a.pair_axes1 = words[1];
  a.pair_axes2 = words[2];
  a.pair_axes3 = words[3];
  FI_REQUIRE((static_cast<int64_t>(a.hq) + 2 * static_cast<int64_t>(a.hkv)) * head_dim <= 0x7fffffffLL, FI_ERR_INVALID_SHAPE,
             n + ": rows are too wide");
  const int64_t blocks =
      static_cast<int64_t>(a.tokens) * ((static_cast<int64_t>(a.hq) + 2 * a.hkv) * (head_dim / 4) / kThreads + 1);
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
  switch (head_dim) {
    case 32:
      launch<32>(ctx, a, kv_dtype);
      break;
    case 64:
      launch<64>(ctx, a, kv_dtype);
      break;
    default:
      launch<128>(ctx, a, kv_dtype);
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
