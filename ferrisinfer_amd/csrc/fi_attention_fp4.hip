// Paged decode attention over a 4-bit KV pool (fi_fp4.h) on v_mfma_f32_16x16x32_bf16, in f32
// accuracy: K and V are exact in bf16, and the f32 operands they meet (query rows,
// probabilities) are carried as three bf16 pieces whose sum is the f32 value exactly (fi::split3_pk).
//
// The pieces cost no extra products.  A 16x16 MFMA tile has sixteen columns; a kv head serves at
// most eight query heads.  Column 4 h + p of a tile is piece p of query head h (p = 3 is zero), so
// one tile carries four heads with their pieces, and the pieces' products are summed over the
// four lanes of a quad afterwards.
//   S^T = K Q^T: keys are the tile's rows.  Lane (m, kb) = (lane & 15, lane >> 4) holds key m's
//     codes of dims kb * D/4 .. + D/4 - 1, as they lie in memory (16 bytes at D = 128); MFMA j takes
//     dims kb * D/4 + 8 j + e as its k index 8 kb + e, and Q is read in the same order.
//   O^T = V^T P^T: dims are the rows.  The scores leave lane (n, kb) with keys 4 kb + r of each
//     16-key tile for its own column n, which is a B operand over 32 keys once the MFMA's k index
//     8 kb + e stands for key 4 kb + e (e < 4) or 16 + 4 kb + e - 4: no exchange between lanes.
//     Lane (m, kb) of A holds those eight keys' codes of dims m * D/16 .. + D/16 - 1; MFMA j takes dim
//     m * D/16 + j.
// Rows past the end are clamped to the last valid row and carry probability 0.
#include <type_traits>

#include "fi_common.h"
#include "fi_decode.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The sum over the four lanes of a quad, in every lane.
__device__ __forceinline__ float quad_sum(float v) { return fi::group_sum<4>(v); }

// Piece p (0, 1, 2; 3: zero) of eight f32 values, as a bf16 operand.
__device__ __forceinline__ bf16x8 piece8(const float (&x)[8], int p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h, m, l;
    fi::split3_pk(x[2 * i], x[2 * i + 1], h, m, l);
    w[i] = p == 0 ? h : (p == 1 ? m : (p == 2 ? l : 0u));
  }
  return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// The low (kHigh = 0) or high halves of eight dwords, in order.
template <int kHigh>
__device__ __forceinline__ bf16x8 halves8(const uint32_t (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], kHigh ? 0x07060302u : 0x05040100u);
  return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// One workgroup = one (sequence, kv head, partition of 4 WT tokens), or in small launches a share of
// its query heads; each wave owns WT consecutive tokens, computes all their scores, then their
// softmax once, then the weighted sum.  T tiles of four query heads.  The waves' (max, sum, acc)
// are combined through LDS in wave order and the partitions as in decode_partition_kernel.
template <int D, int T, int WT>
__global__ __launch_bounds__(kThreads, 2) void decode_fp4_kernel(DecodeArgs a) {
  constexpr int kPartTokens = kWaves * WT;
  constexpr int G = 4 * T;        // query heads
  constexpr int STEPS = WT / 32;  // 32-key steps
  constexpr int KB = D / 8;       // bytes of K codes a lane holds of one key
  constexpr int KJ = D / 32;      // MFMAs of a score tile
  constexpr int VB = D / 32;      // bytes of V codes a lane holds of one key
  constexpr int VJ = D / 16;      // MFMAs of a 32-key step of P V
  constexpr int GROUPS = D / fi::kFp4Group;
  static_assert(WT % 32 == 0, "a wave's tokens are whole steps");

  __shared__ uint32_t s_row[kPartTokens];
  __shared__ float s_ml[kWaves][G][2];
  __shared__ __align__(16) float s_acc[kWaves][G][D];

  const int pairs = a.num_seqs * a.hkv;
  const int part = blockIdx.x / pairs;
  const int pair = blockIdx.x - part * pairs;
  const HeadUnit hu = head_unit<true>(a, pair);
  const int seq = hu.seq, kvh = hu.kvh, group = hu.heads;
  if (group <= 0) return;  // every partition of the share
  const int tid = threadIdx.x;
  int ctx = a.context_lens[seq];
  if (ctx > a.parts_per_seq * kPartTokens) {  // beyond the grid: clamp and report
    if (part == 0 && tid == 0) atomicOr(a.faults, FI_FAULT_CONTEXT_RANGE);
    ctx = a.parts_per_seq * kPartTokens;
  }
  const size_t head0 = hu.head0;
  if (ctx <= 0) {  // no keys: defined output of zeros
    if (part == 0)
      for (int i = tid; i < group * D; i += kThreads) a.out[head0 * D + i] = 0.0f;
    return;
  }
  const int t0 = part * kPartTokens;
  if (t0 >= ctx) return;  // whole workgroup exits together
  const int n_part = min(kPartTokens, ctx - t0);
  const int nparts = (ctx + kPartTokens - 1) / kPartTokens;
  const int w = tid >> 6;
  const int lane = tid & 63;
  const int m = lane & 15, kb = lane >> 4;
  const int piece = m & 3;
  const int n = min(WT, n_part - w * WT);  // the wave's tokens (<= 0: idle wave)

  const size_t code_bytes = fi::fp4_code_bytes(a.num_blocks, a.hkv, a.block_size, D);
  const uint8_t* __restrict__ k_codes = static_cast<const uint8_t*>(a.k_cache);
  const uint8_t* __restrict__ v_codes = static_cast<const uint8_t*>(a.v_cache);
  const uint8_t* __restrict__ k_scales = k_codes + code_bytes;
  const uint8_t* __restrict__ v_scales = v_codes + code_bytes;

  // the partition's token -> pool row indices
  for (int t = tid; t < n_part; t += kThreads) {
    const int pos = t0 + t;
    const int lb = pos / a.block_size;
    int id = lb < a.max_blocks ? a.block_tables[(size_t)seq * a.max_blocks + lb] : -1;
    if (id < 0 || id >= a.num_blocks) {
      atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
      id = 0;
    }
    s_row[t] = (static_cast<uint32_t>(id) * a.hkv + kvh) * a.block_size + (pos - lb * a.block_size);
  }

  // query rows: column m of tile t is piece m & 3 of head 4 t + m / 4
  bf16x8 qf[T][KJ];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int g = 4 * t + (m >> 2);
    const bool live = g < group;
    const float* qp = a.q + (head0 + (live ? g : 0)) * D + kb * (D / 4);
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const float4 lo = *reinterpret_cast<const float4*>(qp + 8 * j);
      const float4 hi = *reinterpret_cast<const float4*>(qp + 8 * j + 4);
      const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      qf[t][j] = piece8(x, live ? piece : 3);
    }
  }
  __syncthreads();

  if (n > 0) {  // wave-uniform
    const uint32_t* rows = s_row + w * WT;
    // ---- scores: sc[t][s][8 i + r] ----
    float sc[T][STEPS][8];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const size_t row = rows[min(32 * s + 16 * i + m, n - 1)];
        fi::Codes<KB> kc;
        kc.load(k_codes + row * (D / 2) + kb * KB);
        const float scale = fi::fp4_scale_f32(k_scales[row * GROUPS + kb * GROUPS / 4]);
        v4f acc[T];
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const bf16x8 kf = __builtin_bit_cast(bf16x8, fi::fp4_widen8(kc.w[j], scale));
#pragma unroll
          for (int t = 0; t < T; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][j], acc[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = quad_sum(acc[t][r]) * a.scale;
            sc[t][s][4 * i + r] = 32 * s + 16 * i + 4 * kb + r < n ? v : -INFINITY;
          }
      }
    }

    // ---- softmax over the wave's tokens (the lanes of column m's quad hold one head) ----
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float mx = -INFINITY;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, sc[t][s][e]);
      mx = fmaxf(mx, fi::lane_xor16(mx, lane));
      mx = fmaxf(mx, fi::lane_xor32(mx, lane));
      float l = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = sc[t][s][e] == -INFINITY ? 0.0f : __expf(sc[t][s][e] - mx);
          sc[t][s][e] = p;
          l += p;
        }
      l += fi::lane_xor16(l, lane);
      l += fi::lane_xor32(l, lane);
      if (kb == 0 && piece == 0) {
        s_ml[w][4 * t + (m >> 2)][0] = mx;
        s_ml[w][4 * t + (m >> 2)][1] = l;
      }
    }

    // ---- O^T += V^T P^T ----
    v4f o[T][VJ];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int j = 0; j < VJ; ++j) o[t][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (32 * s >= n) break;  // wave-uniform: the step holds no key
      fi::Codes<VB> vc[8];
      float scale[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const size_t row = rows[min(32 * s + (e < 4 ? 0 : 16) + 4 * kb + (e & 3), n - 1)];
        vc[e].load(v_codes + row * (D / 2) + m * VB);
        scale[e] = fi::fp4_scale_f32(v_scales[row * GROUPS + m * GROUPS / 16]);
      }
      bf16x8 pf[T];
#pragma unroll
      for (int t = 0; t < T; ++t) pf[t] = piece8(sc[t][s], piece);
#pragma unroll
      for (int j = 0; j < VJ; j += 2) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (j == 0) x[e] = fi::fp4_widen2<0>(vc[e].w[0], scale[e]);
          if (j == 2) x[e] = fi::fp4_widen2<1>(vc[e].w[0], scale[e]);
          if (j == 4) x[e] = fi::fp4_widen2<2>(vc[e].w[0], scale[e]);
          if (j == 6) x[e] = fi::fp4_widen2<3>(vc[e].w[0], scale[e]);
        }
        const bf16x8 even = halves8<0>(x), odd = halves8<1>(x);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, pf[t], o[t][j], 0, 0, 0);
          o[t][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, pf[t], o[t][j + 1], 0, 0, 0);
        }
      }
    }
    // lane (n, kb) holds dims (4 kb + r) * D/16 + j of its column; a quad's lanes store one r each
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float* dst = &s_acc[w][4 * t + (m >> 2)][(4 * kb + piece) * VJ];
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        float sum[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = quad_sum(o[t][j][r]);
        dst[j] = piece == 0 ? sum[0] : (piece == 1 ? sum[1] : (piece == 2 ? sum[2] : sum[3]));
      }
    }
  }
  __syncthreads();

  combine_waves<D, G, WT, true>(a, hu, pairs, pair, part, nparts, n_part, s_ml, s_acc);
}

template <int D, int T, int WT>
int32_t launch(fi_context* ctx, const DecodeArgs& args, dim3 grid) {
  hipLaunchKernelGGL((decode_fp4_kernel<D, T, WT>), grid, dim3(kThreads), 0, ctx->stream, args);
  FI_CHECK_LAUNCH("decode_fp4_kernel");
  if (args.parts_per_seq > 1 && args.counters == nullptr) {
    const dim3 grid2(static_cast<unsigned>(args.num_seqs) * args.hkv, grid.y);
    hipLaunchKernelGGL((decode_merge_kernel<D, 4 * T, WT>), grid2, dim3(kThreads), 0, ctx->stream, args);
    FI_CHECK_LAUNCH("decode_merge_kernel");
  }
  return FI_OK;
}

template <int D>
int32_t launch_dim(fi_context* ctx, const DecodeArgs& args, dim3 grid, int wt) {
  const bool wide = wt == FI_DECODE_WIDE_WAVE_TOKENS;
  if (args.heads_per <= 4)
    return wide ? launch<D, 1, FI_DECODE_WIDE_WAVE_TOKENS>(ctx, args, grid)
                : launch<D, 1, FI_DECODE_NARROW_WAVE_TOKENS>(ctx, args, grid);
  return wide ? launch<D, 2, FI_DECODE_WIDE_WAVE_TOKENS>(ctx, args, grid)
              : launch<D, 2, FI_DECODE_NARROW_WAVE_TOKENS>(ctx, args, grid);
}

}  // namespace

namespace fi {

int32_t decode_fp4(fi_context* ctx, const DecodeArgs& args, int32_t head_dim, dim3 grid, int wave_tokens) {
  switch (head_dim) {
    case 32:
      return launch_dim<32>(ctx, args, grid, wave_tokens);
    case 64:
      return launch_dim<64>(ctx, args, grid, wave_tokens);
    default:
      return launch_dim<128>(ctx, args, grid, wave_tokens);
  }
}

}  // namespace fi
