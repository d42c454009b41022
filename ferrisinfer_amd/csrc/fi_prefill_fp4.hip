// Varlen causal prefill attention over a 4-bit KV pool (fi_fp4.h), in f32 accuracy on
// v_mfma_f32_16x16x32_bf16.
//
// K and V are exact in bf16, so a chunk is widened once, when it is staged, into one bf16 plane;
// only the f32 operands, query rows and probabilities, are carried as three bf16 pieces
// (x = hi + mid + lo exactly), and each product is the sum of three, smallest piece first: half the
// MFMAs of f32 pools, whose K and V need pieces too (prefill_x3_kernel), none of the rounding of
// prefill_bf16_kernel.  The workgroup shape, the tile order, the transposed products, the masking and the
// lazily moved reference point of the exponents are those kernels'.
//
// A chunk is 64 keys: thread (lane, wave) stages key `lane`, elements wave * D/4 .. + D/4 - 1, one load
// of codes and one scale byte each for K and V.  Two LDS buffers, one barrier a chunk; the next
// chunk's codes are in registers (10 of them at D = 128) while the current one is multiplied.
//
// A NaN group of V must reach only the rows that see its key, though a chunk's product multiplies every
// key by every row (0 * NaN is NaN): it is staged as zeros, its key noted in a 64-bit mask of the
// chunk and column quarter, and the rows that see a noted key are set to NaN afterwards.
#include "fi_common.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"
#include "fi_prefill.h"

namespace {

constexpr int kKeys = 64;  // keys per staged chunk

template <int D, int G, int RG, bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void prefill_fp4_kernel(PrefillArgs a) {
  constexpr int QT = kRows * RG / G;    // query tokens per workgroup (RG 16-row groups a wave)
  constexpr int KB = kKeys;
  constexpr int DS = D / 32;             // 32-wide d steps of Q K^T
  constexpr int DT = D / 16;             // 16-wide output d tiles of P V
  constexpr int JT = KB / 16;            // 16-key score tiles per chunk
  constexpr int KS = KB / 32;            // 32-key steps of P V
  constexpr int SEG = D / 4;             // elements a thread stages of its key
  constexpr int GROUPS = D / fi::kFp4Group;
  constexpr int DB = DT < 4 ? DT : 4;    // d tiles whose V fragments are held at once
  constexpr int KP = D + 8;              // padded LDS rows of V (transposing reads)
  constexpr int KPK = D == 128 ? D + 16 : D + 8;  // of K (see prefill_bf16_kernel)
  __shared__ __align__(16) uint16_t Ks[2][KB][KPK];
  __shared__ __align__(16) uint16_t Vs[2][KB][KP];
  __shared__ uint64_t s_nan[2][4];  // keys whose V group is NaN, by column quarter

  const int ntiles = (a.max_query_len + QT - 1) / QT;
  const int wg = blockIdx.x / a.hkv, kvh = blockIdx.x % a.hkv;
  const int rank = SPLIT ? wg / a.kv_splits : wg;
  const int split = SPLIT ? wg - rank * a.kv_splits : 0;
  const int tile = tile_of(a, rank, ntiles, QT);
  const int qt = tile % ntiles, seq = tile / ntiles;
  const int qs = a.cu_seqlens[seq];
  const int qlen = a.cu_seqlens[seq + 1] - qs;
  check_query_length(a, qt, qlen, ntiles * QT);
  const int q0 = qt * QT;
  if (q0 >= qlen) return;
  const int ctx = a.context_lens[seq];
  const int start = ctx - qlen;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, lk = lane >> 4;

  const size_t code_bytes = fi::fp4_code_bytes(a.num_blocks, a.hkv, a.block_size, D);
  const uint8_t* __restrict__ k_codes = static_cast<const uint8_t*>(a.k_cache);
  const uint8_t* __restrict__ v_codes = static_cast<const uint8_t*>(a.v_cache);
  const uint8_t* __restrict__ k_scales = k_codes + code_bytes;
  const uint8_t* __restrict__ v_scales = v_codes + code_bytes;

  // Q pieces: B operand row li of group g, d = 32 t + 8 lk .. + 7
  int qpos[RG];
  bf16x8 qf[RG][DS][3];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const int row = 16 * (w + 4 * g) + li;
    const int ah = row / QT, at = row % QT;
    qpos[g] = start + q0 + at;
    const bool a_ok = ah < a.group && q0 + at < qlen;
    const float* qp = a.q + ((size_t)(qs + q0 + (a_ok ? at : 0)) * a.hq + kvh * a.group + (a_ok ? ah : 0)) * D;
#pragma unroll
    for (int t = 0; t < DS; ++t) {
      const float4 lo = *reinterpret_cast<const float4*>(qp + 32 * t + 8 * lk);
      const float4 hi = *reinterpret_cast<const float4*>(qp + 32 * t + 8 * lk + 4);
      const f32x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      split3(a_ok ? v : z, qf[g][t]);
    }
  }
  v4f o[RG][DT];  // O^T tile dt of group g: d = 16 dt + 4 lk + v, row li
  float m_row[RG], l_part[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[g][dt] = v4f{0.f, 0.f, 0.f, 0.f};
    m_row[g] = -INFINITY;
    l_part[g] = 0.0f;
  }
  const float c2 = a.scale * 1.4426950408889634f;  // scores -> log2 units
  constexpr float kLazy = 8.0f;  // headroom of the exponents' reference point (log2 units)

  const int kend = start + min(qlen, q0 + QT);
  const int nchunks = max((kend + KB - 1) / KB, 1);
  const int c_lo = SPLIT ? split * nchunks / a.kv_splits : 0;
  const int c_hi = SPLIT ? (split + 1) * nchunks / a.kv_splits : nchunks;

  // staging: one block lookup per chunk, looked up a chunk ahead; loads unconditional (clamped key)
  fi::Codes<SEG / 2> kc, vc;
  uint32_t k_scale = 0, v_scale = 0;
  int id_next = 0, off_next = 0;
  bool bad_block = false;
  bool part_next = false, valid_next = true;
  const bool aligned = KB % a.block_size == 0;  // workgroup-uniform
  const int lane_blk = aligned ? lane / a.block_size : 0;
  const int lane_off = aligned ? lane - lane_blk * a.block_size : 0;
  const int chunk_blks = aligned ? KB / a.block_size : 0;
  auto lookup = [&](int c) {
    c = min(c, nchunks - 1);
    const int kpc = max(min(c * KB + lane, kend - 1), 0);
    const bool exact = aligned && c * KB + lane < kend;
    const int lb = exact ? c * chunk_blks + lane_blk : kpc / a.block_size;
    const bool in_table = lb < a.max_blocks;
    const int id = a.block_tables[(size_t)seq * a.max_blocks + (in_table ? lb : 0)];
    id_next = in_table ? id : -1;
    off_next = exact ? lane_off : kpc - lb * a.block_size;
  };
  auto fetch = [&](int c) {
    c = min(c, nchunks - 1);
    part_next = (c + 1) * KB > kend;  // workgroup-uniform: the chunk has padding keys
    valid_next = c * KB + lane < kend;
    const bool bad = id_next < 0 || id_next >= a.num_blocks;
    bad_block |= bad;
    const size_t row = ((size_t)(bad ? 0 : id_next) * a.hkv + kvh) * a.block_size + off_next;
    kc.load(k_codes + row * (D / 2) + w * (SEG / 2));
    vc.load(v_codes + row * (D / 2) + w * (SEG / 2));
    k_scale = k_scales[row * GROUPS + w * GROUPS / 4];
    v_scale = v_scales[row * GROUPS + w * GROUPS / 4];
  };
  // padding keys of a partial chunk are stored as zero (their clamped loads hold a valid row)
  auto stage = [&](int buf) {
    const bool pad = part_next && !valid_next;
    const bool nan = !pad && v_scale == 255u;
    const uint64_t nans = __builtin_amdgcn_ballot_w64(nan);
    if (lane == 0) s_nan[buf][w] = nans;
    const float ks = fi::fp4_scale_f32(pad ? 127u : k_scale), vs = fi::fp4_scale_f32(pad || nan ? 127u : v_scale);
#pragma unroll
    for (int j = 0; j < SEG / 8; ++j) {
      *reinterpret_cast<uint4*>(&Ks[buf][lane][w * SEG + 8 * j]) = fi::fp4_widen8(pad ? 0u : kc.w[j], ks);
      *reinterpret_cast<uint4*>(&Vs[buf][lane][w * SEG + 8 * j]) = fi::fp4_widen8(pad || nan ? 0u : vc.w[j], vs);
    }
  };

  lookup(c_lo);
  fetch(c_lo);
  lookup(c_lo + 1);
  stage(0);
  __syncthreads();
  for (int c = c_lo; c < c_hi; ++c) {
    const int k0 = c * KB;
    const int buf = (c - c_lo) & 1;
    fetch(c + 1);  // the last chunk re-reads itself: the loads stay unconditional
    lookup(c + 2);
    __builtin_amdgcn_sched_barrier(0);

    // ---- S^T = K Q^T: 64 keys x 16 rows per group ----
    v4f s_acc[RG][JT];
#pragma unroll
    for (int g = 0; g < RG; ++g)
#pragma unroll
      for (int jt = 0; jt < JT; ++jt) s_acc[g][jt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < DS; ++t) {
      bf16x8 kf[JT];
#pragma unroll
      for (int jt = 0; jt < JT; ++jt) kf[jt] = *reinterpret_cast<const bf16x8*>(&Ks[buf][16 * jt + li][32 * t + 8 * lk]);
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int g = 0; g < RG; ++g)
#pragma unroll
          for (int jt = 0; jt < JT; ++jt)
            s_acc[g][jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[jt], qf[g][t][p], s_acc[g][jt], 0, 0, 0);
    }
    // causal / context mask only where the chunk reaches past the tile's first query position
    if (k0 + KB - 1 > start + q0) {
#pragma unroll
      for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int jt = 0; jt < JT; ++jt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int kp = k0 + 16 * jt + 4 * lk + v;
            s_acc[g][jt][v] = (kp <= qpos[g] && kp < ctx) ? s_acc[g][jt][v] : -INFINITY;
          }
    }
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      float mx = -INFINITY;
#pragma unroll
      for (int jt = 0; jt < JT; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s_acc[g][jt][v]);
      mx = fmaxf(mx, fi::lane_xor16(mx, lane));
      mx = fmaxf(mx, fi::lane_xor32(mx, lane));
      const float m_chunk = mx * c2;
      const float m_new = m_chunk > m_row[g] + kLazy ? m_chunk : m_row[g];
      // no key seen yet (a split that starts past the row's position, keys that are NaN): the
      // reference point stays -inf; masked scores weigh 0 and NaN ones NaN against any finite point
      const float point = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = m_new == m_row[g] ? 1.0f : __builtin_amdgcn_exp2f(m_row[g] - m_new);
      m_row[g] = m_new;
      float ls = 0.0f;
#pragma unroll
      for (int jt = 0; jt < JT; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float pexp = __builtin_amdgcn_exp2f(fmaf(s_acc[g][jt][v], c2, -point));
          s_acc[g][jt][v] = pexp;
          ls += pexp;
        }
      l_part[g] = l_part[g] * alpha + ls;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[g][dt] *= alpha;
      }
    }

    // ---- O^T += V^T P^T (k index 8 lk + e of step u: key 32 u + 4 lk + e, e < 4, or 32 u + 16 + 4 lk + e - 4) ----
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      bf16x8 pp[RG][3];
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        const f32x8 pf = {s_acc[g][2 * u][0],     s_acc[g][2 * u][1],     s_acc[g][2 * u][2],     s_acc[g][2 * u][3],
                          s_acc[g][2 * u + 1][0], s_acc[g][2 * u + 1][1], s_acc[g][2 * u + 1][2], s_acc[g][2 * u + 1][3]};
        split3(pf, pp[g]);
      }
      // transposing reads as in prefill_bf16_kernel
      const int vrow = 32 * u + 4 * lk + (li >> 2), vcol = 4 * (li & 3);
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += DB) {
        bf16x8 vf[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const v4s lo = lds_read_tr16(&Vs[buf][vrow][16 * (d0 + i) + vcol]);
          const v4s hi = lds_read_tr16(&Vs[buf][vrow + 16][16 * (d0 + i) + vcol]);
          vf[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int g = 0; g < RG; ++g)
              o[g][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], pp[g][p], o[g][d0 + i], 0, 0, 0);
      }
    }
    // rows that see a key with a NaN group of V
    if ((s_nan[buf][0] | s_nan[buf][1] | s_nan[buf][2] | s_nan[buf][3]) != 0) {  // workgroup-uniform
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        const int last = min(qpos[g], ctx - 1) - k0;  // the last key of the chunk that the row sees
        const uint64_t seen = last < 0 ? 0 : (last >= 63 ? ~0ull : (2ull << last) - 1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          if (s_nan[buf][dt * 4 / DT] & seen) o[g][dt] = v4f{NAN, NAN, NAN, NAN};
      }
    }
    // the other buffer was last read in the chunk before, which every wave finished before the
    // previous barrier; this barrier publishes the next chunk and retires this one's buffer
    if (c + 1 < c_hi) stage(buf ^ 1);  // workgroup-uniform
    __syncthreads();
  }

  if (bad_block) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);

  // ---- normalise and store: lane holds row li of each group, d = 16 dt + 4 lk + v ----
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    float l_row = l_part[g] + fi::lane_xor16(l_part[g], lane);
    l_row += fi::lane_xor32(l_row, lane);
    const int row = 16 * (w + 4 * g) + li;
    if constexpr (SPLIT) {
      // this split's partials: O [rows][D] unnormalised, then (reference point, row sum) [rows].  A NaN
      // sum takes a finite point, which the merge does not skip; a row without any key is O = 0 over 1
      constexpr int ROWS = kRows * RG;
      const size_t unit = ((size_t)tile * a.kv_splits + split) * a.hkv + kvh;
      float* po = a.part + unit * ROWS * D + (size_t)row * D;
      float* pml = a.part + (size_t)gridDim.x * ROWS * D + (unit * ROWS + row) * 2;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4*>(po + 16 * dt + 4 * lk) = make_float4(o[g][dt][0], o[g][dt][1], o[g][dt][2], o[g][dt][3]);
      if (lk == 0)
        *reinterpret_cast<float2*>(pml) = qpos[g] < 0 ? make_float2(0.f, 1.f)
                                                      : make_float2(l_row != l_row ? 0.f : m_row[g], l_row);
    } else {
      const int h = row / QT, t = row % QT;
      if (h < a.group && q0 + t < qlen) {
        const float inv = qpos[g] < 0 ? 0.0f : 1.0f / l_row;
        float* op = a.out + ((size_t)(qs + q0 + t) * a.hq + kvh * a.group + h) * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<float4*>(op + 16 * dt + 4 * lk) =
              make_float4(o[g][dt][0] * inv, o[g][dt][1] * inv, o[g][dt][2] * inv, o[g][dt][3] * inv);
      }
    }
  }
}

template <int D, int RG, bool SPLIT>
void launch_g(fi_context* ctx, const PrefillArgs& args, dim3 grid, int g) {
  switch (g) {
    case 1:
      hipLaunchKernelGGL((prefill_fp4_kernel<D, 1, RG, SPLIT>), grid, dim3(kThreads), 0, ctx->stream, args);
      break;
    case 2:
      hipLaunchKernelGGL((prefill_fp4_kernel<D, 2, RG, SPLIT>), grid, dim3(kThreads), 0, ctx->stream, args);
      break;
    case 4:
      hipLaunchKernelGGL((prefill_fp4_kernel<D, 4, RG, SPLIT>), grid, dim3(kThreads), 0, ctx->stream, args);
      break;
    default:
      hipLaunchKernelGGL((prefill_fp4_kernel<D, 8, RG, SPLIT>), grid, dim3(kThreads), 0, ctx->stream, args);
      break;
  }
}

template <int D, int RG>
int32_t launch_rg(fi_context* ctx, PrefillArgs& args, int g) {
  const int qt = kRows * RG / g;
  // Key splits for launches that leave most workgroup slots empty, as for f32 pools: up to four
  // workgroups a CU, each with at least two chunks (a tile's keys are at least max_query_len).
  int splits = 1;
  if (RG == 1) {
    const long cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
    const long wgs = (long)((args.max_query_len + qt - 1) / qt) * args.num_seqs * args.hkv;
    splits = static_cast<int>(std::min<long>(FI_PREFILL_MAX_SPLITS, (4 * cus) / std::max<long>(wgs, 1)));
    splits = std::max(1, std::min(splits, args.max_query_len / (2 * kKeys)));
  }
  dim3 grid;
  FI_TRY(plan_tiles(ctx, args, qt, kKeys, "fi_attn_prefill_paged", &grid, splits, kRows * RG * (D + 2)));
  if constexpr (RG == 1) {
    if (splits > 1) {
      launch_g<D, RG, true>(ctx, args, grid, g);
      FI_CHECK_LAUNCH("prefill_fp4_kernel");
      const int ntiles = (args.max_query_len + qt - 1) / qt;
      hipLaunchKernelGGL((prefill_split_merge_kernel<D, RG>), dim3(grid.x / splits), dim3(kThreads), 0, ctx->stream,
                         args, qt, ntiles);
      FI_CHECK_LAUNCH("prefill_split_merge_kernel");
      return FI_OK;
    }
  }
  launch_g<D, RG, false>(ctx, args, grid, g);
  FI_CHECK_LAUNCH("prefill_fp4_kernel");
  return FI_OK;
}

template <int D>
int32_t launch_dim(fi_context* ctx, const PrefillArgs& args_in) {
  PrefillArgs args = args_in;
  const int g = args.group <= 1 ? 1 : (args.group <= 2 ? 2 : (args.group <= 4 ? 4 : 8));
  return row_groups(ctx, args, g) == 2 ? launch_rg<D, 2>(ctx, args, g) : launch_rg<D, 1>(ctx, args, g);
}

}  // namespace

namespace fi {

int32_t prefill_fp4(fi_context* ctx, const PrefillArgs& args, int32_t head_dim) {
  switch (head_dim) {
    case 32:
      return launch_dim<32>(ctx, args);
    case 64:
      return launch_dim<64>(ctx, args);
    default:
      return launch_dim<128>(ctx, args);
  }
}

}  // namespace fi
