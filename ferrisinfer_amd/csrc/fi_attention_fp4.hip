// Paged decode attention over a 4-bit KV pool (fi_fp4.h) on v_mfma_f32_16x16x32_bf16, in f32
// accuracy: K and V are exact in bf16, and the f32 operands they meet (query rows,
// probabilities) are carried as three bf16 pieces whose sum is the f32 value exactly.
//
// The pieces cost no extra products.  A 16x16 MFMA tile has sixteen columns; a kv head serves at
// most eight query heads.  Column 4 h + p of a tile is piece p of query head h (p = 3 is zero), so
// one tile carries four heads with their pieces, and the pieces' products are summed over the
// four lanes of a quad afterwards.
//   S^T = K Q^T: keys are the tile's rows.  Lane (m, kb) = (lane & 15, lane >> 4) holds key m's
//     codes of dims kb * D/4 .. + D/4 - 1, as they lie in memory (16 bytes at D = 128); MFMA j takes
//     dims kb * D/4 + 8 j + e as its k index 8 kb + e, and Q is read in the same order.
//   O^T = V^T P^T: dims are the rows.  The scores leave lane (n, kb) with keys 4 kb + r of each
//     16-key tile for its own column n, which is a B operand as it stands: no exchange between lanes.
//     Lane (m, kb) of A holds those keys' codes of dims m * D/16 .. + D/16 - 1.  A conversion yields two
//     neighbouring dims of one key in one register, so an operand register is (key, even dim | odd
//     dim), and the product is taken twice, against (p, 0) for the even dims and (0, p) for the odd
//     ones: sixteen MFMAs a 32-key step where eight would do, but no instruction to regroup the
//     values by key (32 a step), and B needs no packing.  The vector pipe is what this kernel runs
//     short of; the matrix pipe has the room.
#include <type_traits>

#include "fi_common.h"
#include "fi_decode.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// One move inside a quad, in the form that folds into the instruction that reads it (fi::dpp_mov's does
// not).
template <int kCtrl>
__device__ __forceinline__ uint32_t quad_move(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, 0xF, 0xF, true);
}

// Lane p of a quad ends with the sum of v[p] over the quad's four lanes: each step hands on the half
// of the values that the neighbour keeps (nine instructions, where four full sums take eight and the
// choice between them three, and leave four copies of each).
__device__ __forceinline__ float quad_scatter_sum(const v4f& v, bool odd, bool high) {
  float k0 = odd ? v[1] : v[0], x0 = odd ? v[0] : v[1];
  float k1 = odd ? v[3] : v[2], x1 = odd ? v[2] : v[3];
  k0 += __uint_as_float(quad_move<0xB1>(__float_as_uint(x0)));
  k1 += __uint_as_float(quad_move<0xB1>(__float_as_uint(x1)));
  const float k = high ? k1 : k0, x = high ? k0 : k1;
  return k + __uint_as_float(quad_move<0x4E>(__float_as_uint(x)));
}

// What lane r of the quad holds, for this lane's piece: a (pieces 0 and 1) or b (2 and 3).
template <int r>
__device__ __forceinline__ uint32_t quad_pick(uint32_t a, uint32_t b, bool high) {
  const uint32_t x = quad_move<r * 0x55>(a), y = quad_move<r * 0x55>(b);
  return high ? y : x;
}

// Piece p (0, 1, 2; 3: zero) of eight f32 values, as a bf16 operand.
__device__ __forceinline__ uint4 piece8(const float (&x)[8], int p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h, m, l;
    fi::split3_pk(x[2 * i], x[2 * i + 1], h, m, l);
    w[i] = p == 0 ? h : (p == 1 ? m : (p == 2 ? l : 0u));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- the merge of a head's partitions ----
// M = max m_p, L = sum l_p 2^(m_p - M), out = sum acc_p 2^(m_p - M) / L.  The partitions are summed in
// four strands, strand s taking p = s, s + 4, .. in order, and the strands then in order: the same
// arithmetic whether four waves take a strand each (decode_merge_fp4_kernel, any number of partitions)
// or one wave all four (the last-arriving workgroup of a partition launch, at most kMergeInline).
constexpr int kStrands = 4;
constexpr int kMergeInline = 16;

// NS strands from s0 on, of this lane's D / 64 dims (D = 32: of the lower half's one): the weighted
// sums, and the strands' shares of L.  BATCH partitions' loads are issued together, the first ones' with the
// statistics'.  MAXP: the partitions that a sequence may have.
template <int D, bool COHERENT, int NS, int BATCH, int MAXP>
__device__ __forceinline__ void merge_strands(const DecodeArgs& a, size_t head, int nparts, int s0, int lane,
                                              float (&sum)[NS][(D + 63) / 64], float (&share)[NS]) {
  constexpr int E = (D + 63) / 64;
  constexpr int STEP = NS == 1 ? kStrands : 1;  // from one of this wave's partitions to the next
  constexpr int PER = (MAXP / STEP + 63) / 64;  // partitions whose statistics a lane keeps
  static_assert(64 % BATCH == 0, "a batch's weights lie in one register");
  float* ml = a.part_ml + head * a.parts_per_seq * 2;
  float* acc = a.part_acc + head * a.parts_per_seq * D + (D < 64 ? lane % D : lane * E);
  const int mine = (nparts - s0 + STEP - 1) / STEP;  // this wave's partitions
  float v[BATCH][E];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) {
    const int p = min(s0 + b * STEP, nparts - 1);  // past the end: read and dropped
#pragma unroll
    for (int e = 0; e < E; ++e) v[b][e] = load_partial<COHERENT>(acc + (size_t)p * D + e);
  }
  float mx = -INFINITY;
#pragma unroll
  for (int p0 = 0; p0 < MAXP; p0 += 64)
    if (p0 + lane < nparts) mx = fmaxf(mx, load_partial<COHERENT>(&ml[2 * (p0 + lane)]));
  // lane i keeps the statistics of this wave's partitions i, i + 64, ..
  float w_own[PER], l_own[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int own = s0 + (lane + 64 * k) * STEP;
    w_own[k] = own < nparts ? load_partial<COHERENT>(&ml[2 * own]) : -INFINITY;
    l_own[k] = own < nparts ? load_partial<COHERENT>(&ml[2 * own + 1]) : 0.0f;
  }
  mx = fi::wave_max(mx);
  const float point = mx == -INFINITY ? 0.0f : mx;
  float wl = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    w_own[k] = __builtin_amdgcn_exp2f(w_own[k] - point);
    wl += l_own[k] * w_own[k];
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    share[s] = fi::wave_sum(NS == 1 || lane % NS == s ? wl : 0.0f);
#pragma unroll
    for (int e = 0; e < E; ++e) sum[s][e] = 0.0f;
  }
  for (int i0 = 0; i0 < mine; i0 += BATCH) {
    if (i0 > 0) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int p = min(s0 + (i0 + b) * STEP, nparts - 1);
#pragma unroll
        for (int e = 0; e < E; ++e) v[b][e] = load_partial<COHERENT>(acc + (size_t)p * D + e);
      }
    }
    const float weights = PER == 1 || i0 < 64 ? w_own[0] : w_own[PER - 1];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (i0 + b < mine) {  // wave-uniform
        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weights), (i0 + b) % 64));
#pragma unroll
        for (int e = 0; e < E; ++e) sum[b % NS][e] += v[b][e] * w;
      }
    }
  }
}

// One workgroup per query head, a wave a strand.  Bound by the chain of its loads: 64 heads of 196 partitions
// of 128 dims, 6.7 MB, in 6.6 us with 32 partitions' loads at a time (8.2 with 8, which is the faster one up
// to 64 partitions: one sequence of 60000 tokens over 2 heads of 64 15.0 against 18.1 us in all, 8 of 4000 9.4
// against 9.0).  Past 256 partitions (MAXP 512): 14 heads of 391 partitions of 64 dims, 1.4 MB, 8.5 us, of 256
// 5.0.
template <int D, int WT, int BATCH, int MAXP>
__global__ __launch_bounds__(64 * kStrands) void decode_merge_fp4_kernel(DecodeArgs a) {
  constexpr int E = (D + 63) / 64;
  __shared__ float s_sum[kStrands][D];
  __shared__ float s_share[kStrands];
  const size_t head = blockIdx.x;
  const int seq = static_cast<int>(blockIdx.x) / a.hq;
  const int ctx = min(a.context_lens[seq], a.parts_per_seq * kWaves * WT);  // clamped as in the partitions
  const int nparts = (ctx + kWaves * WT - 1) / (kWaves * WT);
  if (nparts <= 1) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  float sum[1][E], share[1];
  merge_strands<D, false, 1, BATCH, MAXP>(a, head, nparts, w, lane, sum, share);
  if (D >= 64 || lane < D) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_sum[w][lane * E + e] = sum[0][e];
  }
  if (lane == 0) s_share[w] = share[0];
  __syncthreads();
  if (threadIdx.x < D) {
    float out = s_sum[0][threadIdx.x], l = s_share[0];
#pragma unroll
    for (int s = 1; s < kStrands; ++s) {
      out += s_sum[s][threadIdx.x];
      l += s_share[s];
    }
    a.out[head * D + threadIdx.x] = out * (1.0f / l);
  }
}

// The end of a partition workgroup: the waves' (max, sum, acc) in LDS are combined in wave order.
// A sequence with one partition writes its normalised output; otherwise the partition's partial is
// stored, and where the launch merges by itself the last of the group's partitions merges them, a wave
// a head (the counters' protocol is combine_waves').
template <int D, int G, int WT>
__device__ __forceinline__ void combine_waves_fp4(const DecodeArgs& a, const HeadUnit& hu, int pairs, int pair, int part,
                                                  int nparts, int n_part, const float (*s_ml)[G][2],
                                                  const float (*s_acc)[G][D]) {
  const int tid = threadIdx.x, group = hu.heads;
  const int nw = (n_part + WT - 1) / WT;
  for (int i = tid; i < group * D; i += kThreads) {
    const int g = i / D, d = i - (i / D) * D;
    float mx = s_ml[0][g][0];
    for (int v = 1; v < nw; ++v) mx = fmaxf(mx, s_ml[v][g][0]);
    const float point = mx == -INFINITY ? 0.0f : mx;
    float l = 0.0f, sum = 0.0f;
    for (int v = 0; v < nw; ++v) {
      const float wgt = __builtin_amdgcn_exp2f(s_ml[v][g][0] - point);
      l += s_ml[v][g][1] * wgt;
      sum += s_acc[v][g][d] * wgt;
    }
    const size_t head = hu.head0 + g, slot = head * a.parts_per_seq + part;
    if (nparts == 1) {
      a.out[head * D + d] = sum * (1.0f / l);
    } else if (a.counters) {  // read by another workgroup of this launch: device-coherent stores
      __hip_atomic_store(&a.part_acc[slot * D + d], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0) {
        __hip_atomic_store(&a.part_ml[slot * 2], mx, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&a.part_ml[slot * 2 + 1], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    } else {
      a.part_acc[slot * D + d] = sum;
      if (d == 0) *reinterpret_cast<float2*>(&a.part_ml[slot * 2]) = make_float2(mx, l);
    }
  }
  if (nparts <= 1 || a.counters == nullptr) return;  // workgroup-uniform
  __shared__ int s_last;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const int unit = blockIdx.y * pairs + pair;
    const unsigned arrived =
        __hip_atomic_fetch_add(&a.counters[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    s_last = arrived == static_cast<unsigned>(nparts);
    if (s_last) __hip_atomic_store(&a.counters[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  constexpr int E = (D + 63) / 64;
  const int lane = tid & 63;
  for (int g = tid >> 6; g < group; g += kWaves) {
    const size_t head = hu.head0 + g;
    float sum[kStrands][E], share[kStrands];
    merge_strands<D, true, kStrands, 8, kMergeInline>(a, head, nparts, 0, lane, sum, share);
#pragma unroll
    for (int s = 1; s < kStrands; ++s) {
      share[0] += share[s];
#pragma unroll
      for (int e = 0; e < E; ++e) sum[0][e] += sum[s][e];
    }
    if (D >= 64 || lane < D) {
#pragma unroll
      for (int e = 0; e < E; ++e) a.out[head * D + lane * E + e] = sum[0][e] * (1.0f / share[0]);
    }
  }
}

// One workgroup = one (sequence, kv head, partition of kWaves * WT tokens), or in small launches a share of
// its query heads; each wave owns WT consecutive tokens, computes all their scores, then their
// softmax once, then the weighted sum.  T tiles of four query heads.  The waves' (max, sum, acc)
// are combined through LDS in wave order, the partitions by the last of them to arrive or in a launch
// of their own.
//
// QUAD (block sizes that are multiples of four): the pool rows of keys 4 i .. 4 i + 3 follow each
// other, so a lane's keys need one address and immediate offsets; the rows of the last group that lie past the
// end are read as they are (they are rows of the same block) and masked.  Otherwise every key has
// its own address, clamped to the last valid row.
//
// The wave's K codes, and V codes two steps ahead, are in flight together (a wave has 10 KB
// outstanding at D = 128).  114 registers at D = 128 and four heads leave four workgroups a CU, 24 of them
// hold one scale byte each, and 40 of a wave's 80 pool loads fetch one.  128 sequences of 512 to 8192 tokens over 8
// heads of 128, 610 MB of codes and scales (679 read), 142 us with the merge, 4.3 TB/s, where a large copy
// moves 4.7, a pure read of paged blocks 5.8, and the matrix pipe is busy 16 %; 64 of 128 to 2048 (78 MB) 24 us, 3.3
// TB/s, by the workgroups' own chain (rows, codes, scores, softmax, sum): 1328 of them with keys, 1024 at a time.
template <int D, int T, int WT, bool QUAD>
__global__ __launch_bounds__(kThreads, T == 1 ? 4 : 2) void decode_fp4_kernel(DecodeArgs a) {
  constexpr int kPartTokens = kWaves * WT;
  constexpr int G = 4 * T;        // query heads
  constexpr int STEPS = WT / 32;  // 32-key steps
  constexpr int KB = D / 8;       // bytes of K codes a lane holds of one key
  constexpr int KJ = D / 32;      // MFMAs of a score tile
  constexpr int VB = D / 32;      // bytes of V codes a lane holds of one key
  constexpr int VJ = D / 16;      // dims of a lane
  constexpr int VD = STEPS < 2 ? STEPS : 2;  // steps of V in flight
  constexpr int GROUPS = D / fi::kFp4Group;
  constexpr int QP = D + 8;  // padded LDS rows of the query operand
  constexpr int ROWS = QUAD ? kPartTokens / 4 : kPartTokens;
  static_assert(WT % 32 == 0, "a wave's tokens are whole steps");

  __shared__ uint32_t s_row[ROWS];  // pool rows of the partition's tokens (QUAD: of every fourth)
  __shared__ __align__(16) uint16_t s_q[16 * T][QP];
  __shared__ float s_ml[kWaves][G][2];
  __shared__ __align__(16) float s_acc[kWaves][G][D];

  const int pairs = a.num_seqs * a.hkv;
  const int part = blockIdx.z, pair = blockIdx.x;
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
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int m = lane & 15, kb = lane >> 4;
  const int piece = m & 3;
  const bool odd = piece & 1, high = piece >> 1;
  const int n = min(WT, n_part - w * WT);  // the wave's tokens (<= 0: idle wave)

  const size_t code_bytes = fi::fp4_code_bytes(a.num_blocks, a.hkv, a.block_size, D);
  // this lane's place in a row (QUAD: of key m & 3 of the K group whose row is looked up)
  const int k_row = QUAD ? m & 3 : 0;
  const uint8_t* __restrict__ k_codes = static_cast<const uint8_t*>(a.k_cache) + k_row * (D / 2) + kb * KB;
  const uint8_t* __restrict__ v_codes = static_cast<const uint8_t*>(a.v_cache) + m * VB;
  const uint8_t* __restrict__ k_scales =
      static_cast<const uint8_t*>(a.k_cache) + code_bytes + k_row * GROUPS + kb * GROUPS / 4;
  const uint8_t* __restrict__ v_scales = static_cast<const uint8_t*>(a.v_cache) + code_bytes + m * GROUPS / 16;

  // the partition's pool rows; entries past the end repeat the last one
  for (int i = tid; i < ROWS; i += kThreads) {
    const int last = QUAD ? (n_part - 1) & ~3 : n_part - 1;
    const int pos = t0 + min(QUAD ? 4 * i : i, last);
    const int lb = static_cast<int>(a.blocks.div(pos));
    int id = lb < a.max_blocks ? a.block_tables[(size_t)seq * a.max_blocks + lb] : -1;
    if (id < 0 || id >= a.num_blocks) {
      atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
      id = 0;
    }
    s_row[i] = (static_cast<uint32_t>(id) * a.hkv + kvh) * a.block_size + (pos - lb * a.block_size);
  }
  // the query operand, once for the workgroup: row 4 h + p is piece p of head h
  for (int i = tid; i < 16 * T * (D / 8); i += kThreads) {
    const int col = i / (D / 8), d = 8 * (i % (D / 8));
    const bool live = (col >> 2) < group;
    const float* qp = a.q + (head0 + (live ? col >> 2 : 0)) * D + d;
    const float4 lo = *reinterpret_cast<const float4*>(qp), hi = *reinterpret_cast<const float4*>(qp + 4);
    const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    *reinterpret_cast<uint4*>(&s_q[col][d]) = piece8(x, live ? col & 3 : 3);
  }
  __syncthreads();

  if (n > 0) {  // wave-uniform
    const uint32_t* rows = s_row + w * (QUAD ? WT / 4 : WT);
    fi::Codes<KB> kc[2 * STEPS];
    uint32_t ks[2 * STEPS];
#pragma unroll
    for (int i = 0; i < 2 * STEPS; ++i) {
      const int key = 16 * i + m;
      const size_t row = rows[QUAD ? key >> 2 : min(key, n - 1)];
      kc[i].load(k_codes + row * (D / 2));
      ks[i] = k_scales[row * GROUPS];
    }
    fi::Codes<VB> vc[VD][8];
    uint32_t vs[VD][8];
    // V of step s: keys 32 s + 4 kb + r and 16 more
    auto issue_v = [&](int s, fi::Codes<VB> (&c)[8], uint32_t (&sc)[8]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = 32 * s + 16 * i + 4 * kb;
        const size_t row = rows[QUAD ? key >> 2 : min(key, n - 1)];
        const uint8_t* pc = v_codes + row * (D / 2);
        const uint8_t* ps = v_scales + row * GROUPS;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!QUAD && e > 0) {
            const size_t own = rows[min(key + e, n - 1)];
            pc = v_codes + own * (D / 2) - e * (D / 2);
            ps = v_scales + own * GROUPS - e * GROUPS;
          }
          c[4 * i + e].load(pc + e * (D / 2));
          sc[4 * i + e] = ps[e * GROUPS];
        }
      }
    };
#pragma unroll
    for (int s = 0; s < VD; ++s) issue_v(s, vc[s], vs[s]);
    bf16x8 qf[T][KJ];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int j = 0; j < KJ; ++j)
        qf[t][j] = *reinterpret_cast<const bf16x8*>(&s_q[16 * t + m][kb * (D / 4) + 8 * j]);
    sched_fence();

    // ---- scores in log2 units: lane (4 h + r, kb) keeps keys 16 i + 4 kb + r of head h ----
    const float c2 = a.scale * 1.4426950408889634f;
    float sc[T][2 * STEPS];
    float mx[T];
#pragma unroll
    for (int t = 0; t < T; ++t) mx[t] = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2 * STEPS; ++i) {
      const float scale = fi::fp4_scale_f32(ks[i]);
      v4f acc[T];
#pragma unroll
      for (int t = 0; t < T; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, fi::fp4_widen8(kc[i].w[j], scale));
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][j], acc[t], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float v = quad_scatter_sum(acc[t], odd, high) * c2;
        sc[t][i] = 16 * i + 4 * kb + piece < n ? v : -INFINITY;
        mx[t] = fmaxf(mx[t], sc[t][i]);
      }
    }

    // ---- softmax over the wave's tokens ----
#pragma unroll
    for (int t = 0; t < T; ++t) {
      mx[t] = fmaxf(mx[t], __uint_as_float(quad_move<0xB1>(__float_as_uint(mx[t]))));
      mx[t] = fmaxf(mx[t], __uint_as_float(quad_move<0x4E>(__float_as_uint(mx[t]))));
      mx[t] = fmaxf(mx[t], fi::lane_xor16(mx[t], lane));
      mx[t] = fmaxf(mx[t], fi::lane_xor32(mx[t], lane));
      // every score -inf or NaN: weights 0 and NaN, against any finite point
      const float point = mx[t] == -INFINITY ? 0.0f : mx[t];
      float l = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * STEPS; ++i) {
        sc[t][i] = __builtin_amdgcn_exp2f(sc[t][i] - point);
        l += sc[t][i];
      }
      l = fi::group_sum<4>(l);
      l += fi::lane_xor16(l, lane);
      l += fi::lane_xor32(l, lane);
      if (kb == 0 && piece == 0) {
        s_ml[w][4 * t + (m >> 2)][0] = mx[t];
        s_ml[w][4 * t + (m >> 2)][1] = l;
      }
    }

    // ---- O^T += V^T P^T ----
    // A probability's pieces by truncation: h keeps the upper 16 bits of x (8 significant ones), m those
    // of x - h, and l = x - h - m is what is left, exactly (weights near 2^-126, whose pieces have fewer
    // bits, lose what lies below; the mask keeps it out of the lower half).  The lane that holds x packs (h, m) and (l, 0);
    // column 4 h + p takes piece p of the four keys from its quad's lanes, into the upper half (odd
    // dims) and the lower half (even dims) of a register.
    const uint32_t to_high = odd ? 0x05040c0cu : 0x07060c0cu, to_low = odd ? 0x0c0c0504u : 0x0c0c0706u;
    v4f o[T][VJ];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int j = 0; j < VJ; ++j) o[t][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      uint32_t be[T][8], bo[T][8];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = sc[t][2 * s + i];
          const uint32_t h = __float_as_uint(x) & 0xffff0000u;
          const float y = x - __uint_as_float(h);
          const uint32_t mid = __float_as_uint(y) & 0xffff0000u;
          const uint32_t rest = __float_as_uint(y - __uint_as_float(mid)) & 0xffff0000u;
          const uint32_t hm = __builtin_amdgcn_perm(h, mid, 0x07060302u);
          const uint32_t own[4] = {quad_pick<0>(hm, rest, high), quad_pick<1>(hm, rest, high),
                                   quad_pick<2>(hm, rest, high), quad_pick<3>(hm, rest, high)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bo[t][4 * i + r] = __builtin_amdgcn_perm(own[r], 0u, to_high);
            be[t][4 * i + r] = __builtin_amdgcn_perm(own[r], 0u, to_low);
          }
        }
      float scale[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) scale[e] = fi::fp4_scale_f32(vs[s % VD][e]);
      if (QUAD && 32 * s + 32 > n) {  // wave-uniform: rows past the end hold anything, a NaN scale too
#pragma unroll
        for (int e = 0; e < 8; ++e)
          scale[e] = 32 * s + (e < 4 ? 0 : 16) + 4 * kb + (e & 3) < n ? scale[e] : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < VJ; j += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t c = vc[s % VD][4 * i + e].w[0];
            const float sv = scale[4 * i + e];
            if (j == 0) x[e] = fi::fp4_widen2<0>(c, sv);
            if (j == 2) x[e] = fi::fp4_widen2<1>(c, sv);
            if (j == 4) x[e] = fi::fp4_widen2<2>(c, sv);
            if (j == 6) x[e] = fi::fp4_widen2<3>(c, sv);
          }
          const bf16x8 va = __builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3]));
#pragma unroll
          for (int t = 0; t < T; ++t) {
            const bf16x8 even = __builtin_bit_cast(bf16x8, make_uint4(be[t][4 * i], be[t][4 * i + 1], be[t][4 * i + 2], be[t][4 * i + 3]));
            const bf16x8 odd = __builtin_bit_cast(bf16x8, make_uint4(bo[t][4 * i], bo[t][4 * i + 1], bo[t][4 * i + 2], bo[t][4 * i + 3]));
            o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, even, o[t][j], 0, 0, 0);
            o[t][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, odd, o[t][j + 1], 0, 0, 0);
          }
        }
      }
      if (s + VD < STEPS) issue_v(s + VD, vc[s % VD], vs[s % VD]);
      sched_fence();
    }
    // lane (n, kb) holds dims (4 kb + r) * D/16 + j of its column; a quad's lanes store one r each
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float* dst = &s_acc[w][4 * t + (m >> 2)][(4 * kb + piece) * VJ];
#pragma unroll
      for (int j = 0; j < VJ; ++j) dst[j] = quad_scatter_sum(o[t][j], odd, high);
    }
  }
  __syncthreads();

  combine_waves_fp4<D, G, WT>(a, hu, pairs, pair, part, nparts, n_part, s_ml, s_acc);
}

template <int D, int T, int WT, bool QUAD>
int32_t launch(fi_context* ctx, const DecodeArgs& args, dim3 grid) {
  hipLaunchKernelGGL((decode_fp4_kernel<D, T, WT, QUAD>), grid, dim3(kThreads), 0, ctx->stream, args);
  FI_CHECK_LAUNCH("decode_fp4_kernel");
  if (args.parts_per_seq > 1 && args.counters == nullptr) {
    auto merge = args.parts_per_seq > 64 ? decode_merge_fp4_kernel<D, WT, 32, kMaxParts> : decode_merge_fp4_kernel<D, WT, 8, kMaxParts>;
    constexpr int kLongest = fi::kFp4MaxContext / (kWaves * WT);
    if constexpr (kLongest > kMaxParts) {  // narrow rows: two statistics a lane
      if (args.parts_per_seq > kMaxParts) merge = decode_merge_fp4_kernel<D, WT, 32, kLongest>;
    }
    hipLaunchKernelGGL(merge, dim3(static_cast<unsigned>(args.num_seqs) * args.hq), dim3(64 * kStrands), 0, ctx->stream,
                       args);
    FI_CHECK_LAUNCH("decode_merge_fp4_kernel");
  }
  return FI_OK;
}

template <int D, int T, int WT>
int32_t launch_quad(fi_context* ctx, const DecodeArgs& args, dim3 grid) {
  return args.block_size % 4 == 0 ? launch<D, T, WT, true>(ctx, args, grid) : launch<D, T, WT, false>(ctx, args, grid);
}

template <int D>
int32_t launch_dim(fi_context* ctx, const DecodeArgs& args, dim3 grid, int wt) {
  const bool wide = wt == FI_DECODE_WIDE_WAVE_TOKENS;
  if (args.heads_per <= 4)
    return wide ? launch_quad<D, 1, FI_DECODE_WIDE_WAVE_TOKENS>(ctx, args, grid)
                : launch_quad<D, 1, FI_DECODE_NARROW_WAVE_TOKENS>(ctx, args, grid);
  return wide ? launch_quad<D, 2, FI_DECODE_WIDE_WAVE_TOKENS>(ctx, args, grid)
              : launch_quad<D, 2, FI_DECODE_NARROW_WAVE_TOKENS>(ctx, args, grid);
}

}  // namespace

namespace fi {

bool decode_fp4_merges(int64_t workgroups, int parts, int heads, int64_t cus) {
  return parts <= kMergeInline / 2 || (parts <= kMergeInline && heads <= 4 && workgroups > 2 * cus);
}

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
