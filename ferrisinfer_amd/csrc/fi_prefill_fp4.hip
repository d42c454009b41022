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
// of codes and one scale byte each for K and V; the next chunk's codes are in registers (10 of them at
// D = 128) while the current one is multiplied.  One LDS buffer (36 KB at D = 128) and two barriers a chunk
// leave room for three workgroups a CU: 222 us for 16 prompts of 32 to 1024 tokens after up to 512 cached ones
// (32/8 heads of 128; 240 with two buffers and two workgroups), 359 TFLOP/s, three products a product:
// 1.08 PFLOP/s of bf16 products, where a large library product reaches 1.26 on the same card.  Measured and
// no faster: 32 rows a wave on 32x32x16 products (250), two 16-row groups a wave (234, at 256 registers),
// the next chunk's scores beside this one's softmax (255), K and V fragments read ahead (246).  The products
// take 45-50% of the time, the vector instructions about as much, and beside each other they overlap
// little: a 16x16x32 product costs another wave's vector instructions 5.8 ns of its 7.2.
//
// A NaN group of V must reach only the rows that see its key, though a chunk's product multiplies every
// key by every row (0 * NaN is NaN): it is staged as zeros, its key noted in a 64-bit mask of the
// chunk and column quarter, and the rows that see a noted key are set to NaN afterwards.  So is a group with a
// scale that appending never writes, 253 or 254, whose values may be infinite.
#include "fi_common.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"
#include "fi_prefill.h"

namespace {

// A chunk's way from the pool to LDS: KB keys, thread tid stages key tid % KB, elements
// seg * SEG .. + SEG - 1.  One block lookup per chunk, a chunk ahead of its loads; loads unconditional
// (clamped key), codes and scales in registers until they are widened into the chunk's planes.
template <int D, int KB>
struct ChunkLoader {
  static constexpr int SEG = D * KB / kThreads;
  static constexpr int GROUPS = D / fi::kFp4Group;
  static constexpr int KPK = D == 128 ? D + 16 : D + 8;  // padded LDS rows of K (see prefill_bf16_kernel)
  static constexpr int KP = D + 8;                       // of V (transposing reads)
  static_assert(KB == 64 && SEG % 8 == 0, "a wave stages a column quarter of every key, in whole dwords of codes");

  const uint8_t *k_codes, *v_codes, *k_scales, *v_scales;  // of this thread's segment
  const int* table;                                        // the sequence's blocks
  int max_blocks, num_blocks, hkv, kvh, block_size;
  int skey, kend, nchunks;
  bool aligned;  // blocks that divide the chunk: the key's block within it and its offset are constants
  int key_blk, key_off, chunk_blks;
  fi::Codes<SEG / 2> kc, vc;
  uint32_t k_scale, v_scale;
  int id_next, off_next;
  bool bad_block, part_next, valid_next;

  __device__ __forceinline__ void init(const PrefillArgs& a, int seq, int kv_head, int tid, int end, int chunks) {
    const size_t code_bytes = fi::fp4_code_bytes(a.num_blocks, a.hkv, a.block_size, D);
    const int seg = tid / KB;
    skey = tid % KB;
    k_codes = static_cast<const uint8_t*>(a.k_cache) + seg * (SEG / 2);
    v_codes = static_cast<const uint8_t*>(a.v_cache) + seg * (SEG / 2);
    k_scales = static_cast<const uint8_t*>(a.k_cache) + code_bytes + seg * SEG / fi::kFp4Group;
    v_scales = static_cast<const uint8_t*>(a.v_cache) + code_bytes + seg * SEG / fi::kFp4Group;
    table = a.block_tables + (size_t)seq * a.max_blocks;
    max_blocks = a.max_blocks;
    num_blocks = a.num_blocks;
    hkv = a.hkv;
    kvh = kv_head;
    block_size = a.block_size;
    kend = end;
    nchunks = chunks;
    aligned = KB % block_size == 0;  // workgroup-uniform
    key_blk = aligned ? skey / block_size : 0;
    key_off = aligned ? skey - key_blk * block_size : 0;
    chunk_blks = aligned ? KB / block_size : 0;
    bad_block = false;
  }
  __device__ __forceinline__ void lookup(int c) {
    c = min(c, nchunks - 1);
    const int kpc = max(min(c * KB + skey, kend - 1), 0);
    const bool exact = aligned && c * KB + skey < kend;
    const int lb = exact ? c * chunk_blks + key_blk : kpc / block_size;
    const bool in_table = lb < max_blocks;
    const int id = table[in_table ? lb : 0];
    id_next = in_table ? id : -1;
    off_next = exact ? key_off : kpc - lb * block_size;
  }
  __device__ __forceinline__ void fetch(int c) {
    c = min(c, nchunks - 1);
    part_next = (c + 1) * KB > kend;  // workgroup-uniform: the chunk has padding keys
    valid_next = c * KB + skey < kend;
    const bool bad = id_next < 0 || id_next >= num_blocks;
    bad_block |= bad && valid_next;  // a tile without keys looks up one block all the same
    const size_t row = ((size_t)(bad ? 0 : id_next) * hkv + kvh) * block_size + off_next;
    kc.load(k_codes + row * (D / 2));
    vc.load(v_codes + row * (D / 2));
    k_scale = k_scales[row * GROUPS];
    v_scale = v_scales[row * GROUPS];
  }
  // Padding keys of a partial chunk are stored as zero (their clamped loads hold a valid row); so is a
  // NaN (or overflowing) group of V, whose key goes into nan_keys[wave] (a wave stages a quarter of the columns).
  __device__ __forceinline__ void stage(uint16_t (*ks)[KPK], uint16_t (*vs)[KP], uint64_t* nan_keys, int tid) {
    const bool pad = part_next && !valid_next;
    const bool nan = !pad && v_scale > fi::kFp4MaxScale;
    const uint64_t nans = __builtin_amdgcn_ballot_w64(nan);
    if ((tid & 63) == 0) nan_keys[tid >> 6] = nans;
    const float k2 = fi::fp4_scale_f32(pad ? 127u : k_scale), v2 = fi::fp4_scale_f32(pad || nan ? 127u : v_scale);
    const int col = tid / KB * SEG;
#pragma unroll
    for (int j = 0; j < SEG / 8; ++j) {
      *reinterpret_cast<uint4*>(&ks[skey][col + 8 * j]) = fi::fp4_widen8(pad ? 0u : kc.w[j], k2);
      *reinterpret_cast<uint4*>(&vs[skey][col + 8 * j]) = fi::fp4_widen8(pad || nan ? 0u : vc.w[j], v2);
    }
  }
};

// The keys of a chunk from k0 on that a row at position qpos sees, as a mask.
__device__ __forceinline__ uint64_t seen_keys(int qpos, int kend, int k0) {
  const int last = min(qpos, kend - 1) - k0;
  return last < 0 ? 0 : (last >= 63 ? ~0ull : (2ull << last) - 1);
}

constexpr int kChunk = 64;      // keys
constexpr int kMaxSplits = 32;  // key splits of a tile, at most

// How many key splits a tile of `chunks` chunks runs as; the launch's other workgroups of it end at once.
__device__ __forceinline__ int tile_splits(const PrefillArgs& a, int chunks) {
  return max(1, min(a.kv_splits, chunks / a.split_chunks));
}

// The position of a sequence's first new row.  Below 0 its row sees no key; context lengths below 0 count as 0,
// for the difference to stay in 32 bits.
__device__ __forceinline__ int first_position(const PrefillArgs& a, int seq, int qlen) {
  return max(a.context_lens[seq], 0) - qlen;
}

// The end of the keys that a tile's last row sees, none past the block table's width (rows that ask for
// more are reported: a context length that is wrong must not make a loop of a billion chunks), and
// their chunks: at least one, of rows without keys too.
__device__ __forceinline__ int tile_end(const PrefillArgs& a, int start, int qlen, int q_end) {
  const int64_t width = (int64_t)a.max_blocks * a.block_size;
  return static_cast<int>(min((int64_t)start + min(qlen, q_end), min(width, (int64_t)0x7fffffff - kChunk)));
}
__device__ __forceinline__ int tile_chunks(int end) { return max((end + kChunk - 1) / kChunk, 1); }

template <int D, int G, bool SPLIT>
__global__ __launch_bounds__(kThreads, 3) void prefill_fp4_kernel(PrefillArgs a) {
  constexpr int QT = kRows / G;    // query tokens per workgroup
  constexpr int KB = kChunk;
  constexpr int DS = D / 32;             // 32-wide d steps of Q K^T
  constexpr int DT = D / 16;             // 16-wide output d tiles of P V
  constexpr int JT = KB / 16;            // 16-key score tiles per chunk
  constexpr int KS = KB / 32;            // 32-key steps of P V
  constexpr int DB = DT < 4 ? DT : 4;    // d tiles whose V fragments are held at once
  using Loader = ChunkLoader<D, KB>;
  __shared__ __align__(16) uint16_t Ks[KB][Loader::KPK];
  __shared__ __align__(16) uint16_t Vs[KB][Loader::KP];
  __shared__ uint64_t s_nan[4];  // keys whose V group is NaN, by column quarter

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
  const int start = first_position(a, seq, qlen);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, lk = lane >> 4;
  const int row = 16 * w + li;
  const int qpos = start + q0 + row % QT;
  const int kend = tile_end(a, start, qlen, q0 + QT);
  const int nchunks = tile_chunks(kend);
  const int splits = SPLIT ? tile_splits(a, nchunks) : 1;
  if (SPLIT && split >= splits) return;

  // Q pieces: B operand row li, d = 32 t + 8 lk .. + 7
  bf16x8 qf[DS][3];
  {
    const int ah = row / QT, at = row % QT;
    const bool a_ok = ah < a.group && q0 + at < qlen;
    const float* qp = a.q + ((size_t)(qs + q0 + (a_ok ? at : 0)) * a.hq + kvh * a.group + (a_ok ? ah : 0)) * D + 8 * lk;
#pragma unroll
    for (int t = 0; t < DS; ++t) {
      const float4 lo = *reinterpret_cast<const float4*>(qp + 32 * t);
      const float4 hi = *reinterpret_cast<const float4*>(qp + 32 * t + 4);
      const f32x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      split3(a_ok ? v : z, qf[t]);
    }
  }
  v4f o[DT];  // O^T tile dt: d = 16 dt + 4 lk + v, row li
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
  float m_row = -INFINITY, l_part = 0.0f;
  const float c2 = a.scale * 1.4426950408889634f;  // scores -> log2 units
  constexpr float kLazy = 8.0f;  // headroom of the exponents' reference point (log2 units)

  const int c_lo = SPLIT ? split * nchunks / splits : 0;
  const int c_hi = SPLIT ? (split + 1) * nchunks / splits : nchunks;
  Loader in;
  in.init(a, seq, kvh, tid, kend, nchunks);

  in.lookup(c_lo);
  in.fetch(c_lo);
  in.lookup(c_lo + 1);
  in.stage(Ks, Vs, s_nan, tid);
  __syncthreads();
  for (int c = c_lo; c < c_hi; ++c) {
    const int k0 = c * KB;
    in.fetch(c + 1);  // the last chunk re-reads itself: the loads stay unconditional
    in.lookup(c + 2);
    __builtin_amdgcn_sched_barrier(0);

    // ---- S^T = K Q^T: 64 keys x 16 rows ----
    v4f s[JT];
#pragma unroll
    for (int jt = 0; jt < JT; ++jt) s[jt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < DS; ++t) {
      bf16x8 kf[JT];
#pragma unroll
      for (int jt = 0; jt < JT; ++jt) kf[jt] = *reinterpret_cast<const bf16x8*>(&Ks[16 * jt + li][32 * t + 8 * lk]);
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int jt = 0; jt < JT; ++jt)
          s[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[jt], qf[t][p], s[jt], 0, 0, 0);
    }
    // causal / context mask only where the chunk reaches past the tile's first query position or its keys
    if (k0 + KB - 1 > min(start + q0, kend - 1)) {
#pragma unroll
      for (int jt = 0; jt < JT; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int kp = k0 + 16 * jt + 4 * lk + v;
          s[jt][v] = (kp <= qpos && kp < kend) ? s[jt][v] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[jt][v]);
    mx = fmaxf(mx, fi::lane_xor16(mx, lane));
    mx = fmaxf(mx, fi::lane_xor32(mx, lane));
    const float m_chunk = mx * c2;
    const float m_new = m_chunk > m_row + kLazy ? m_chunk : m_row;
    // no key seen yet (a split that starts past the row's position, keys that are NaN): the
    // reference point stays -inf; masked scores weigh 0 and NaN ones NaN against any finite point
    const float point = m_new == -INFINITY ? 0.0f : m_new;
    // rows whose point moved (after the first chunks, hardly any)
    if (__builtin_amdgcn_ballot_w64(m_new != m_row) != 0) {
      const float alpha = m_new == m_row ? 1.0f : __builtin_amdgcn_exp2f(m_row - m_new);
      l_part *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
    m_row = m_new;
    float ls = 0.0f;
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        s[jt][v] = __builtin_amdgcn_exp2f(fmaf(s[jt][v], c2, -point));
        ls += s[jt][v];
      }
    l_part += ls;

    // ---- O^T += V^T P^T (k index 8 lk + e of step u: key 32 u + 4 lk + e, e < 4, or 32 u + 16 + 4 lk + e - 4) ----
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const f32x8 pf = {s[2 * u][0],     s[2 * u][1],     s[2 * u][2],     s[2 * u][3],
                        s[2 * u + 1][0], s[2 * u + 1][1], s[2 * u + 1][2], s[2 * u + 1][3]};
      bf16x8 pp[3];
      split3(pf, pp);
      // transposing reads as in prefill_bf16_kernel
      const int vrow = 32 * u + 4 * lk + (li >> 2), vcol = 4 * (li & 3);
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += DB) {
        bf16x8 vf[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const v4s lo = lds_read_tr16(&Vs[vrow][16 * (d0 + i) + vcol]);
          const v4s hi = lds_read_tr16(&Vs[vrow + 16][16 * (d0 + i) + vcol]);
          vf[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int i = 0; i < DB; ++i)
            o[d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], pp[p], o[d0 + i], 0, 0, 0);
      }
    }
    // rows that see a key with a NaN group of V
    if ((s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3]) != 0) {  // workgroup-uniform
      const uint64_t seen = seen_keys(qpos, kend, k0);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        if (s_nan[dt * 4 / DT] & seen) o[dt] = v4f{NAN, NAN, NAN, NAN};
    }
    __syncthreads();  // every wave is done with this chunk's K and V
    if (c + 1 < c_hi) {  // workgroup-uniform
      in.stage(Ks, Vs, s_nan, tid);
      __syncthreads();
    }
  }

  if (in.bad_block || kend < (int64_t)start + min(qlen, q0 + QT)) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);

  float l_row = l_part + fi::lane_xor16(l_part, lane);
  l_row += fi::lane_xor32(l_row, lane);
  if constexpr (SPLIT) {
    // this split's partials: O [rows][D] unnormalised, then (reference point, row sum) [rows].  A NaN
    // sum takes a finite point, which the merge does not skip; a row without any key is O = 0 over 1
    const size_t unit = ((size_t)tile * a.kv_splits + split) * a.hkv + kvh;
    float* po = a.part + unit * kRows * D + (size_t)row * D;
    float* pml = a.part + (size_t)gridDim.x * kRows * D + (unit * kRows + row) * 2;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(po + 16 * dt + 4 * lk) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
    if (lk == 0)
      *reinterpret_cast<float2*>(pml) = qpos < 0 ? make_float2(0.f, 1.f) : make_float2(l_row != l_row ? 0.f : m_row, l_row);
  } else {
    const int h = row / QT, t = row % QT;
    if (h < a.group && q0 + t < qlen) {
      const float inv = qpos < 0 ? 0.0f : 1.0f / l_row;
      float* op = a.out + ((size_t)(qs + q0 + t) * a.hq + kvh * a.group + h) * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4*>(op + 16 * dt + 4 * lk) =
            make_float4(o[dt][0] * inv, o[dt][1] * inv, o[dt][2] * inv, o[dt][3] * inv);
    }
  }
}

// One output row quad a thread: the splits' partials of its row combined in split order, four loaded at a
// time, each rescaled from its own reference point to the largest so far (a split without a key that the
// row sees carries -inf and adds nothing; the one with key 0 always has one), divided by the combined sum.
template <int D>
__global__ __launch_bounds__(kThreads) void prefill_merge_fp4_kernel(PrefillArgs a, int qt_tokens, int ntiles) {
  constexpr int DQ = D / 4, BLOCKS = kRows * DQ / kThreads;  // workgroups a (tile, kv head)
  constexpr int N = 4;
  const int pair = blockIdx.x / BLOCKS, idx = blockIdx.x % BLOCKS * kThreads + threadIdx.x;
  const int tile = pair / a.hkv, kvh = pair % a.hkv;
  const int seq = tile / ntiles, q0 = (tile % ntiles) * qt_tokens;
  const int qs = a.cu_seqlens[seq], qlen = a.cu_seqlens[seq + 1] - qs;
  const int r = idx / DQ, dq = idx % DQ;
  const int h = r / qt_tokens, t = r % qt_tokens;
  if (h >= a.group || q0 + t >= qlen) return;
  const int splits = tile_splits(a, tile_chunks(tile_end(a, first_position(a, seq, qlen), qlen, q0 + qt_tokens)));
  const size_t units = (size_t)(gridDim.x / BLOCKS) * a.kv_splits;
  const float* pml = a.part + units * kRows * D;
  const size_t first = (size_t)tile * a.kv_splits * a.hkv + kvh;  // split s: first + s * hkv
  float mx = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < splits; s0 += N) {
    float2 ml[N];
    float4 o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const size_t unit = first + (size_t)min(s0 + i, splits - 1) * a.hkv;
      ml[i] = *reinterpret_cast<const float2*>(pml + (unit * kRows + r) * 2);
      o[i] = *reinterpret_cast<const float4*>(a.part + (unit * kRows + r) * D + 4 * dq);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (s0 + i >= splits || ml[i].x == -INFINITY) continue;
      const float to = fmaxf(mx, ml[i].x);
      const float old = __builtin_amdgcn_exp2f(mx - to), now = __builtin_amdgcn_exp2f(ml[i].x - to);
      mx = to;
      l = l * old + now * ml[i].y;
      acc = make_float4(acc.x * old + now * o[i].x, acc.y * old + now * o[i].y, acc.z * old + now * o[i].z,
                        acc.w * old + now * o[i].w);
    }
  }
  const float inv = 1.0f / l;
  *reinterpret_cast<float4*>(a.out + ((size_t)(qs + q0 + t) * a.hq + kvh * a.group + h) * D + 4 * dq) =
      make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <int D, int G>
void launch_group(fi_context* ctx, const PrefillArgs& args, dim3 grid) {
  if (args.kv_splits > 1) {
    hipLaunchKernelGGL((prefill_fp4_kernel<D, G, true>), grid, dim3(kThreads), 0, ctx->stream, args);
  } else {
    hipLaunchKernelGGL((prefill_fp4_kernel<D, G, false>), grid, dim3(kThreads), 0, ctx->stream, args);
  }
}

template <int D>
int32_t launch_dim(fi_context* ctx, const PrefillArgs& args_in) {
  PrefillArgs args = args_in;
  const int g = args.group <= 1 ? 1 : (args.group <= 2 ? 2 : (args.group <= 4 ? 4 : 8));
  const int qt = kRows / g;
  // Key splits for launches that leave workgroup slots empty: up to three workgroups a CU, the most that
  // run at a time, and (tile_splits) four chunks of keys or more each.  What the host knows of a tile's
  // chunks is the block tables' width less half of the new rows, the mean over a sequence's tiles (500 rows
  // after none over 14/2 heads of 64, tiles of one to eight chunks: 17.9 us with the longer ones cut, 14.6
  // whole).  32/8 heads of 128, us cut against whole: 64 rows after 1000 cached 20.9 against 44, after 4000 33 against
  // 124, after 16000 59 against 468.  Where the launch has a workgroup for half the CUs without them, eight
  // chunks: the partials' way through memory costs a range 3 us (300 rows after 8000 112 against 246, 300
  // after 2000 50 and with sixteen chunks 59, four sequences of 100 after up to 4000 67 and with sixteen 80, but of
  // 100 after up to 1000 43 and with sixteen 40, 500 after 500 36 and with six 45; 1000 after 4000, two workgroups
  // a CU without splits, 194 against 188).
  const int64_t cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int64_t wgs = static_cast<int64_t>((args.max_query_len + qt - 1) / qt) * args.num_seqs * args.hkv;
  const int64_t chunks = (static_cast<int64_t>(args.max_blocks) * args.block_size + kChunk - 1) / kChunk -
                         args.max_query_len / (2 * kChunk);
  args.split_chunks = 2 * wgs <= cus ? 4 : 8;
  const int splits = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({kMaxSplits, 3 * cus / std::max<int64_t>(wgs, 1), chunks / args.split_chunks})));
  dim3 grid;
  FI_TRY(plan_tiles(ctx, args, qt, 64, "fi_attn_prefill_paged", &grid, splits, kRows * (D + 2)));
  switch (g) {
    case 1:
      launch_group<D, 1>(ctx, args, grid);
      break;
    case 2:
      launch_group<D, 2>(ctx, args, grid);
      break;
    case 4:
      launch_group<D, 4>(ctx, args, grid);
      break;
    default:
      launch_group<D, 8>(ctx, args, grid);
      break;
  }
  FI_CHECK_LAUNCH("prefill_fp4_kernel");
  if (splits > 1) {
    const int ntiles = (args.max_query_len + qt - 1) / qt;
    const unsigned blocks = kRows * (D / 4) / kThreads;  // of the merge, a (tile, kv head)
    hipLaunchKernelGGL((prefill_merge_fp4_kernel<D>), dim3(grid.x / splits * blocks), dim3(kThreads), 0, ctx->stream, args,
                       qt, ntiles);
    FI_CHECK_LAUNCH("prefill_merge_fp4_kernel");
  }
  return FI_OK;
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
