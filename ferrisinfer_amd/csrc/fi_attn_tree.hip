// Attention of a tree's rows over the paged pool, in f32 accuracy on v_mfma_f32_16x16x32_bf16.  Node i of
// sequence b attends the cached prefix and the nodes whose bits its mask row has set, read in the pool
// behind the prefix.  No counterpart in the reference, whose sessions feed one sampled token a step
// (crates/ferrisinfer-runtime/src/session.rs:246-262).
//
// Rows are packed: row r of a (sequence, kv head) is head r % G of node r / G, so that any group size fills
// 64-row tiles (four waves of 16 rows).  The keys are cut into parts of part_chunks chunks, one workgroup a
// (part, sequence, kv head, tile); a sequence of several parts stores unnormalised partials that
// tree_merge_kernel joins.  The products are the prefill kernels': S^T = K Q^T leaves a lane the scores of
// one row, O^T = V^T P^T takes them as its B operand from registers, the f32 operands go as three bf16
// pieces (x = hi + mid + lo exactly), and the exponents' reference point moves only when a chunk's maximum
// passes it by 2^8.  K and V of bf16 and 4-bit pools are exact in bf16 (three products a product), f32 pools'
// are split as well (the six cross products above 2^-24).
//
// Only chunks that reach past the prefix (one or two a tile of up to 64 nodes) look at masks.  There an element of V that is
// not finite must reach only the rows that see its key, though the product multiplies every key by every row
// (0 * NaN is NaN): it is staged as zero, its key noted, and added afterwards to the rows that see it.
#include <algorithm>

#include "fi_common.h"
#include "fi_device.h"
#include "fi_fp4.h"
#include "fi_fp4_ops.h"
#include "fi_mfma.h"
#include "fi_tree.h"

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 64;  // (node, head) rows of a workgroup

struct TreeArgs {
  const float* q;  // [T, Hq, D]
  const void* k_cache;
  const void* v_cache;
  const int* block_tables;   // [B, max_blocks]
  const int* cu_seqlens;     // [B + 1]
  const int* context_lens;   // [B]
  const uint64_t* mask;      // [T, words]
  float* out;                // [T, Hq, D]
  float* part_acc;           // [B * max_query_len * Hq * parts, D]
  float* part_ml;            // [.., 2]
  uint32_t* faults;
  int words, max_blocks, hq, hkv, group, block_size, num_blocks;
  int num_seqs, max_query_len, max_context_len;
  int ntiles, parts, part_chunks;
  float scale;
  fi::FastDiv by_block, by_group;
};

// The keys of a sequence that the launch reads (lengths past max_context_len are cut off there), and the
// parts that they make: one at least, for rows without keys too.
__device__ __forceinline__ int key_end(const TreeArgs& a, const fi::TreeSpan& t) {
  return min(t.prefix + t.nodes, a.max_context_len);
}
template <int KB>
__device__ __forceinline__ int key_parts(const TreeArgs& a, int kend) {
  return max(1, (kend + KB * a.part_chunks - 1) / (KB * a.part_chunks));
}

// ---- a chunk's way from the pool to LDS ----
// A thread holds PT pieces of K and of V in registers, piece r of key tid / LANES + r * (256 / LANES); LANES
// neighbouring lanes read a whole row.
template <int POOL, int D>
struct Pool;

template <int D>
struct Pool<FI_DTYPE_BF16, D> {
  static constexpr int KB = 64, PLANES = 1, LANES = D / 8, PT = KB * LANES / kThreads;
  uint4 k[PT], v[PT];
  __device__ __forceinline__ void load(int r, const TreeArgs& a, size_t row, int col) {
    k[r] = reinterpret_cast<const uint4*>(a.k_cache)[row * LANES + col];
    v[r] = reinterpret_cast<const uint4*>(a.v_cache)[row * LANES + col];
  }
  __device__ __forceinline__ void zero(int r) { k[r] = v[r] = make_uint4(0u, 0u, 0u, 0u); }
  static __device__ __forceinline__ bool special(uint32_t& w) {
    const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
    w = (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
    return lo || hi;
  }
  // clears what is not finite in V
  __device__ __forceinline__ bool clean(int r) {
    const bool x = special(v[r].x), y = special(v[r].y), z = special(v[r].z), w = special(v[r].w);
    return x || y || z || w;
  }
  template <int KP, int VP, int K>
  __device__ __forceinline__ void store(int r, int key, int col, uint16_t (&ks)[PLANES][K][KP], uint16_t (&vs)[PLANES][K][VP]) {
    *reinterpret_cast<uint4*>(&ks[0][key][8 * col]) = k[r];
    *reinterpret_cast<uint4*>(&vs[0][key][8 * col]) = v[r];
  }
  static __device__ __forceinline__ float value(const TreeArgs& a, size_t row, int d) {
    return fi::bf16_bits_to_f32(static_cast<const uint16_t*>(a.v_cache)[row * D + d]);
  }
};

template <int D>
struct Pool<FI_DTYPE_F32, D> {
  static constexpr int KB = 32, PLANES = 3, LANES = D / 4, PT = KB * LANES / kThreads;
  float4 k[PT], v[PT];
  __device__ __forceinline__ void load(int r, const TreeArgs& a, size_t row, int col) {
    k[r] = reinterpret_cast<const float4*>(a.k_cache)[row * LANES + col];
    v[r] = reinterpret_cast<const float4*>(a.v_cache)[row * LANES + col];
  }
  __device__ __forceinline__ void zero(int r) { k[r] = v[r] = make_float4(0.f, 0.f, 0.f, 0.f); }
  static __device__ __forceinline__ bool special(float& x) {
    const bool s = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
    x = s ? 0.0f : x;
    return s;
  }
  __device__ __forceinline__ bool clean(int r) {
    const bool x = special(v[r].x), y = special(v[r].y), z = special(v[r].z), w = special(v[r].w);
    return x || y || z || w;
  }
  template <int KP, int VP, int K>
  __device__ __forceinline__ void store(int r, int key, int col, uint16_t (&ks)[PLANES][K][KP], uint16_t (&vs)[PLANES][K][VP]) {
    uint2 pk[3], pv[3];
    fi::split3_pk(k[r].x, k[r].y, pk[0].x, pk[1].x, pk[2].x);
    fi::split3_pk(k[r].z, k[r].w, pk[0].y, pk[1].y, pk[2].y);
    fi::split3_pk(v[r].x, v[r].y, pv[0].x, pv[1].x, pv[2].x);
    fi::split3_pk(v[r].z, v[r].w, pv[0].y, pv[1].y, pv[2].y);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      *reinterpret_cast<uint2*>(&ks[p][key][4 * col]) = pk[p];
      *reinterpret_cast<uint2*>(&vs[p][key][4 * col]) = pv[p];
    }
  }
  static __device__ __forceinline__ float value(const TreeArgs& a, size_t row, int d) {
    return static_cast<const float*>(a.v_cache)[row * D + d];
  }
};

// A thread holds a quarter of a row: D / 4 elements, a group at D = 128, its codes and scale byte.
template <int D>
struct Pool<FI_DTYPE_MXFP4, D> {
  static constexpr int KB = 64, PLANES = 1, LANES = 4, PT = 1, SEG = D / 4, GROUPS = D / fi::kFp4Group;
  fi::Codes<SEG / 2> k, v;
  uint32_t ks8, vs8;
  static __device__ __forceinline__ size_t code_bytes(const TreeArgs& a) {
    return fi::fp4_code_bytes(a.num_blocks, a.hkv, a.block_size, D);
  }
  __device__ __forceinline__ void load(int, const TreeArgs& a, size_t row, int col) {
    const uint8_t *kp = static_cast<const uint8_t*>(a.k_cache), *vp = static_cast<const uint8_t*>(a.v_cache);
    k.load(kp + row * (D / 2) + col * (SEG / 2));
    v.load(vp + row * (D / 2) + col * (SEG / 2));
    const size_t at = code_bytes(a) + row * GROUPS + col * SEG / fi::kFp4Group;
    ks8 = kp[at];
    vs8 = vp[at];
  }
  __device__ __forceinline__ void zero(int) {
#pragma unroll
    for (int j = 0; j < SEG / 8; ++j) k.w[j] = v.w[j] = 0u;
    ks8 = vs8 = 127u;
  }
  __device__ __forceinline__ bool clean(int) {
    if (vs8 <= fi::kFp4MaxScale) return false;
#pragma unroll
    for (int j = 0; j < SEG / 8; ++j) v.w[j] = 0u;
    vs8 = 127u;
    return true;
  }
  template <int KP, int VP, int K>
  __device__ __forceinline__ void store(int, int key, int col, uint16_t (&ks)[PLANES][K][KP], uint16_t (&vs)[PLANES][K][VP]) {
    const float k2 = fi::fp4_scale_f32(ks8), v2 = fi::fp4_scale_f32(vs8);
#pragma unroll
    for (int j = 0; j < SEG / 8; ++j) {
      *reinterpret_cast<uint4*>(&ks[0][key][col * SEG + 8 * j]) = fi::fp4_widen8(k.w[j], k2);
      *reinterpret_cast<uint4*>(&vs[0][key][col * SEG + 8 * j]) = fi::fp4_widen8(v.w[j], v2);
    }
  }
  // NaN, whatever the code, for the scales that clean() takes out (253 and 254 are not for a host to write)
  static __device__ __forceinline__ float value(const TreeArgs& a, size_t row, int d) {
    const uint32_t s = static_cast<const uint8_t*>(a.v_cache)[code_bytes(a) + row * GROUPS + d / fi::kFp4Group];
    return s > fi::kFp4MaxScale ? NAN : 0.0f;
  }
};

// acc += A B over the operands' pieces, smallest products first
template <int PLANES>
__device__ __forceinline__ v4f product(const bf16x8 (&x)[PLANES], const bf16x8 (&f)[3], v4f acc) {
  if constexpr (PLANES == 3) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[2], f[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], f[2], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], f[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], f[0], acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], f[2], acc, 0, 0, 0);
  }
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], f[1], acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], f[0], acc, 0, 0, 0);
}

template <int D, int POOL>
__global__ __launch_bounds__(kThreads, 2) void attn_tree_kernel(TreeArgs a) {
  using P = Pool<POOL, D>;
  constexpr int KB = P::KB, PLANES = P::PLANES, PT = P::PT, LANES = P::LANES;
  constexpr int DS = D / 32;             // 32-wide d steps of Q K^T
  constexpr int DT = D / 16;             // 16-wide output d tiles of P V
  constexpr int JT = KB / 16;            // 16-key score tiles per chunk
  constexpr int KS = KB / 32;            // 32-key steps of P V
  constexpr int KPK = D == 128 && PLANES == 1 ? D + 16 : D + 8;  // padded LDS rows of K (see prefill_bf16_kernel)
  constexpr int KPV = D + 8;                                     // of V (transposing reads)
  __shared__ __align__(16) uint16_t Ks[PLANES][KB][KPK];
  __shared__ __align__(16) uint16_t Vs[PLANES][KB][KPV];
  __shared__ unsigned long long s_special[2];  // by the chunk's parity: keys whose V is not finite throughout

  // the tiles of a (part, sequence, kv head) run one after the other on one XCD (workgroup L runs on XCD
  // L % 8), whose L2 then holds the keys that they share
  const int slot = blockIdx.x >> 3;
  const int unit = slot / a.ntiles * 8 + (blockIdx.x & 7), tile = slot % a.ntiles;
  if (unit >= a.parts * a.num_seqs * a.hkv) return;
  const int kvh = unit % a.hkv, seq = unit / a.hkv % a.num_seqs, part = unit / a.hkv / a.num_seqs;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, lk = lane >> 4;

  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, seq);
  const int nodes = min(t.nodes, a.max_query_len);
  if (part == 0 && tile == 0 && kvh == 0 && tid == 0) {
    if (t.nodes > a.max_query_len) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
    if (t.prefix + t.nodes > a.max_context_len) atomicOr(a.faults, FI_FAULT_CONTEXT_RANGE);
  }
  if (tile * kRows >= nodes * a.group) return;
  const int kend = key_end(a, t);
  const int nchunks = (kend + KB - 1) / KB;
  const int nparts = key_parts<KB>(a, kend);
  if (part >= nparts) return;
  const int c_lo = part * a.part_chunks, c_hi = min(c_lo + a.part_chunks, nchunks);

  const int r = tile * kRows + 16 * w + li;
  const int node = static_cast<int>(a.by_group.div(r)), head = kvh * a.group + (r - node * a.group);
  const bool live = node < nodes;
  const size_t row = (size_t)(t.first + (live ? node : 0)) * a.hq + head;
  const uint64_t* mask = a.mask + (size_t)(t.first + (live ? node : 0)) * a.words;

  // Q pieces: B operand row li, d = 32 s + 8 lk .. + 7
  bf16x8 qf[DS][3];
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    const float* qp = a.q + row * D + 32 * s + 8 * lk;
    const float4 lo = *reinterpret_cast<const float4*>(qp), hi = *reinterpret_cast<const float4*>(qp + 4);
    const f32x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    split3(live ? v : z, qf[s]);
  }
  v4f o[DT];  // O^T tile dt: d = 16 dt + 4 lk + v, row li
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
  float m_row = -INFINITY, l_part = 0.0f;
  const float c2 = a.scale * 1.4426950408889634f;  // scores -> log2 units
  constexpr float kLazy = 8.0f;  // headroom of the exponents' reference point (log2 units)

  // Staging: a wave's lanes look up the blocks of a chunk's keys, a chunk ahead of its loads; a thread takes
  // its keys' from them.  Loads are unconditional (clamped keys; the last chunk re-reads itself).
  P in;
  int id_next = 0, off_next = 0;
  bool bad_block = false;
  const int* table = a.block_tables + (size_t)seq * a.max_blocks;
  auto lookup = [&](int c) {
    const int kp = min(min(c, c_hi - 1) * KB + lane % KB, kend - 1);
    const int lb = static_cast<int>(a.by_block.div(kp));
    id_next = table[lb];
    off_next = kp - lb * a.block_size;
  };
  auto fetch = [&]() {
    const bool bad = id_next < 0 || id_next >= a.num_blocks;
    bad_block |= bad;
    const int id = bad ? 0 : id_next;
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      const int key = tid / LANES + x * (kThreads / LANES);
      const size_t at = ((size_t)__shfl(id, key, 64) * a.hkv + kvh) * a.block_size + __shfl(off_next, key, 64);
      in.load(x, a, at, tid % LANES);
    }
  };
  auto reaches = [&](int c) { return (c + 1) * KB > min(t.prefix, kend); };  // past the prefix, or the keys
  auto stage = [&](int c) {
    if (reaches(c)) {  // workgroup-uniform
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int key = tid / LANES + x * (kThreads / LANES);
        if (c * KB + key >= kend)
          in.zero(x);
        else if (in.clean(x))
          atomicOr(&s_special[c & 1], 1ull << key);
      }
    }
#pragma unroll
    for (int x = 0; x < PT; ++x) in.store(x, tid / LANES + x * (kThreads / LANES), tid % LANES, Ks, Vs);
  };

  if (tid < 2) s_special[tid] = 0;
  if (c_lo < c_hi) {  // workgroup-uniform
    lookup(c_lo);
    fetch();
    lookup(c_lo + 1);
    __syncthreads();
    stage(c_lo);
    __syncthreads();
  }
  for (int c = c_lo; c < c_hi; ++c) {
    const int k0 = c * KB;
    if (tid == 0) s_special[(c + 1) & 1] = 0;  // last read in chunk c - 1
    fetch();
    lookup(c + 2);
    __builtin_amdgcn_sched_barrier(0);

    // ---- S^T = K Q^T: KB keys x 16 rows ----
    v4f s[JT];
#pragma unroll
    for (int jt = 0; jt < JT; ++jt) s[jt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < DS; ++x)
#pragma unroll
      for (int jt = 0; jt < JT; ++jt) {
        bf16x8 kf[PLANES];
#pragma unroll
        for (int p = 0; p < PLANES; ++p) kf[p] = *reinterpret_cast<const bf16x8*>(&Ks[p][16 * jt + li][32 * x + 8 * lk]);
        s[jt] = product<PLANES>(kf, qf[x], s[jt]);
      }
    uint64_t seen = ~0ull;
    if (reaches(c)) {
      seen = fi::mask_window(mask, a.words, k0 - t.prefix);
      if (kend - k0 < 64) seen &= (1ull << (kend - k0)) - 1;
#pragma unroll
      for (int jt = 0; jt < JT; ++jt)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[jt][v] = (seen >> (16 * jt + 4 * lk + v)) & 1 ? s[jt][v] : -INFINITY;
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
    // no key seen yet: the point stays -inf, and scores of -inf weigh 0 against any finite one
    const float point = m_new == -INFINITY ? 0.0f : m_new;
    if (__builtin_amdgcn_ballot_w64(m_new != m_row) != 0) {  // after the first chunks, hardly ever
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
      const int vrow = 32 * u + 4 * lk + (li >> 2), vcol = 4 * (li & 3);  // as in prefill_bf16_kernel
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x8 vf[PLANES];
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
          const v4s lo = lds_read_tr16(&Vs[p][vrow][16 * dt + vcol]);
          const v4s hi = lds_read_tr16(&Vs[p][vrow + 16][16 * dt + vcol]);
          vf[p] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        o[dt] = product<PLANES>(vf, pp, o[dt]);
      }
    }
    // what is not finite in V, for the rows that see it
    for (uint64_t keys = s_special[c & 1]; keys != 0; keys &= keys - 1) {  // workgroup-uniform
      const int key = __builtin_ctzll(keys), lb = static_cast<int>(a.by_block.div(k0 + key));
      const int id = table[lb];
      if (id < 0 || id >= a.num_blocks || !((seen >> key) & 1)) continue;
      const size_t at = ((size_t)id * a.hkv + kvh) * a.block_size + (k0 + key - lb * a.block_size);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float x = P::value(a, at, 16 * dt + 4 * lk + v);
          if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[dt][v] += x;
        }
    }
    __syncthreads();  // every wave is done with this chunk's K and V
    if (c + 1 < c_hi) {  // workgroup-uniform
      stage(c + 1);
      __syncthreads();
    }
  }
  if (bad_block) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);

  float l_row = l_part + fi::lane_xor16(l_part, lane);
  l_row += fi::lane_xor32(l_row, lane);
  if (!live) return;
  if (nparts > 1) {
    const size_t at = (((size_t)seq * a.max_query_len + node) * a.hq + head) * a.parts + part;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(a.part_acc + at * D + 16 * dt + 4 * lk) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
    // a NaN sum takes a finite point, which the merge does not skip
    if (lk == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(l_row != l_row ? 0.f : m_row, l_row);
    return;
  }
  float inv = 1.0f / l_row;
  if (l_row == 0.0f && t.prefix <= 0) {  // a row that sees no key is zero
    uint64_t any = 0;
    for (int k0 = 0; k0 < kend; k0 += 64)
      any |= fi::mask_window(mask, a.words, k0 - t.prefix) & (kend - k0 < 64 ? (1ull << (kend - k0)) - 1 : ~0ull);
    if (any == 0) inv = 0.0f;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    *reinterpret_cast<float4*>(a.out + row * D + 16 * dt + 4 * lk) =
        make_float4(o[dt][0] * inv, o[dt][1] * inv, o[dt][2] * inv, o[dt][3] * inv);
}

// One output row quad a thread: the partials of its row joined in part order, four loaded at a time, each
// rescaled from its own reference point to the largest so far (a part without a key that the row sees
// carries -inf and adds nothing), divided by the combined sum.
template <int D, int KB>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(TreeArgs a, int64_t quads) {
  constexpr int N = 4;
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (idx >= quads) return;
  const int64_t prow = idx / (D / 4);  // (sequence, node, head)
  const int dq = static_cast<int>(idx % (D / 4));
  const int64_t at_node = prow / a.hq;
  const int head = static_cast<int>(prow - at_node * a.hq);
  const int seq = static_cast<int>(at_node / a.max_query_len), node = static_cast<int>(at_node - (int64_t)seq * a.max_query_len);
  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, seq);
  if (node >= t.nodes) return;
  const int kend = key_end(a, t), nparts = key_parts<KB>(a, kend);
  if (nparts <= 1) return;  // written by the launch before
  const float* acc_at = a.part_acc + prow * a.parts * D + 4 * dq;
  const float* ml_at = a.part_ml + prow * a.parts * 2;
  float mx = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < nparts; s0 += N) {
    float2 ml[N];
    float4 o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = min(s0 + i, nparts - 1);
      ml[i] = *reinterpret_cast<const float2*>(ml_at + 2 * s);
      o[i] = *reinterpret_cast<const float4*>(acc_at + (size_t)s * D);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (s0 + i >= nparts || ml[i].x == -INFINITY) continue;
      const float to = fmaxf(mx, ml[i].x);
      const float old = __builtin_amdgcn_exp2f(mx - to), now = __builtin_amdgcn_exp2f(ml[i].x - to);
      mx = to;
      l = l * old + now * ml[i].y;
      acc = make_float4(acc.x * old + now * o[i].x, acc.y * old + now * o[i].y, acc.z * old + now * o[i].z,
                        acc.w * old + now * o[i].w);
    }
  }
  // several parts and prefix <= 0: a tree longer than a part, of whose keys the row may see none
  float inv = 1.0f / l;
  if (l == 0.0f && t.prefix <= 0) {
    const uint64_t* mask = a.mask + (size_t)(t.first + node) * a.words;
    uint64_t any = 0;
    for (int k0 = 0; k0 < kend; k0 += 64)
      any |= fi::mask_window(mask, a.words, k0 - t.prefix) & (kend - k0 < 64 ? (1ull << (kend - k0)) - 1 : ~0ull);
    if (any == 0) inv = 0.0f;
  }
  *reinterpret_cast<float4*>(a.out + ((size_t)(t.first + node) * a.hq + head) * D + 4 * dq) =
      make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <int D, int POOL>
int32_t launch_tree(fi_context* ctx, TreeArgs& a) {
  constexpr int KB = Pool<POOL, D>::KB;
  const int64_t cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int64_t rows = static_cast<int64_t>(a.max_query_len) * a.group;
  FI_REQUIRE(rows < (1 << 30), FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: too many rows");
  a.ntiles = static_cast<int>((rows + kRows - 1) / kRows);
  const int64_t tiles = static_cast<int64_t>(a.num_seqs) * a.hkv * a.ntiles;
  const int64_t chunks = std::max<int64_t>(1, (static_cast<int64_t>(a.max_context_len) + KB - 1) / KB);
  const int64_t wanted = std::max<int64_t>(1, 4 * cus / tiles);
  a.part_chunks = static_cast<int>(std::max<int64_t>(256 / KB, (chunks + wanted - 1) / wanted));
  a.parts = static_cast<int>((chunks + a.part_chunks - 1) / a.part_chunks);
  const int64_t units = static_cast<int64_t>(a.parts) * a.num_seqs * a.hkv;
  const int64_t grid = (units + 7) / 8 * 8 * a.ntiles;
  FI_REQUIRE(grid <= 0x7fffffff, FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: grid too large");
  const int64_t prows = static_cast<int64_t>(a.num_seqs) * a.max_query_len * a.hq;
  if (a.parts > 1) {
    const size_t acc = static_cast<size_t>(prows) * a.parts * D * sizeof(float);
    FI_TRY(fi::ensure_workspace(ctx, acc + static_cast<size_t>(prows) * a.parts * 2 * sizeof(float)));
    a.part_acc = static_cast<float*>(ctx->workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ctx->workspace) + acc);
  }
  hipLaunchKernelGGL((attn_tree_kernel<D, POOL>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, ctx->stream, a);
  FI_CHECK_LAUNCH("attn_tree_kernel");
  if (a.parts > 1) {
    const int64_t quads = prows * (D / 4);
    FI_REQUIRE(quads / kThreads < 0x7fffffff, FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: too many rows");
    hipLaunchKernelGGL((tree_merge_kernel<D, KB>), dim3(static_cast<unsigned>((quads + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, ctx->stream, a, quads);
    FI_CHECK_LAUNCH("tree_merge_kernel");
  }
  return FI_OK;
}

template <int POOL>
int32_t launch_tree_dim(fi_context* ctx, TreeArgs& a, int32_t head_dim) {
  switch (head_dim) {
    case 32:
      return launch_tree<32, POOL>(ctx, a);
    case 64:
      return launch_tree<64, POOL>(ctx, a);
    default:
      return launch_tree<128, POOL>(ctx, a);
  }
}

}  // namespace

extern "C" {

int32_t fi_attn_tree_paged(fi_context* ctx, const float* d_q, const void* d_k_cache, const void* d_v_cache, int32_t kv_dtype,
                           const int32_t* d_block_tables, int32_t max_blocks_per_seq, const int32_t* d_cu_seqlens,
                           const int32_t* d_context_lens, const uint64_t* d_tree_mask, int32_t mask_words, int32_t num_seqs,
                           int32_t max_query_len, int32_t max_context_len, int32_t num_q_heads, int32_t num_kv_heads,
                           int32_t head_dim, int32_t block_size, int32_t num_blocks, float scale, float* d_out) {
  FI_TRY(fi::enter(ctx));
  FI_REQUIRE(num_seqs >= 0 && max_query_len >= 0 && max_context_len >= 0 && mask_words >= 0, FI_ERR_INVALID_SHAPE,
             "fi_attn_tree_paged: negative sizes");
  FI_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, FI_ERR_INVALID_SHAPE,
             "number of query heads must be divisible by number of KV heads");
  FI_REQUIRE(block_size > 0 && num_blocks > 0 && max_blocks_per_seq > 0, FI_ERR_INVALID_CONFIG,
             "fi_attn_tree_paged: pool dimensions must be greater than zero");
  FI_REQUIRE(kv_dtype == FI_DTYPE_F32 || kv_dtype == FI_DTYPE_BF16 || kv_dtype == FI_DTYPE_MXFP4, FI_ERR_INVALID_TYPE,
             "fi_attn_tree_paged: KV dtype must be f32, bf16 or mxfp4");
  FI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, FI_ERR_UNSUPPORTED,
             "fi_attn_tree_paged: head_dim must be 32, 64 or 128");
  FI_REQUIRE(static_cast<int64_t>(max_context_len) <= static_cast<int64_t>(max_blocks_per_seq) * block_size,
             FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: max_context_len exceeds the block-table width");
  FI_REQUIRE(max_context_len <= (1 << 30), FI_ERR_UNSUPPORTED, "fi_attn_tree_paged: contexts of more than 2^30 tokens");
  FI_REQUIRE(max_query_len <= fi::kMaxTreeNodes, FI_ERR_UNSUPPORTED,
             "fi_attn_tree_paged: trees of more than " + std::to_string(fi::kMaxTreeNodes) + " nodes");
  FI_REQUIRE(mask_words <= (1 << 20) && max_query_len <= 64 * mask_words, FI_ERR_INVALID_SHAPE,
             "fi_attn_tree_paged: mask_words must hold a bit for each of max_query_len nodes");
  FI_REQUIRE(scale > 0.0f && scale < INFINITY, FI_ERR_INVALID_CONFIG,
             "fi_attn_tree_paged: scale must be positive and finite");
  if (num_seqs == 0 || max_query_len == 0) return FI_OK;
  FI_REQUIRE(d_q && d_k_cache && d_v_cache && d_block_tables && d_cu_seqlens && d_context_lens && d_tree_mask && d_out,
             FI_ERR_INVALID_CONFIG, "fi_attn_tree_paged: null pointer");
  FI_REQUIRE(((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out) | reinterpret_cast<uintptr_t>(d_k_cache) |
               reinterpret_cast<uintptr_t>(d_v_cache)) & 15) == 0,
             FI_ERR_INVALID_LAYOUT, "fi_attn_tree_paged: q, out and the K/V pools must be 16-byte aligned (vector accesses)");
  TreeArgs a{};
  a.q = d_q;
  a.k_cache = d_k_cache;
  a.v_cache = d_v_cache;
  a.block_tables = d_block_tables;
  a.cu_seqlens = d_cu_seqlens;
  a.context_lens = d_context_lens;
  a.mask = d_tree_mask;
  a.out = d_out;
  a.faults = ctx->d_faults;
  a.words = mask_words;
  a.max_blocks = max_blocks_per_seq;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.num_seqs = num_seqs;
  a.max_query_len = max_query_len;
  a.max_context_len = max_context_len;
  a.scale = scale;
  a.by_block = fi::FastDiv(static_cast<uint32_t>(block_size));
  a.by_group = fi::FastDiv(static_cast<uint32_t>(a.group));
  if (kv_dtype == FI_DTYPE_F32) return launch_tree_dim<FI_DTYPE_F32>(ctx, a, head_dim);
  if (kv_dtype == FI_DTYPE_BF16) return launch_tree_dim<FI_DTYPE_BF16>(ctx, a, head_dim);
  return launch_tree_dim<FI_DTYPE_MXFP4>(ctx, a, head_dim);
}

}  // extern "C"
