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

// Whether a row sees no key at all: then it is zero, where a row whose scores are all -inf is NaN.
__device__ __forceinline__ bool sees_nothing(const TreeArgs& a, const fi::TreeSpan& t, int kend, const uint64_t* mask) {
  if (t.prefix > 0) return false;
  for (int k0 = 0; k0 < kend; k0 += 64)
    if (fi::mask_window(mask, a.words, k0 - t.prefix) & (kend - k0 < 64 ? (1ull << (kend - k0)) - 1 : ~0ull)) return false;
  return true;
}

// What of two bf16 elements is not finite, cleared.
struct Bf16 {
  static __device__ __forceinline__ bool clear(uint32_t& w) {
    const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
    w = (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
    return lo || hi;
  }
};
template <int D>
struct Bf16Pool {
  static __device__ __forceinline__ float4 values(const TreeArgs& a, size_t row, int d) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.v_cache) + row * D + d);
    return fi::bf16x4_to_f32(w.x, w.y);
  }
};

// ---- a chunk's way from the pool to LDS: f32 and 4-bit pools ----
// A thread holds PT pieces of K and of V in registers, piece r of key tid / LANES + r * (256 / LANES); LANES
// neighbouring lanes read a whole row.
template <int POOL, int D>
struct Pool;

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
  static __device__ __forceinline__ float4 values(const TreeArgs& a, size_t row, int d) {
    return *reinterpret_cast<const float4*>(static_cast<const float*>(a.v_cache) + row * D + d);
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
  static __device__ __forceinline__ float4 values(const TreeArgs& a, size_t row, int d) {
    const uint32_t s = static_cast<const uint8_t*>(a.v_cache)[code_bytes(a) + row * GROUPS + d / fi::kFp4Group];
    const float x = s > fi::kFp4MaxScale ? NAN : 0.0f;
    return make_float4(x, x, x, x);
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

// What a workgroup does: 64 rows of one (part, sequence, kv head), its chunks [c_lo, c_hi).
struct Unit {
  int seq, kvh, part, tile;
  fi::TreeSpan t;
  int nodes, kend, nparts, c_lo, c_hi;
};

// False: nothing (the whole workgroup).  The tiles of a (part, sequence, kv head) run one after the other on one XCD
// (workgroup L runs on XCD L % 8), whose L2 then holds the keys that they share.
template <int KB>
__device__ __forceinline__ bool find_unit(const TreeArgs& a, Unit& u) {
  const int slot = blockIdx.x >> 3;
  const int unit = slot / a.ntiles * 8 + (blockIdx.x & 7);
  u.tile = slot % a.ntiles;
  if (unit >= a.parts * a.num_seqs * a.hkv) return false;
  u.kvh = unit % a.hkv;
  u.seq = unit / a.hkv % a.num_seqs;
  u.part = unit / a.hkv / a.num_seqs;
  u.t = fi::tree_span(a.cu_seqlens, a.context_lens, u.seq);
  u.nodes = min(u.t.nodes, a.max_query_len);
  if (u.part == 0 && u.tile == 0 && u.kvh == 0 && threadIdx.x == 0) {
    if (u.t.nodes > a.max_query_len) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
    if (u.t.prefix + u.t.nodes > a.max_context_len) atomicOr(a.faults, FI_FAULT_CONTEXT_RANGE);
  }
  if (u.tile * kRows >= u.nodes * a.group) return false;
  u.kend = key_end(a, u.t);
  u.nparts = key_parts<KB>(a, u.kend);
  if (u.part >= u.nparts) return false;
  u.c_lo = u.part * a.part_chunks;
  u.c_hi = min(u.c_lo + a.part_chunks, (u.kend + KB - 1) / KB);
  return true;
}

// Whether a chunk reaches past the prefix, or past the keys.
template <int KB>
__device__ __forceinline__ bool reaches(const Unit& u, int c) {
  return (c + 1) * KB > min(u.t.prefix, u.kend);
}

// A lane's row: row li of its wave's sixteen, shared by four lanes (lk).
template <int D>
struct Row {
  static constexpr int DS = D / 32;  // 32-wide d steps of Q K^T
  static constexpr int DT = D / 16;  // 16-wide output d tiles of P V
  int lane, li, lk;
  bf16x8 qf[DS][3];  // Q pieces: B operand row li, d = 32 s + 8 lk .. + 7
  v4f o[DT];         // O^T tile dt: d = 16 dt + 4 lk + v, row li
  float m, l;        // the exponents' reference point (log2 units), this lane's share of the weights' sum
  float c2;          // scores -> log2 units

  // The row's place, found again where it is needed (registers are at the limit): its node and head, its index
  // among the step's rows [T, Hq].  Rows behind the tree's last take node 0's.
  struct Place {
    int node, head;
    bool live;
    size_t row, index;
  };
  __device__ __forceinline__ Place place(const TreeArgs& a, const Unit& u) const {
    Place p;
    const int r = u.tile * kRows + 16 * (threadIdx.x >> 6) + li;
    p.node = static_cast<int>(a.by_group.div(r));
    p.head = u.kvh * a.group + (r - p.node * a.group);
    p.live = p.node < u.nodes;
    p.row = u.t.first + (p.live ? p.node : 0);
    p.index = p.row * a.hq + p.head;
    return p;
  }
  __device__ __forceinline__ void init(const TreeArgs& a, const Unit& u) {
    lane = threadIdx.x & 63;
    li = lane & 15;
    lk = lane >> 4;
    const Place at = place(a, u);
    const float* q = a.q + at.index * D + 8 * lk;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const float4 lo = *reinterpret_cast<const float4*>(q + 32 * s), hi = *reinterpret_cast<const float4*>(q + 32 * s + 4);
      const f32x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      split3(at.live ? v : z, qf[s]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.0f;
    c2 = a.scale * 1.4426950408889634f;
  }

  // Which of the keys k0 .. k0 + 63 the row sees, and -inf for the scores of the others: s[jt][v] is that of key
  // 16 jt + 4 lk + v.
  template <int JT>
  __device__ __forceinline__ uint64_t hide(const TreeArgs& a, const Unit& u, int k0, v4f (&s)[JT]) const {
    uint64_t seen = fi::mask_window(a.mask + place(a, u).row * a.words, a.words, k0 - u.t.prefix);
    if (u.kend - k0 < 64) seen &= (1ull << (u.kend - k0)) - 1;
    const uint64_t mine = seen >> (4 * lk);
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) s[jt][v] = (mine >> (16 * jt + v)) & 1 ? s[jt][v] : -INFINITY;
    return seen;
  }

  // The scores' weights in their place, by a reference point that moves when a chunk's maximum passes it by 2^8.
  template <int JT>
  __device__ __forceinline__ void weigh(v4f (&s)[JT]) {
    float mx = -INFINITY;
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[jt][v]);
    mx = fmaxf(mx, fi::lane_xor16(mx, lane));
    mx = fmaxf(mx, fi::lane_xor32(mx, lane));
    const float m_chunk = mx * c2;
    const float m_new = m_chunk > m + 8.0f ? m_chunk : m;
    // no key seen yet: the point stays -inf, and scores of -inf weigh 0 against any finite one
    const float point = m_new == -INFINITY ? 0.0f : m_new;
    if (__builtin_amdgcn_ballot_w64(m_new != m) != 0) {  // after the first chunks, hardly ever
      const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
    m = m_new;
    float sum = 0.0f;
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        s[jt][v] = __builtin_amdgcn_exp2f(fmaf(s[jt][v], c2, -point));
        sum += s[jt][v];
      }
    l += sum;
  }

  // The weights of 32 keys as B operand pieces (k index 8 lk + e: key 4 lk + e, e < 4, or 16 + 4 lk + e - 4).
  static __device__ __forceinline__ void pieces(const v4f& lo, const v4f& hi, bf16x8 (&pp)[3]) {
    const f32x8 pf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    split3(pf, pp);
  }

  // What is not finite in V, for the rows that see it: `keys` of the chunk at k0.
  template <typename P>
  __device__ __forceinline__ void add_special(const TreeArgs& a, const Unit& u, int k0, uint64_t keys, uint64_t seen) {
    for (; keys != 0; keys &= keys - 1) {  // workgroup-uniform
      const int key = __builtin_ctzll(keys), lb = static_cast<int>(a.by_block.div(k0 + key));
      const int id = a.block_tables[(size_t)u.seq * a.max_blocks + lb];
      if (id < 0 || id >= a.num_blocks || !((seen >> key) & 1)) continue;
      const size_t at = ((size_t)id * a.hkv + u.kvh) * a.block_size + (k0 + key - lb * a.block_size);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const float4 x = P::values(a, at, 16 * dt + 4 * lk);
        const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if ((__float_as_uint(e[v]) & 0x7f800000u) == 0x7f800000u) o[dt][v] += e[v];
        __builtin_amdgcn_sched_barrier(0);  // one quad's registers at a time: this is hardly ever run
      }
    }
  }

  __device__ __forceinline__ void finish(const TreeArgs& a, const Unit& u) {
    float sum = l + fi::lane_xor16(l, lane);
    sum += fi::lane_xor32(sum, lane);
    const Place p = place(a, u);
    if (!p.live) return;
    if (u.nparts > 1) {
      const size_t at = (((size_t)u.seq * a.max_query_len + p.node) * a.hq + p.head) * a.parts + u.part;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4*>(a.part_acc + at * D + 16 * dt + 4 * lk) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
      // a NaN sum takes a finite point, which the merge does not skip
      if (lk == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(sum != sum ? 0.f : m, sum);
      return;
    }
    const float inv = sum == 0.0f && sees_nothing(a, u.t, u.kend, a.mask + p.row * a.words) ? 0.0f : 1.0f / sum;
    float* out = a.out + p.index * D + 4 * lk;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(out + 16 * dt) = make_float4(o[dt][0] * inv, o[dt][1] * inv, o[dt][2] * inv, o[dt][3] * inv);
  }
};

// ---- bf16 pools ----

// One load of a wave from the pool to LDS: lane i's 16 bytes to lds + 16 i.  In assembly, because the
// compiler would wait for every such load before the next read of the same LDS array; what waits for them is
// wait_loads and a barrier.
__device__ __forceinline__ void load_to_lds(const uint8_t* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "m0", "memory");
}
// Until at most N of this wave's loads are on their way (they end in the order of their issue).
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 16, "four bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A chunk's K and V rows go from the pool to LDS as they are, so that none of them pass through registers.
// Three slots of a chunk's K or V each, taken in turn: while one is multiplied the next two are on their way,
// 32 KB at D = 128, 96 KB a CU, about what the memory's latency asks for.  One barrier a product: the
// slot's loads have landed, and every wave is done with the slot that is loaded next.  The LDS rows are not
// padded (a wave's load fills 1 KB in lane order); instead piece p (16 bytes) of a row lies at p ^ turn(key), so that
// the rows of a fragment meet all banks evenly.
template <int D>
__global__ __launch_bounds__(kThreads, 3) void attn_tree_bf16_kernel(TreeArgs a) {
  constexpr int KB = 64, JT = KB / 16, KS = KB / 32;
  constexpr int DS = Row<D>::DS, DT = Row<D>::DT;
  constexpr int JB = 2;                // score tiles whose K fragments are held at once, twice
  constexpr int DB = DT < 4 ? DT : 2;  // d tiles whose V fragments are
  constexpr int PIECES = D / 8;        // 16-byte pieces of a row
  constexpr int PT = KB * PIECES / kThreads;  // a thread's loads of K (and of V)
  auto turn = [](int key) { return D == 128 ? 2 * (key & 7) : (D == 64 ? key & 7 : 2 * ((key >> 2) & 1)); };
  __shared__ __align__(1024) uint16_t slots[3][KB * D];
  __shared__ unsigned long long s_special;

  Unit u;
  if (!find_unit<KB>(a, u)) return;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  Row<D> row;
  row.init(a, u);
  const int lane = row.lane, li = row.li, lk = row.lk;

  // Thread tid loads piece tid % PIECES (as it lies in LDS) of keys key_of(0), key_of(1), ..: 64 / PIECES
  // neighbouring keys a wave's load.
  auto key_of = [&](int x) { return (PT * w + x) * (64 / PIECES) + lane / PIECES; };
  const int* table = a.block_tables + (size_t)u.seq * a.max_blocks;
  int first_block = 0, ids = 0;  // lane: the id of block first_block + lane
  int held = 0;                  // blocks behind first_block that ids holds
  bool bad_block = false;
  uint32_t at_row = 0;  // lane: the pool row of a chunk's key
  auto find_rows = [&](int c) {  // of a chunk's keys (the last key again past the end)
    const int last = static_cast<int>(a.by_block.div(min(c * KB + KB, u.kend) - 1));
    if (last >= first_block + held) {  // workgroup-uniform; 1024 keys apart with blocks of 16
      first_block = static_cast<int>(a.by_block.div(c * KB));
      held = 64;
      ids = table[min(first_block + lane, static_cast<int>(a.by_block.div(u.kend - 1)))];
      __builtin_amdgcn_s_waitcnt(0);  // here, not where ids is used: V's loads go on in the other chunks
    }
    const int kp = min(c * KB + lane, u.kend - 1), lb = static_cast<int>(a.by_block.div(kp));
    const int id = __shfl(ids, lb - first_block, 64);
    const bool bad = id < 0 || id >= a.num_blocks;
    bad_block |= bad;
    at_row = (static_cast<uint32_t>(bad ? 0 : id) * a.hkv + u.kvh) * a.block_size + (kp - lb * a.block_size);
  };
  typedef __attribute__((address_space(3))) uint16_t* lds_ptr;
  typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
  auto load = [&](const void* pool, int slot) {
    const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)&slots[0][0])) + slot * (2 * KB * D) + PT * w * 1024;
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      const size_t from = (size_t)__shfl(at_row, key_of(x), 64) * (2 * D) + 16 * ((lane % PIECES) ^ turn(key_of(x)));
      load_to_lds(static_cast<const uint8_t*>(pool) + from, to + 1024 * x);
    }
  };

  if (tid == 0) s_special = 0;
  if (u.c_lo < u.c_hi) {  // workgroup-uniform
    find_rows(u.c_lo);
    load(a.k_cache, 0);
    load(a.v_cache, 1);
  }
  int k_slot = 0, v_slot = 1;  // of the chunk; the next one's are two further
  for (int c = u.c_lo; c < u.c_hi; ++c) {
    const int k0 = c * KB;
    const bool more = c + 1 < u.c_hi;
    const int k_next = k_slot == 0 ? 2 : k_slot - 1, v_next = v_slot == 0 ? 2 : v_slot - 1;
    wait_loads<PT>();  // K; V is on its way
    __syncthreads();
    if (more) {
      find_rows(c + 1);
      load(a.k_cache, k_next);
    }

    // ---- S^T = K Q^T: KB keys x 16 rows ----
    uint32_t k_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)&slots[0][0])) + k_slot * (2 * KB * D) + 2 * D * li +
                    16 * (lk ^ turn(li));
    v4f s[JT];
#pragma unroll
    for (int jt = 0; jt < JT; ++jt) s[jt] = v4f{0.f, 0.f, 0.f, 0.f};
    bf16x8 kf[2][JB];  // fragments a step ahead of their products
    auto read_k = [&](int g) {  // score tiles g % (JT / JB) * JB .. at d step g / (JT / JB)
#pragma unroll
      for (int i = 0; i < JB; ++i)
        kf[g & 1][i] = *(const lds_bf16x8*)((k_at ^ (g / (JT / JB) * 64)) + 32 * D * (g % (JT / JB) * JB + i));
    };
    read_k(0);
#pragma unroll
    for (int g = 0; g < DS * JT / JB; ++g) {
      if (g + 1 < DS * JT / JB) read_k(g + 1);
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < JB; ++i) {
          v4f& t = s[g % (JT / JB) * JB + i];
          t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[g & 1][i], row.qf[g / (JT / JB)][p], t, 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool past = reaches<KB>(u, c);  // workgroup-uniform
    uint64_t seen = ~0ull;
    if (past) seen = row.hide(a, u, k0, s);
    row.weigh(s);

    if (more)
      wait_loads<PT>();  // V; the next K is on its way
    else
      wait_loads<0>();
    __syncthreads();
    uint16_t* vs = slots[v_slot];
    if (past) {  // what is not finite in V is noted and cleared
#pragma unroll 1
      for (int x = 0; x < PT; ++x) {
        uint4* at = reinterpret_cast<uint4*>(&vs[(PT * w + x) * 512 + 8 * lane]);
        uint4 v = *at;
        bool any = Bf16::clear(v.x);
        any |= Bf16::clear(v.y);
        any |= Bf16::clear(v.z);
        any |= Bf16::clear(v.w);
        if (any) {
          *at = v;
          atomicOr(&s_special, 1ull << key_of(x));
        }
      }
      __syncthreads();
    }
    if (more) load(a.v_cache, v_next);

    // ---- O^T += V^T P^T ----
    constexpr int GROUPS = KS * DT / DB;
    bf16x8 vf[2][DB];
    // transposing reads as in prefill_bf16_kernel
    const uint32_t v_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)vs)) + 2 * D * (4 * lk + (li >> 2)) +
                          16 * (((li >> 1) & 1) ^ turn(4 * lk + (li >> 2))) + 8 * (li & 1);
    auto read_v = [&](int g) {  // d tiles g % (DT / DB) * DB .. of 32-key step g / (DT / DB)
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        const uint32_t at = (v_at ^ (32 * (g % (DT / DB) * DB + i))) + 64 * D * (g / (DT / DB));
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 32 * D));
        vf[g & 1][i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    read_v(0);
    bf16x8 pp[3];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g % (DT / DB) == 0) row.pieces(s[2 * (g / (DT / DB))], s[2 * (g / (DT / DB)) + 1], pp);
      if (g + 1 < GROUPS) read_v(g + 1);
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          v4f& o = row.o[g % (DT / DB) * DB + i];
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[g & 1][i], pp[p], o, 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (past) {
      row.template add_special<Bf16Pool<D>>(a, u, k0, s_special, seen);
      __syncthreads();
      if (tid == 0) s_special = 0;  // a barrier before the next chunk's V is looked at
    }
    k_slot = k_next;
    v_slot = v_next;
  }
  if (bad_block) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
  row.finish(a, u);
}

// ---- f32 and 4-bit pools: through registers, which convert them ----
template <int D, int POOL>
__global__ __launch_bounds__(kThreads, D == 128 && POOL == FI_DTYPE_F32 ? 2 : 3) void attn_tree_kernel(TreeArgs a) {
  using P = Pool<POOL, D>;
  constexpr int KB = P::KB, PLANES = P::PLANES, PT = P::PT, LANES = P::LANES;
  constexpr int JT = KB / 16, KS = KB / 32, DS = Row<D>::DS, DT = Row<D>::DT;
  constexpr int KPK = D == 128 && PLANES == 1 ? D + 16 : D + 8;  // padded LDS rows of K (see prefill_bf16_kernel)
  constexpr int KPV = D + 8;                                     // of V (transposing reads)
  __shared__ __align__(16) uint16_t Ks[PLANES][KB][KPK];
  __shared__ __align__(16) uint16_t Vs[PLANES][KB][KPV];
  __shared__ unsigned long long s_special[2];  // by the chunk's parity: keys whose V is not finite throughout

  Unit u;
  if (!find_unit<KB>(a, u)) return;
  const int tid = threadIdx.x;
  Row<D> row;
  row.init(a, u);
  const int lane = row.lane, li = row.li, lk = row.lk;

  // Staging: a wave's lanes look up the blocks of a chunk's keys, a chunk ahead of its loads; a thread takes
  // its keys' from them.  Loads are unconditional (clamped keys; the last chunk re-reads itself).
  P in;
  int id_next = 0, off_next = 0;
  bool bad_block = false;
  const int* table = a.block_tables + (size_t)u.seq * a.max_blocks;
  auto lookup = [&](int c) {
    const int kp = min(min(c, u.c_hi - 1) * KB + lane % KB, u.kend - 1);
    const int lb = static_cast<int>(a.by_block.div(kp));
    id_next = table[lb];
    off_next = kp - lb * a.block_size;
  };
  auto fetch = [&]() {
    const bool bad = id_next < 0 || id_next >= a.num_blocks;
    bad_block |= bad;
    const uint32_t at = (static_cast<uint32_t>(bad ? 0 : id_next) * a.hkv + u.kvh) * a.block_size + off_next;
#pragma unroll
    for (int x = 0; x < PT; ++x) in.load(x, a, __shfl(at, tid / LANES % 64 + x * (kThreads / LANES), 64), tid % LANES);
  };
  auto stage = [&](int c) {
    if (reaches<KB>(u, c)) {  // workgroup-uniform
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int key = tid / LANES + x * (kThreads / LANES);
        if (c * KB + key >= u.kend)
          in.zero(x);
        else if (in.clean(x))
          atomicOr(&s_special[c & 1], 1ull << key);
      }
    }
#pragma unroll
    for (int x = 0; x < PT; ++x) in.store(x, tid / LANES + x * (kThreads / LANES), tid % LANES, Ks, Vs);
  };

  if (tid < 2) s_special[tid] = 0;
  if (u.c_lo < u.c_hi) {  // workgroup-uniform
    lookup(u.c_lo);
    fetch();
    lookup(u.c_lo + 1);
    __syncthreads();
    stage(u.c_lo);
    __syncthreads();
  }
  for (int c = u.c_lo; c < u.c_hi; ++c) {
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
        s[jt] = product<PLANES>(kf, row.qf[x], s[jt]);
      }
    const bool past = reaches<KB>(u, c);
    uint64_t seen = ~0ull;
    if (past) seen = row.hide(a, u, k0, s);
    row.weigh(s);

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      bf16x8 pp[3];
      row.pieces(s[2 * t], s[2 * t + 1], pp);
      const int vrow = 32 * t + 4 * lk + (li >> 2), vcol = 4 * (li & 3);  // as in prefill_bf16_kernel
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x8 vf[PLANES];
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
          const v4s lo = lds_read_tr16(&Vs[p][vrow][16 * dt + vcol]);
          const v4s hi = lds_read_tr16(&Vs[p][vrow + 16][16 * dt + vcol]);
          vf[p] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        row.o[dt] = product<PLANES>(vf, pp, row.o[dt]);
      }
    }
    if (past) row.template add_special<P>(a, u, k0, s_special[c & 1], seen);
    __syncthreads();  // every wave is done with this chunk's K and V
    if (c + 1 < u.c_hi) {  // workgroup-uniform
      stage(c + 1);
      __syncthreads();
    }
  }
  if (bad_block) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
  row.finish(a, u);
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
  // (several parts and no prefix: a tree longer than a part)
  const float inv = l == 0.0f && sees_nothing(a, t, kend, a.mask + (size_t)(t.first + node) * a.words) ? 0.0f : 1.0f / l;
  *reinterpret_cast<float4*>(a.out + ((size_t)(t.first + node) * a.hq + head) * D + 4 * dq) =
      make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <int D, int POOL>
int32_t launch_tree(fi_context* ctx, TreeArgs& a) {
  constexpr int KB = POOL == FI_DTYPE_F32 ? 32 : 64;  // keys of a chunk
  const int64_t cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int64_t rows = static_cast<int64_t>(a.max_query_len) * a.group;
  FI_REQUIRE(rows < (1 << 30), FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: too many rows");
  a.ntiles = static_cast<int>((rows + kRows - 1) / kRows);
  const int64_t tiles = static_cast<int64_t>(a.num_seqs) * a.hkv * a.ntiles;
  const int64_t chunks = std::max<int64_t>(1, (static_cast<int64_t>(a.max_context_len) + KB - 1) / KB);
  const int64_t wanted = std::max<int64_t>(1, 8 * cus / tiles);
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
  if constexpr (POOL == FI_DTYPE_BF16)
    hipLaunchKernelGGL((attn_tree_bf16_kernel<D>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, ctx->stream, a);
  else
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
  // the kernels keep pool rows in 32 bits (2^32 of them are 64 GiB of an array at 4 bits and head_dim 32)
  FI_REQUIRE(static_cast<int64_t>(num_blocks) * block_size <= (int64_t{1} << 32) / num_kv_heads, FI_ERR_UNSUPPORTED,
             "fi_attn_tree_paged: pools are served up to 2^32 rows of one head");
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
