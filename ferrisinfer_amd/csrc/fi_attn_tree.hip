// Attention of a tree's rows over the paged pool, in f32 accuracy on v_mfma_f32_16x16x32_bf16.  Node i of
// sequence b attends the cached prefix and the nodes whose bits its mask row has set, read in the pool
// behind the prefix.  No counterpart in the reference, whose sessions feed one sampled token a step
// (crates/ferrisinfer-runtime/src/session.rs:246-262).
//
// Rows are packed: row r of a (sequence, kv head) is head r % G of node r / G, so that any group size fills
// 64-row tiles (four waves of 16 rows).  One workgroup a (sequence, kv head, tile), or, where those leave CUs
// idle, a part of its keys: the lengths are on the device, so each workgroup works out the cut from them
// (find_unit), and a tile's unnormalised partials are joined by its last workgroup, or by a launch of their own
// (tree_join_rows_kernel, tree_join_kernel).  The products are the prefill kernels': S^T = K Q^T leaves a lane the scores of
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
  // what a cut launch joins: each workgroup's unnormalised rows [pieces, 64, D], their reference points and
  // sums [pieces, 64, 2], and each sequence's pieces (its first, its parts) for a join in a launch of its own
  float* part_acc;
  float* part_ml;
  int2* plan;          // null: the last workgroup of a tile joins its parts
  unsigned* counters;  // of them, one a tile: those that are done, zero between launches
  uint32_t* faults;
  int words, max_blocks, hq, hkv, group, block_size, num_blocks;
  int num_seqs, max_query_len, max_context_len;
  int ntiles;      // tiles of a tree of max_query_len nodes
  int slots;       // pieces of a cut launch, at most; 0: none is cut
  int cus, least;  // the least chunks of a part
  float scale;
  fi::FastDiv by_block, by_group;
};

// The keys of a sequence that the launch reads: lengths past max_context_len are cut off there.
__device__ __forceinline__ int key_end(const TreeArgs& a, const fi::TreeSpan& t) {
  return min(t.prefix + t.nodes, a.max_context_len);
}
// Whether a row sees no key at all: then it is zero, where a row whose scores are all -inf is NaN.
__device__ __forceinline__ bool sees_nothing(const TreeArgs& a, const fi::TreeSpan& t, int kend, const uint64_t* mask) {
  if (t.prefix > 0 && kend > 0) return false;
  for (int k0 = 0; k0 < kend; k0 += 64)
    if (fi::mask_window(mask, a.words, k0 - t.prefix) & fi::keys_before(kend, k0)) return false;
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

// What a workgroup does: 64 rows of one (sequence, kv head), chunks [c_lo, c_hi) of its keys.
struct Unit {
  int seq, kvh, part, tile, nparts;
  int piece;   // among the launch's
  int tiles;   // of the sequence
  fi::TreeSpan t;
  int nodes, kend, c_lo, c_hi;
};

constexpr int kRowJoins = 128;      // tiles up to which the join is a workgroup a row
constexpr int kPlanned = kThreads;  // sequences of a planned launch, at most: a thread each

struct PlanShared {
  uint32_t key[kPlanned];  // chunks, then the place in the batch: the order of the sequences
  int count[kPlanned];     // pieces a kv head
  int sums[2][kThreads / 64][3];
  int found[4];  // sequence, its first piece, parts, tiles
};

// Lane 63's combination of a wave's values (none below 0), in a scalar register.
template <typename F>
__device__ __forceinline__ int wave_combine(int v, F f) {
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));  // row_shr:1, 2, 4, 8
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast:15, 31
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int add_int(int x, int y) { return x + y; }
__device__ __forceinline__ int max_int(int x, int y) { return max(x, y); }

// The launch's pieces, which every workgroup lays out for itself from the lengths, a thread a sequence.  Tiles that
// fill the device are not cut: they are taken as they are, those of long sequences first, folded where they all
// run at once, so that a CU gets a long one and a short one.  Otherwise, where the longest sequence's tile has more
// chunks than a CU's share of them all, sequences are cut into parts of as few chunks as make no more pieces
// than run at a time.
// False: this workgroup has none.
template <int KB>
__device__ __forceinline__ bool find_unit(const TreeArgs& a, Unit& u) {
  int at = blockIdx.x;  // the piece
  u.piece = at;
  u.part = 0;
  u.nparts = 1;
  int cut = 0x7fffffff;  // chunks of a part
  auto chunks_of = [&](const fi::TreeSpan& t) { return max((key_end(a, t) + KB - 1) / KB, 1); };
  auto tiles_of = [&](const fi::TreeSpan& t) { return (min(t.nodes, a.max_query_len) * a.group + kRows - 1) / kRows; };
  if (a.num_seqs == 1 || a.num_seqs > kPlanned) {
    u.kvh = at % a.hkv;
    at /= a.hkv;
    if (a.num_seqs == 1) {
      u.seq = 0;
      const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, 0);
      const int chunks = chunks_of(t), tiles = max(tiles_of(t), 1), all = tiles * a.hkv;
      if (a.slots > 0 && chunks > a.least) cut = max(a.least, (chunks + a.slots / all - 1) / max(a.slots / all, 1));
      u.part = at / tiles;
      u.tile = at - u.part * tiles;
      u.nparts = (chunks + min(cut, chunks) - 1) / min(cut, chunks);
      if (u.part >= u.nparts) return false;
      if (a.plan && blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = make_int2(0, u.nparts);
    } else {
      u.tile = at % a.ntiles;
      u.seq = at / a.ntiles;
    }
  } else {
    __shared__ PlanShared sh;
    const int tid = threadIdx.x, w = tid >> 6;
    int chunks = 0, tiles = 0;
    if (tid < a.num_seqs) {
      const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, tid);
      tiles = tiles_of(t);
      chunks = tiles > 0 ? chunks_of(t) : 0;
    }
    // of the workgroup's threads: sums of x and y, the largest z
    int turn = 0;
    auto combine = [&](int& x, int& y, int& z) {
      int(*sums)[3] = sh.sums[turn];
      turn ^= 1;  // one barrier a turn: the one before last has been read
      const int wx = wave_combine(x, add_int), wy = wave_combine(y, add_int), wz = wave_combine(z, max_int);
      if ((tid & 63) == 0) {
        sums[w][0] = wx;
        sums[w][1] = wy;
        sums[w][2] = wz;
      }
      __syncthreads();
      x = y = z = 0;
      for (int i = 0; i < kThreads / 64; ++i) {
        x += sums[i][0];
        y += sums[i][1];
        z = max(z, sums[i][2]);
      }
      x = __builtin_amdgcn_readfirstlane(x);
      y = __builtin_amdgcn_readfirstlane(y);
      z = __builtin_amdgcn_readfirstlane(z);
    };
    // (a sequence counts for 2^22 chunks at most, which keeps the sum in 32 bits)
    int all = tiles, work = static_cast<int>(min(static_cast<int64_t>(chunks) * tiles, int64_t{1} << 22)), longest = chunks;
    combine(all, work, longest);
    all *= a.hkv;
    int pieces = all;
    const float total = static_cast<float>(work) * a.hkv;
    if (a.slots > all && static_cast<float>(longest) * a.cus > total) {
      int want = max(a.least, static_cast<int>(total / a.slots));
      for (int round = 0; round < 8 && want < longest; ++round) {
        int n = tiles * ((chunks + want - 1) / want), none = 0, zero = 0;
        combine(n, none, zero);
        n *= a.hkv;
        if (n <= a.slots) {
          cut = want;
          pieces = n;
          break;
        }
        want = max(want + 1, static_cast<int>(static_cast<float>(want) * n / a.slots));
      }
    }
    if (at >= pieces) return false;
    if (cut >= longest && pieces <= 3 * a.cus && (at / a.cus) % 2 == 1) {  // folded: rows of a workgroup a CU
      const int first = at / a.cus * a.cus;
      at = first + min(a.cus, pieces - first) - 1 - (at - first);
    }
    u.kvh = at % a.hkv;
    at /= a.hkv;
    const uint32_t key = static_cast<uint32_t>(min(chunks, 0xffffff)) * kPlanned + (kPlanned - 1 - tid);
    const int parts = cut >= longest ? min(chunks, 1) : (chunks + cut - 1) / cut, mine = tiles * parts;
    sh.key[tid] = tid < a.num_seqs ? key : 0;
    sh.count[tid] = mine;
    __syncthreads();
    int before = 0;  // pieces of the sequences that come first
    for (int j = 0; j < a.num_seqs; j += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(&sh.key[j]);
      const int4 n = *reinterpret_cast<const int4*>(&sh.count[j]);
      before += (k.x > key ? n.x : 0) + (k.y > key ? n.y : 0) + (k.z > key ? n.z : 0) + (k.w > key ? n.w : 0);
    }
    if (before <= at && at < before + mine) {
      sh.found[0] = tid;
      sh.found[1] = before;
      sh.found[2] = parts;
      sh.found[3] = tiles;
    }
    if (a.plan && blockIdx.x == 0 && tid < a.num_seqs) a.plan[tid] = make_int2(before, parts);
    __syncthreads();
    u.seq = __builtin_amdgcn_readfirstlane(sh.found[0]);
    u.nparts = __builtin_amdgcn_readfirstlane(sh.found[2]);
    const int n = __builtin_amdgcn_readfirstlane(sh.found[3]), place = at - __builtin_amdgcn_readfirstlane(sh.found[1]);
    u.part = place / n;
    u.tile = place - u.part * n;
  }
  u.t = fi::tree_span(a.cu_seqlens, a.context_lens, u.seq);
  u.nodes = min(u.t.nodes, a.max_query_len);
  if (u.part == 0 && u.tile == 0 && u.kvh == 0 && threadIdx.x == 0) {
    if (u.t.nodes > a.max_query_len) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
    if (u.t.prefix + u.t.nodes > a.max_context_len) atomicOr(a.faults, FI_FAULT_CONTEXT_RANGE);
  }
  u.tiles = tiles_of(u.t);
  if (u.tile >= u.tiles) return false;
  u.kend = key_end(a, u.t);
  const int chunks = (u.kend + KB - 1) / KB;
  u.c_lo = u.nparts > 1 ? u.part * cut : 0;
  u.c_hi = u.nparts > 1 ? min(u.c_lo + cut, chunks) : chunks;
  return true;
}

// Whether a chunk reaches past the prefix, or past the keys.
template <int KB>
__device__ __forceinline__ bool reaches(const Unit& u, int c) {
  return (c + 1) * KB > min(u.t.prefix, u.kend);
}

// ---- parts ----
// A piece's partials, and the join of a tile's.  Where the last workgroup of a tile joins them, they are read by
// another workgroup of the launch: device-coherent stores and loads (past the XCDs' private L2s), eight
// bytes each.

__device__ __forceinline__ void put2(float* p, float x, float y, bool coherent) {
  const uint64_t v = static_cast<uint64_t>(__float_as_uint(x)) | (static_cast<uint64_t>(__float_as_uint(y)) << 32);
  if (coherent)
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    *reinterpret_cast<uint64_t*>(p) = v;
}
template <bool COHERENT>
__device__ __forceinline__ float2 get2(const float* p) {
  uint64_t v;
  if constexpr (COHERENT)
    v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    v = *reinterpret_cast<const uint64_t*>(p);
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// A lane's share of row r: O at d = 16 dt + 4 lk .. + 3; its reference point (a finite one where the sum is NaN,
// which the join does not skip) and sum.
template <int D>
__device__ __forceinline__ void store_part(const TreeArgs& a, const Unit& u, int r, int lk, const v4f (&o)[D / 16], float m,
                                           float sum) {
  const bool coherent = a.plan == nullptr;
  float* acc = a.part_acc + ((size_t)u.piece * kRows + r) * D + 4 * lk;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) {
    put2(acc + 16 * dt, o[dt][0], o[dt][1], coherent);
    put2(acc + 16 * dt + 2, o[dt][2], o[dt][3], coherent);
  }
  if (lk == 0) put2(a.part_ml + ((size_t)u.piece * kRows + r) * 2, m, sum, coherent);
}

// Row r's elements 4 dq .. + 3 of the tile whose parts are the pieces first + step * part, joined in part order, each
// rescaled from its own reference point to the largest so far (a part without a key that the row sees carries
// -inf and adds nothing), divided by the combined sum.
template <int D, int ITEMS, bool COHERENT>
__device__ __forceinline__ void join_parts(const TreeArgs& a, const fi::TreeSpan& t, int kvh, int tile, int first, int step,
                                           int nparts, int from, int stride) {
  constexpr int N = 16 / ITEMS < 8 ? 16 / ITEMS : 8, DQ = D / 4;  // N parts' loads are issued together
  float mx[ITEMS], l[ITEMS];
  float4 acc[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    mx[i] = -INFINITY;
    l[i] = 0.0f;
    acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int s0 = 0; s0 < nparts; s0 += N) {
    float2 ml[N][ITEMS], lo[N][ITEMS], hi[N][ITEMS];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int idx = from + i * stride;
        const size_t row = (size_t)(first + step * min(s0 + n, nparts - 1)) * kRows + idx / DQ;
        ml[n][i] = get2<COHERENT>(a.part_ml + row * 2);
        lo[n][i] = get2<COHERENT>(a.part_acc + row * D + 4 * (idx % DQ));
        hi[n][i] = get2<COHERENT>(a.part_acc + row * D + 4 * (idx % DQ) + 2);
      }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (s0 + n >= nparts || ml[n][i].x == -INFINITY) continue;
        const float to = fmaxf(mx[i], ml[n][i].x);
        const float old = __builtin_amdgcn_exp2f(mx[i] - to), now = __builtin_amdgcn_exp2f(ml[n][i].x - to);
        mx[i] = to;
        l[i] = l[i] * old + now * ml[n][i].y;
        acc[i] = make_float4(acc[i].x * old + now * lo[n][i].x, acc[i].y * old + now * lo[n][i].y,
                             acc[i].z * old + now * hi[n][i].x, acc[i].w * old + now * hi[n][i].y);
      }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int idx = from + i * stride, r = tile * kRows + idx / DQ;
    const int node = static_cast<int>(a.by_group.div(r)), head = kvh * a.group + (r - node * a.group);
    if (node >= min(t.nodes, a.max_query_len)) continue;
    // (several parts and no prefix: a tree longer than a part)
    const float inv = l[i] == 0.0f && sees_nothing(a, t, key_end(a, t), a.mask + (size_t)(t.first + node) * a.words) ? 0.0f : 1.0f / l[i];
    *reinterpret_cast<float4*>(a.out + ((size_t)(t.first + node) * a.hq + head) * D + 4 * (idx % DQ)) =
        make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
  }
}

// The end of a workgroup of a cut tile where the launch joins by itself: the tile's last joins its parts.  Each
// thread waits until its coherent stores have completed, so when the counter shows every part's arrival, every
// partial can be read.  The last resets the counter for the next launch or graph replay.
template <int D>
__device__ __forceinline__ void join_last(const TreeArgs& a, const Unit& u) {
  if (u.nparts <= 1 || a.plan != nullptr) return;  // workgroup-uniform
  __shared__ int s_last;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* counter = a.counters + ((size_t)u.seq * a.ntiles + u.tile) * a.hkv + u.kvh;
    const unsigned arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    s_last = arrived == static_cast<unsigned>(u.nparts);
    if (s_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  const int step = u.tiles * a.hkv;
  join_parts<D, kRows * (D / 4) / kThreads, true>(a, u.t, u.kvh, u.tile, u.piece - u.part * step, step, u.nparts, threadIdx.x, kThreads);
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
    c2 = a.scale * 1.4426950408889634f;
#pragma unroll
    for (int s = 0; s < DS; ++s) split3(query(a, at, s), qf[s]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.0f;
  }
  __device__ __forceinline__ f32x8 query(const TreeArgs& a, const Place& at, int s) const {
    const float* q = a.q + at.index * D + 8 * lk + 32 * s;
    const float4 lo = *reinterpret_cast<const float4*>(q), hi = *reinterpret_cast<const float4*>(q + 4);
    const f32x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    return at.live ? v : z;
  }

  // Which of the keys k0 .. k0 + 63 the row sees, and -inf for the scores of the others: s[jt][v] is that of key
  // 16 jt + 4 lk + v.
  template <int JT>
  __device__ __forceinline__ uint64_t hide(const TreeArgs& a, const Unit& u, int k0, v4f (&s)[JT]) const {
    const uint64_t seen = fi::mask_window(a.mask + place(a, u).row * a.words, a.words, k0 - u.t.prefix) & fi::keys_before(u.kend, k0);
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

  // What is not finite in V, for the rows that see it: `keys` of the chunk at k0, all before u.kend (their blocks are
  // looked up again).
  template <typename P>
  __device__ __forceinline__ void add_special(const TreeArgs& a, const Unit& u, int k0, uint64_t keys, uint64_t seen) {
    for (; keys != 0; keys &= keys - 1) {  // workgroup-uniform
      const int key = __builtin_ctzll(keys), lb = static_cast<int>(a.by_block.div(k0 + key));
      if (!((seen >> key) & 1)) continue;
      const int id = a.block_tables[(size_t)u.seq * a.max_blocks + lb];
      if (id < 0 || id >= a.num_blocks) continue;
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
    if (u.nparts > 1) {
      store_part<D>(a, u, 16 * (threadIdx.x >> 6) + li, lk, o, sum != sum ? 0.f : m, sum);
      return;
    }
    const Place p = place(a, u);
    if (!p.live) return;
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
// wait_loads and a barrier.  m0, the LDS address, needs a wait state between its write and the load.
__device__ __forceinline__ void load_to_lds(const uint8_t* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
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
    if (past) {  // what is not finite in V is noted and cleared; the copies of the last key that lie past the end are cleared alone
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
          atomicOr(&s_special, (1ull << key_of(x)) & fi::keys_before(u.kend, k0));
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
  join_last<D>(a, u);
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
  auto stage = [&](int c) {  // and a barrier
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
    __syncthreads();
  };

  if (tid < 2) s_special[tid] = 0;
  if (u.c_lo < u.c_hi) {  // workgroup-uniform
    lookup(u.c_lo);
    fetch();
    lookup(u.c_lo + 1);
    __syncthreads();
    stage(u.c_lo);
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
    if (c + 1 < u.c_hi) stage(c + 1);  // workgroup-uniform
  }
  if (bad_block) atomicOr(a.faults, FI_FAULT_BLOCK_RANGE);
  row.finish(a, u);
  join_last<D>(a, u);
}

// The join in a launch of its own, of many tiles: 256 quads of a (sequence, tile, kv head) at a time.
template <int D>
__global__ __launch_bounds__(kThreads) void tree_join_kernel(TreeArgs a, int units) {
  constexpr int BLOCKS = kRows * (D / 4) / kThreads;
  for (int i = blockIdx.x; i < units * BLOCKS; i += gridDim.x) {
    const int share = i % BLOCKS, kvh = i / BLOCKS % a.hkv;
    const int tile = i / BLOCKS / a.hkv % a.ntiles, seq = i / BLOCKS / a.hkv / a.ntiles;
    const int2 plan = a.plan[seq];
    if (plan.y <= 1) continue;  // written by the launch before
    const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, seq);
    const int tiles = (min(t.nodes, a.max_query_len) * a.group + kRows - 1) / kRows;
    if (tile >= tiles) continue;
    join_parts<D, 1, false>(a, t, kvh, tile, (plan.x + tile) * a.hkv + kvh, tiles * a.hkv, plan.y, share * kThreads + threadIdx.x, 0);
  }
}

// The same where few tiles have many parts: a workgroup a row, whose threads share the parts (strands of every S-th, each in
// order, then joined in pairs), so that the partials' way is not one part behind the other: one sequence of 100000
// tokens, 2 kv heads of 64, 320 parts: 7 us, 52 with 256 quads a workgroup.
template <int D>
__global__ __launch_bounds__(kThreads) void tree_join_rows_kernel(TreeArgs a, int rows) {
  constexpr int DQ = D / 4, S = kThreads / DQ, N = 4;
  __shared__ float4 s_acc[S][DQ];
  __shared__ float2 s_ml[S];
  const int q = threadIdx.x % DQ, strand = threadIdx.x / DQ;
  for (int i = blockIdx.x; i < rows; i += gridDim.x) {  // what is skipped is so for the workgroup
    const int kvh = i / kRows % a.hkv, tile = i / kRows / a.hkv % a.ntiles, seq = i / kRows / a.hkv / a.ntiles;
    const int2 plan = a.plan[seq];
    if (plan.y <= 1) continue;
    const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, a.context_lens, seq);
    const int nodes = min(t.nodes, a.max_query_len), tiles = (nodes * a.group + kRows - 1) / kRows;
    const int r = tile * kRows + i % kRows, node = static_cast<int>(a.by_group.div(r));
    if (node >= nodes) continue;
    const size_t first = (size_t)((plan.x + tile) * a.hkv + kvh) * kRows + i % kRows, step = (size_t)tiles * a.hkv * kRows;
    float mx = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 x) {
      if (ml.x == -INFINITY) return;
      const float to = fmaxf(mx, ml.x), old = __builtin_amdgcn_exp2f(mx - to), now = __builtin_amdgcn_exp2f(ml.x - to);
      mx = to;
      l = l * old + now * ml.y;
      acc = make_float4(acc.x * old + now * x.x, acc.y * old + now * x.y, acc.z * old + now * x.z, acc.w * old + now * x.w);
    };
    for (int p0 = strand; p0 < plan.y; p0 += N * S) {
      float2 ml[N];
      float4 x[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const size_t row = first + step * min(p0 + n * S, plan.y - 1);
        ml[n] = get2<false>(a.part_ml + row * 2);
        x[n] = *reinterpret_cast<const float4*>(a.part_acc + row * D + 4 * q);
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (p0 + n * S < plan.y) add(ml[n], x[n]);
    }
    for (int half = S / 2; half >= 1; half /= 2) {
      __syncthreads();  // the last step's (row's) readers are done
      if (strand >= half && strand < 2 * half) {
        s_acc[strand][q] = acc;
        if (q == 0) s_ml[strand] = make_float2(mx, l);
      }
      __syncthreads();
      if (strand < half) add(s_ml[strand + half], s_acc[strand + half][q]);
    }
    if (strand != 0) continue;
    const int head = kvh * a.group + (r - node * a.group);
    const float inv = l == 0.0f && sees_nothing(a, t, key_end(a, t), a.mask + (size_t)(t.first + node) * a.words) ? 0.0f : 1.0f / l;
    *reinterpret_cast<float4*>(a.out + ((size_t)(t.first + node) * a.hq + head) * D + 4 * q) =
        make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
}

template <int D, int POOL>
int32_t launch_tree(fi_context* ctx, TreeArgs& a) {
  constexpr int KB = POOL == FI_DTYPE_F32 ? 32 : 64;  // keys of a chunk
  const int64_t cus = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int64_t rows = static_cast<int64_t>(a.max_query_len) * a.group;
  FI_REQUIRE(rows < (1 << 30), FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: too many rows");
  a.ntiles = static_cast<int>((rows + kRows - 1) / kRows);
  const int64_t tiles = static_cast<int64_t>(a.num_seqs) * a.hkv * a.ntiles;
  FI_REQUIRE(tiles <= 0x7fffffff, FI_ERR_INVALID_SHAPE, "fi_attn_tree_paged: grid too large");
  const int64_t chunks = (static_cast<int64_t>(a.max_context_len) + KB - 1) / KB;
  a.cus = static_cast<int>(cus);
  // Parts of four chunks and more (us with two, three and four: 8 sequences of 200 to 1000 tokens, 32/8 heads of 128,
  // 29.4, 25.6, 25.2; 16 of 200 to 1500 over 14/2 heads of 64, f32, 24.1, 22.9, 21.1; one of 4000 25.2, 25.0, 23.4).
  a.least = 4;
  // Workgroups that run at a time: three a CU, two where f32 rows of 128 take the registers.  Launches of two tiles a CU
  // are not cut (64 sequences of 128 to 2048: 80 us, cut into parts of 16 chunks 81 and the join).
  const int64_t slots = (D == 128 && POOL == FI_DTYPE_F32 ? 2 : 3) * cus;
  int64_t grid = tiles;
  bool join = false;
  if (a.num_seqs <= kPlanned && tiles < 2 * cus && chunks > a.least) {  // may be cut
    a.slots = static_cast<int>(slots);
    grid = slots;
    const size_t acc = static_cast<size_t>(slots) * kRows * D * sizeof(float), ml = static_cast<size_t>(slots) * kRows * 2 * sizeof(float);
    FI_TRY(fi::ensure_workspace(ctx, acc + ml + kPlanned * sizeof(int2)));
    a.part_acc = static_cast<float*>(ctx->workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ctx->workspace) + acc);
    // The last workgroup of a tile joins its parts by itself where they are few and tiles many; otherwise a launch does
    // (one sequence of 700 tokens over 14/2 heads of 64, f32, six parts: 19.1 us by itself, 16.6 by a launch; 32
    // sequences of 200 to 1900 over 32/8 heads of 128, 256 tiles of up to eight: 64.5 and 59.6; 60 of them, 480 tiles: 75.4
    // and 80.1).
    join = chunks > (tiles <= cus ? 4 : 8) * a.least;
    if (join)
      a.plan = reinterpret_cast<int2*>(static_cast<char*>(ctx->workspace) + acc + ml);
    else
      a.counters = ctx->d_merge_counters;  // a tile each: fewer than slots
  }
  if constexpr (POOL == FI_DTYPE_BF16)
    hipLaunchKernelGGL((attn_tree_bf16_kernel<D>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL((attn_tree_kernel<D, POOL>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, ctx->stream, a);
  FI_CHECK_LAUNCH("attn_tree_kernel");
  if (join && tiles <= kRowJoins) {
    const int64_t rows = tiles * kRows;
    hipLaunchKernelGGL((tree_join_rows_kernel<D>), dim3(static_cast<unsigned>(std::min<int64_t>(rows, 8 * cus))), dim3(kThreads), 0,
                       ctx->stream, a, static_cast<int>(rows));
    FI_CHECK_LAUNCH("tree_join_rows_kernel");
  } else if (join) {
    const int64_t blocks = std::min<int64_t>(tiles * (kRows * (D / 4) / kThreads), 8 * cus);
    hipLaunchKernelGGL((tree_join_kernel<D>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, ctx->stream, a,
                       static_cast<int>(tiles));
    FI_CHECK_LAUNCH("tree_join_kernel");
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
