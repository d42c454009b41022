// Verification of drafted tokens: a walk from a tree's root that accepts a child of the node it is at, or
// ends there and draws one more token, so that the tokens are distributed as sampling from the model's own
// logits would give them.  No counterpart in the reference, whose sessions draw one token a step
// (crates/ferrisinfer-runtime/src/session.rs:246-262, sampler.rs:121-241).
//
// At a node with the model's distribution p, children x_1, x_2, ... in node order are tried against the rest
// of p that earlier ones have left: rho_0 = p, Z = sum(rho).
//   tokens given (no draft probabilities): x is accepted when u Z < rho(x); otherwise rho(x) becomes 0;
//   tokens drawn from q: x is accepted when u c q(x) < rho(x), c = Z / (1 - s) (that is min(1, rho / (Z q')),
//     q' = q without the s of the earlier children where they are distinct); otherwise rho becomes
//     max(rho - c q, 0).
// max(max(p - a q, 0) - c q, 0) = max(p - (a + c) q, 0) for q, c >= 0, so rho is never stored: it is
// max(p - a q, 0) with a number a, and each rejection costs one pass over the two rows.  (A rejected child's rho is 0
// from then on: it was below c q.  So taking it out of q as well changes nothing.)  The token at the end is
// the first index at which the running sum of rho passes u Z.
//
// Tokens are compared with u at borders that lie 1e-7 and less apart in a flat row, so what decides is in 64
// bits: exponentials and sums to 1e-14.
//
// A workgroup reads a row at 50 GB/s at most, whatever it keeps in flight (12 us for 600 KB), so a row is split over
// one workgroup a segment of 4096, and a walk goes from launch to launch: in each, a sequence's segments are summed
// for the row that its walk is at, and the last workgroup to finish takes the walk on, to the next row or to
// the end.  No workgroup waits for another.  The host knows how many launches a walk can need; those of
// sequences that have ended are left at once.
#include <algorithm>
#include <type_traits>

#include "fi_common.h"
#include "fi_device.h"
#include "fi_tree.h"

namespace {

struct VerifyArgs {
  const float* logits;  // [T, ld]
  const int* tokens;    // [T]
  const int* parents;   // [T]
  const int* cu_seqlens;
  const float* temperature;  // [B]
  const float* probs;        // [T, ld_probs] or null
  const float* accept_u;     // [T]
  const float* pick_u;       // [B]
  int* out_tokens;           // [B, max_path + 1]
  int* out_path;             // [B, max_path]
  int* out_count;            // [B]
  float* out_prob;           // [B]
  struct Walk* walks;        // [B]
  struct RowSums* sums;      // [B, segments] of the row that the walk is at, or [B * max_query_len, segments] of all
  double* rests;             // [B, segments] of what is left of it
  unsigned* counters;        // [B] (and [B * max_query_len] behind them, where all rows are summed), `apart` apart; zero between launches
  uint32_t* faults;
  int64_t ld, ld_probs;
  int vocab, distinct, max_path, max_query_len, segments;
  int all_rows;  // sums are of all rows
  int apart;
};

enum Phase : int {
  kTotal,  // the row's sums are asked for
  kRest,   // children were rejected: the sums of what is left
  kDone,
};

// Where a sequence's walk is.
struct Walk {
  int node, count;  // the node; how many tokens are accepted
  int phase;
  int child;     // the last one rejected (tokens drawn)
  float ref;     // the reference point of the row's weights
  double off, taken;  // a and s
};

// Weights by a reference point are 2^(k (l - point)): k = log2(e) / temperature, l the logit.  (The difference comes first:
// k l and k point are 2^128 where a row is masked by finite numbers, and their roundings 2^75.  As one fused operation with k point
// rounded beforehand it was no faster.)
struct Weights {
  double k, point;
};

constexpr double kLog2E = 1.4426950408889634;
constexpr float kMinTemperature = 1.1920929e-7f;  // as sampling has it (f32::EPSILON)

__device__ __forceinline__ double row_scale(float temperature) {
  return kLog2E / static_cast<double>(fmaxf(temperature, kMinTemperature));
}

// 2^x for x in [-1100, 0]: 2^n times a polynomial in f, |f| <= 1/2, through 2^f at the eleven Chebyshev
// points; it is within 3.2e-16 of 2^f.
__device__ __forceinline__ double exp2_64(double x) {
  const double n = __builtin_rint(x), f = x - n;
  double s = 7.072585949269223e-09;
  s = __builtin_fma(s, f, 1.0208690299958306e-07);
  s = __builtin_fma(s, f, 1.321544258792169e-06);
  s = __builtin_fma(s, f, 1.5252657260200837e-05);
  s = __builtin_fma(s, f, 0.0001540353044173605);
  s = __builtin_fma(s, f, 0.0013333558230164974);
  s = __builtin_fma(s, f, 0.009618129107606888);
  s = __builtin_fma(s, f, 0.05550410866444772);
  s = __builtin_fma(s, f, 0.24022650695910097);
  s = __builtin_fma(s, f, 0.69314718055995);
  s = __builtin_fma(s, f, 1.0);
  return __builtin_ldexp(s, static_cast<int>(n));
}

// A logit's weight, by a reference point that none of those summed passes; one of -inf (and, where k is 0, NaN from it) weighs
// nothing.
__device__ __forceinline__ double weight(double l, const Weights& w) {
  return exp2_64(__builtin_fmax((l - w.point) * w.k, -1100.0));
}

// What weights by `from` are multiplied with to be weights by `to`, which is no less.
__device__ __forceinline__ double change_of_ref(double k, float from, float to) {
  return weight(from, Weights{k, to});
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.0f; }

__device__ __forceinline__ bool unusable(float l) { return !(l <= 3.402823466e38f); }  // NaN or +inf

// What another lane holds, or `otherwise`, on the vector pipe (a shuffle is an LDS round trip).
template <int kCtrl, int kRows>
__device__ __forceinline__ int from_lane(int v, int otherwise) {
  return __builtin_amdgcn_update_dpp(otherwise, v, kCtrl, kRows, 0xf, false);
}
// f over the lanes up to each one, in order, and so over the wave in its last: within rows of 16 lanes (row_shr:1, 2, 4, 8),
// then a row's last to the next (row_bcast:15) and the half's last to the next half (:31).
template <typename F>
__device__ __forceinline__ void up_the_wave(F f) {
  f(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});
  f(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  f(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  f(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  f(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  f(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
}
__device__ __forceinline__ double wave_scan64(double v) {
  up_the_wave([&](auto ctrl, auto rows) {
    const int2 x = __builtin_bit_cast(int2, v);
    v += __builtin_bit_cast(double, make_int2(from_lane<ctrl.value, rows.value>(x.x, 0), from_lane<ctrl.value, rows.value>(x.y, 0)));
  });
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
  const int2 x = __builtin_bit_cast(int2, wave_scan64(v));
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(x.x, 63), __builtin_amdgcn_readlane(x.y, 63)));
}
__device__ __forceinline__ float wave_top(float v) {
  up_the_wave([&](auto ctrl, auto rows) {
    const int x = __builtin_bit_cast(int, v);
    v = fmaxf(v, __builtin_bit_cast(float, from_lane<ctrl.value, rows.value>(x, x)));
  });
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// The least of the wave's indexes whose value is the wave's largest.
__device__ __forceinline__ int first_of(float value, float top, int index) {
  int at = value == top ? index : 0x7fffffff;
  up_the_wave([&](auto ctrl, auto rows) { at = min(at, from_lane<ctrl.value, rows.value>(at, at)); });
  return __builtin_amdgcn_readlane(at, 63);
}

// Four logits (probabilities) from `at` on, those past the row's end as `pad`; VEC: rows of whole,
// 16-byte aligned quads.
template <bool VEC>
__device__ __forceinline__ float4 quad_at(const float* __restrict__ row, int at, int vocab, float pad) {
  if constexpr (VEC) {
    return at < vocab ? *reinterpret_cast<const float4*>(row + at) : make_float4(pad, pad, pad, pad);
  } else {
    return make_float4(at < vocab ? row[at] : pad, at + 1 < vocab ? row[at + 1] : pad, at + 2 < vocab ? row[at + 2] : pad,
                       at + 3 < vocab ? row[at + 3] : pad);
  }
}

// ---------------------------------------------------------------- segments of a row

// 16 elements a thread: 64 sequences of five rows of 128k logits 90 us (8: 92, 32: 111), 16 trees 98 (92, 121), one
// sequence of 152k 22 (22, 25).
constexpr int kEndThreads = 256;
constexpr int kEndElems = 16;
constexpr int kSegment = kEndThreads * kEndElems;   // 4096
constexpr int kMaxSegments = 256;                   // four a lane when they are joined
constexpr int kMaxVocab = kSegment * kMaxSegments;  // 1048576

constexpr int64_t kAllRows = 20000000;  // logits up to which every row is summed in the first launch
constexpr int kRejections = 4;          // launches for rejected drawn children
constexpr int kDepth = 16;              // for rows behind the root's

// A workgroup is one group of threads for a segment, or four of them side by side (verify_finish_kernel), of which each sums
// a segment and all do the rest alike.
__device__ __forceinline__ int thread_of() { return threadIdx.x % kEndThreads; }
__device__ __forceinline__ int group_of() { return threadIdx.x / kEndThreads; }

// Of a segment: the weights' sum by its maximum (by 0 where that is not finite; NaN if there is a logit that is NaN or
// +inf), the maximum and its first index.
struct alignas(16) RowSums {
  double sum;
  float top;
  int first;
};

struct SegmentShared {
  double scan[kEndThreads / 64];
  float tops[kEndThreads / 64];
  int firsts[kEndThreads / 64];
};

// The workgroup's maximum; its first index too, if that is asked for.
__device__ __forceinline__ void segment_top(SegmentShared& sh, float& top, int& first, bool index) {
  const int lane = thread_of() & 63, w = thread_of() >> 6;
  const float wave = wave_top(top);
  const int at = index ? first_of(top, wave, first) : 0;
  __syncthreads();  // the last use is over
  if (lane == 0) {
    sh.tops[w] = wave;
    sh.firsts[w] = at;
  }
  __syncthreads();
  top = -INFINITY;
  first = 0x7fffffff;
  for (int i = 0; i < kEndThreads / 64; ++i)
    if (sh.tops[i] > top || (sh.tops[i] == top && sh.firsts[i] < first)) {  // (a wave's elements are not all before the next one's)
      top = sh.tops[i];
      first = sh.firsts[i];
    }
}
// The workgroup's sum of x.
__device__ __forceinline__ double segment_sum(SegmentShared& sh, double x) {
  x = wave_sum64(x);
  __syncthreads();  // the last use is over
  if ((thread_of() & 63) == 0) sh.scan[thread_of() >> 6] = x;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < kEndThreads / 64; ++i) all += sh.scan[i];
  return all;
}

// A thread's 16 elements of a segment: quads 256 apart (whole lines a wave), or one behind the other (in order).
template <bool VEC, bool IN_ORDER>
__device__ __forceinline__ void segment_load(const float* __restrict__ row, int begin, int vocab, float pad, float (&v)[kEndElems]) {
#pragma unroll
  for (int j = 0; j < kEndElems / 4; ++j) {
    const float4 x = quad_at<VEC>(row, begin + (IN_ORDER ? thread_of() * kEndElems + 4 * j : 4 * thread_of() + 4 * kEndThreads * j), vocab, pad);
    v[4 * j] = x.x;
    v[4 * j + 1] = x.y;
    v[4 * j + 2] = x.z;
    v[4 * j + 3] = x.w;
  }
}
// The place in the segment of a thread's element e, as they are loaded out of order.
__device__ __forceinline__ int element_at(int e) { return 4 * thread_of() + 4 * kEndThreads * (e / 4) + e % 4; }

// ---------------------------------------------------------------- a launch's part

constexpr int kGroups = 4;

struct VerifyShared {
  SegmentShared seg[kGroups];
  uint32_t out[kGroups][kSegment / 32];   // tokens given and rejected
  uint64_t kids[fi::kMaxTreeNodes / 64];  // the node's children, as bits
  int tokens[fi::kMaxTreeNodes];
  float accept[fi::kMaxTreeNodes];
  float probs[fi::kMaxTreeNodes];
  double mass[fi::kMaxTreeNodes];  // weights of the children's tokens
  int last;
};

template <typename T>
__device__ __forceinline__ void put(T* to, T x) {  // for another workgroup of this launch
  __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(T* from) {
  return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A sequence: its nodes, its row scale, its outputs.
struct Sequence {
  int index, first, n;
  bool greedy;
  double k;
};

__device__ __forceinline__ Sequence sequence_of(const VerifyArgs& a, int index) {
  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, nullptr, index);
  const float temperature = a.temperature[index];
  const bool greedy = temperature <= 0.0f;
  return Sequence{index, t.first, min(t.nodes, a.max_query_len), greedy, greedy ? kLog2E : row_scale(temperature)};
}

// A node, and its token's logit and draft probability where it is a child of the node that the walk is at.
struct Node {
  int parent, token;
  float accept, logit, prob;
  bool child;
};

__device__ __forceinline__ Node node_at(const VerifyArgs& a, const Sequence& s, int j) {
  Node x{-2, -1, 0.0f, 0.0f, 0.0f, false};
  if (j < s.n) {
    x.parent = a.parents[s.first + j];
    x.token = a.tokens[s.first + j];
    x.accept = a.accept_u[s.first + j];
  }
  return x;
}
__device__ __forceinline__ void look_up(const VerifyArgs& a, const Sequence& s, int node, int j, Node& x) {
  x.child = j > node && x.parent == node && x.token >= 0 && x.token < a.vocab;  // (no token: as if it were not there)
  if (x.child && !s.greedy) {
    x.logit = a.logits[(int64_t)(s.first + node) * a.ld + x.token];
    if (a.probs) x.prob = a.probs[(int64_t)(s.first + node) * a.ld_probs + x.token];
  }
}

// Marks the tokens of a segment that were tried (tokens given, and rejected).
__device__ __forceinline__ void mark_tried(const VerifyArgs& a, VerifyShared& sh, const Sequence& q, int node, int begin) {
  __syncthreads();
  for (int i = thread_of(); i < kSegment / 32; i += kEndThreads) sh.out[group_of()][i] = 0;
  __syncthreads();
  for (int j = node + 1 + thread_of(); j < q.n; j += kEndThreads) {
    const int x = a.tokens[q.first + j];
    if (a.parents[q.first + j] == node && x >= begin && x < min(begin + kSegment, a.vocab))
      atomicOr(&sh.out[group_of()][(x - begin) >> 5], 1u << ((x - begin) & 31));
  }
  __syncthreads();
}
__device__ __forceinline__ bool was_tried(const VerifyShared& sh, int e) { return ((sh.out[group_of()][e >> 5] >> (e & 31)) & 1) != 0; }

// The sums of a segment that the walk asks for; thread 0 stores them.  Meanwhile the thread's node is looked up, as a child of
// node `from`: only the last workgroup needs it, but that then waits for nothing.
template <bool VEC>
__device__ __forceinline__ void sum_segment(const VerifyArgs& a, VerifyShared& sh, const Sequence& s, const Walk& walk, int segment,
                                            int from, Node& mine) {
  const int begin = segment * kSegment;
  const bool less = walk.phase == kRest && a.probs;
  float v[kEndElems], q[kEndElems];
  segment_load<VEC, false>(a.logits + (int64_t)(s.first + walk.node) * a.ld, begin, a.vocab, -INFINITY, v);
  if (less) segment_load<VEC, false>(a.probs + (int64_t)(s.first + walk.node) * a.ld_probs, begin, a.vocab, 0.0f, q);
  mine = node_at(a, s, thread_of());
  look_up(a, s, from, thread_of(), mine);
  double sum = 0.0;
  if (less) {
    const Weights by{s.k, walk.ref};
#pragma unroll
    for (int e = 0; e < kEndElems; ++e) sum += __builtin_fmax(weight(v[e], by) - walk.off * q[e], 0.0);
    sum = segment_sum(sh.seg[group_of()], sum);
    if (thread_of() == 0 && segment < a.segments) put(&a.rests[(size_t)s.index * a.segments + segment], sum);
    return;
  }
  float top = walk.ref;
  int first = 0x7fffffff;
  bool bad = false;
  if (walk.phase == kRest) {
    mark_tried(a, sh, s, walk.node, begin);
#pragma unroll
    for (int e = 0; e < kEndElems; ++e) v[e] = was_tried(sh, element_at(e)) ? -INFINITY : v[e];
  } else {
    top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kEndElems; ++e) {
      bad |= unusable(v[e]);
      top = fmaxf(top, v[e]);
    }
    if (s.greedy) {
#pragma unroll
      for (int e = kEndElems - 1; e >= 0; --e)  // (a thread's elements rise)
        if (v[e] == top) first = begin + element_at(e);
    }
    segment_top(sh.seg[group_of()], top, first, s.greedy);
  }
  const Weights by{s.k, finite_or_zero(top)};
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) sum += weight(v[e], by);
  sum = segment_sum(sh.seg[group_of()], bad ? NAN : sum);
  if (thread_of() != 0 || segment >= a.segments) return;
  if (walk.phase == kRest) {
    put(&a.rests[(size_t)s.index * a.segments + segment], sum);
  } else {
    RowSums* to = a.sums + (a.all_rows ? (size_t)s.index * a.max_query_len + walk.node : (size_t)s.index) * a.segments + segment;
    put(&to->sum, sum);
    put(reinterpret_cast<uint64_t*>(&to->top), __builtin_bit_cast(uint64_t, make_int2(__float_as_int(top), first)));
  }
}

// The node's children: their tokens' weights, draft probabilities and random numbers.  `mine` is the thread's own
// node, looked up before.
__device__ __forceinline__ void find_children(const VerifyArgs& a, VerifyShared& sh, const Sequence& s, const Walk& walk, const Weights& by,
                                              const Node& mine) {
  __syncthreads();  // the last use is over
  for (int j = thread_of(); j < (s.n + 63) / 64 * 64; j += kEndThreads) {  // whole waves
    Node x = mine;
    if (j >= kEndThreads) {
      x = node_at(a, s, j);
      look_up(a, s, walk.node, j, x);
    }
    if (x.child) {
      sh.tokens[j] = x.token;
      sh.accept[j] = x.accept;
      sh.mass[j] = weight(x.logit, by);
      sh.probs[j] = x.prob;
    }
    const uint64_t bits = __builtin_amdgcn_ballot_w64(x.child);
    if ((j & 63) == 0) sh.kids[j >> 6] = bits;
  }
  __syncthreads();
}

// The first child behind node j, or -1.
__device__ __forceinline__ int next_child(const VerifyShared& sh, int n, int j) {
  ++j;
  for (int word = j >> 6; word < (n + 63) >> 6; ++word) {
    const uint64_t bits = sh.kids[word] & (word == j >> 6 ? ~0ull << (j & 63) : ~0ull);
    if (bits != 0) return 64 * word + __builtin_ctzll(bits);
  }
  return -1;
}

// What a segment's sums come to by the row's reference point; a lane has those of kPer segments on end, every wave all.
constexpr int kPer = kMaxSegments / 64;
constexpr double kNothing = 1e-290;  // less than this is no share (a million of the least normal numbers)

__device__ __forceinline__ int lane_of(uint64_t some, uint64_t any) {
  return some != 0 ? __builtin_ctzll(some) : any != 0 ? 63 - __builtin_clzll(any) : 0;
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  const int2 x = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(x.x, lane), __builtin_amdgcn_readlane(x.y, lane)));
}

// Draws the last token by the segments' shares: the segment, wave, lane and element at which the running sum of what is
// left passes u times all of it, each of those that have anything; past the last of them (u of 1 and more, or the sums'
// roundings) the last.
template <bool VEC>
__device__ __forceinline__ void pick_token(const VerifyArgs& a, VerifyShared& sh, const Sequence& s, const Walk& walk,
                                           const double (&part)[kPer], bool rest, float pick_u) {
  const int tid = thread_of(), lane = tid & 63, per = (a.segments + 63) / 64;
  const float* row = a.logits + (int64_t)(s.first + walk.node) * a.ld;
  const bool less = rest && a.probs, without = rest && !a.probs;
  double share = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) share += part[i];
  double run = wave_scan64(share);
  const double total = of_lane(run, 63), target = static_cast<double>(pick_u) * total;
  int from = lane_of(__builtin_amdgcn_ballot_w64(share > kNothing && run > target), __builtin_amdgcn_ballot_w64(share > kNothing));
  int segment = 0;
  double before = 0.0, at = run - share;
  bool passed = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (part[i] > kNothing / kPer && !passed) {
      segment = per * lane + i;
      before = at;
      passed = at + part[i] > target;
    }
    at += part[i];
  }
  segment = __builtin_amdgcn_readlane(segment, from);
  before = of_lane(before, from);
  float v[kEndElems], q[kEndElems];
  const int begin = segment * kSegment;
  segment_load<VEC, true>(row, begin, a.vocab, -INFINITY, v);
  if (less) {
    segment_load<VEC, true>(a.probs + (int64_t)(s.first + walk.node) * a.ld_probs, begin, a.vocab, 0.0f, q);
  } else {
#pragma unroll
    for (int e = 0; e < kEndElems; ++e) q[e] = 0.0f;
  }
  if (without) {
    mark_tried(a, sh, s, walk.node, begin);
#pragma unroll
    for (int e = 0; e < kEndElems; ++e) v[e] = was_tried(sh, tid * kEndElems + e) ? -INFINITY : v[e];
  }
  const Weights by{s.k, walk.ref};
  const double off = less ? walk.off : 0.0;
  double left[kEndElems], here = 0.0;
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    left[e] = __builtin_fmax(weight(v[e], by) - off * q[e], 0.0);
    here += left[e];
  }
  run = wave_scan64(here);
  __syncthreads();  // the last use is over
  if (lane == 63) sh.seg[0].scan[tid >> 6] = run;
  __syncthreads();
  int wave = 0;
  passed = false;
#pragma unroll
  for (int i = 0; i < kEndThreads / 64; ++i) {
    const double all = sh.seg[0].scan[i];
    if (all > 0.0 && !passed) {
      wave = i;
      at = before;
      passed = before + all > target;
    }
    before += all;
  }
  if (tid >> 6 != wave) return;
  run += at;
  from = lane_of(__builtin_amdgcn_ballot_w64(here > 0.0 && run > target), __builtin_amdgcn_ballot_w64(here > 0.0));
  if (lane != from) return;
  at = run - here;
  int token = -1;
  double mass = 0.0;
  passed = false;
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    at += left[e];
    if (left[e] > 0.0 && !passed) {
      token = begin + tid * kEndElems + e;
      mass = left[e];
      passed = at > target;
    }
  }
  // (behind barriers from where other threads cleared them)
  a.out_tokens[(size_t)s.index * (a.max_path + 1) + walk.count] = token;
  a.out_prob[s.index] = static_cast<float>(mass / total);
}

// Takes the walk on from the sums that it asked for, until it asks for others or ends.  Every wave does, so that what they
// need of each other is their lanes' nodes.
template <bool VEC>
__device__ __forceinline__ void advance(const VerifyArgs& a, VerifyShared& sh, const Sequence& s, Walk& walk, Node& mine, float pick_u) {
  const int tid = thread_of(), lane = tid & 63, per = (a.segments + 63) / 64;
  while (true) {  // mine is looked up at the walk's node
    const bool rest = walk.phase == kRest;
    double part[kPer] = {}, total;
    float top = -INFINITY;
    int first = 0x7fffffff;
    auto row_parts = [&]() {
      const RowSums* sums = a.sums + (a.all_rows ? (size_t)s.index * a.max_query_len + walk.node : (size_t)s.index) * a.segments;
      float tops[kPer];
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        tops[i] = -INFINITY;
        if (i < per && per * lane + i < a.segments) {
          const RowSums* from = sums + per * lane + i;
          part[i] = get(&from->sum);
          const int2 at = __builtin_bit_cast(int2, get(reinterpret_cast<const uint64_t*>(&from->top)));
          tops[i] = __int_as_float(at.x);
          if (tops[i] > top) {
            top = tops[i];
            first = at.y;
          }
        }
      }
      const float mine_top = top;
      top = wave_top(top);
      if (s.greedy) first = first_of(mine_top, top, first);
      walk.ref = finite_or_zero(top);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < per && tops[i] != -INFINITY) part[i] *= change_of_ref(s.k, finite_or_zero(tops[i]), walk.ref);
    };
    if (rest) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < per && per * lane + i < a.segments) part[i] = get(&a.rests[(size_t)s.index * a.segments + per * lane + i]);
    } else {
      row_parts();
    }
    total = (part[0] + part[1]) + (part[2] + part[3]);
    total = wave_sum64(total);
    if (!rest) {
      if ((!s.greedy && !(total == total)) || top == -INFINITY) {
        if (tid == 0) atomicOr(a.faults, FI_FAULT_SAMPLE_NONFINITE);
        walk.phase = kDone;
        return;
      }
    }
    // the children
    int accepted = -1;
    bool rejected = false;
    if (walk.count < a.max_path && (!rest || a.probs)) {
      find_children(a, sh, s, walk, Weights{s.k, walk.ref}, mine);
      if (s.greedy) {
        int best = 0x7fffffff;
        for (int j = lane; j < s.n; j += 64)
          if ((sh.kids[j >> 6] >> lane & 1) != 0 && sh.tokens[j] == first) best = min(best, j);
        best = first_of(0.0f, 0.0f, best);
        accepted = best == 0x7fffffff ? -1 : best;
      } else if (!a.probs) {
        // (a difference: within 1e-14 of the row's sum.  Summing the row again where little is left costs registers, a wave a SIMD
        // less: 96 us for 90 where 64 drafts of four tokens are verified.)
        double left = total;
        for (int j = next_child(sh, s.n, walk.node); j >= 0; j = next_child(sh, s.n, j)) {
          bool out = false;  // an earlier child of the same token has been taken out
          for (int i = next_child(sh, s.n, walk.node); i < j; i = next_child(sh, s.n, i)) out |= sh.tokens[i] == sh.tokens[j];
          const double mass = out ? 0.0 : sh.mass[j];
          if (sh.accept[j] * left < mass) {
            accepted = j;
            break;
          }
          left -= mass;
          rejected = true;
        }
      } else {
        const int j = walk.taken < 1.0 ? next_child(sh, s.n, max(walk.child, walk.node)) : -1;
        if (j >= 0) {
          const double q = sh.probs[j], c = total / (1.0 - walk.taken);
          if (sh.accept[j] * c * q < __builtin_fmax(sh.mass[j] - walk.off * q, 0.0)) {
            accepted = j;
          } else {
            rejected = true;
            walk.off += c;
            if (a.distinct) walk.taken += q;
            walk.child = j;
          }
        }
      }
    }
    if (accepted >= 0) {
      if (tid == walk.count % kEndThreads) {  // the thread that has cleared these
        a.out_path[(size_t)s.index * a.max_path + walk.count] = accepted;
        a.out_tokens[(size_t)s.index * (a.max_path + 1) + walk.count] = sh.tokens[accepted];
      }
      if (tid == 0) a.out_count[s.index] = walk.count + 1;
      walk = Walk{accepted, walk.count + 1, kTotal, -1, 0.0f, 0.0, 0.0};
      if (!a.all_rows) return;
      look_up(a, s, walk.node, tid, mine);
      continue;
    }
    if (rejected) {
      walk.phase = kRest;
      return;
    }
    // the end
    if (s.greedy) {
      if (tid == walk.count % kEndThreads) a.out_tokens[(size_t)s.index * (a.max_path + 1) + walk.count] = first;
      if (tid == 0) a.out_prob[s.index] = static_cast<float>(1.0 / total);
    } else {
      const bool whole = rest && !(total > kNothing);  // nothing left (p = a q but for rounding): the draw is from the distribution itself
      if (whole) row_parts();
      pick_token<VEC>(a, sh, s, walk, part, rest && !whole, pick_u);
    }
    walk.phase = kDone;
    return;
  }
}

// What a sequence's first advance finds: nothing accepted yet.
__device__ __forceinline__ void begin_outputs(const VerifyArgs& a, const Sequence& s, const Node& mine) {
  const int tid = thread_of();
  for (int i = tid; i < a.max_path; i += kEndThreads) a.out_path[(size_t)s.index * a.max_path + i] = -1;
  for (int i = tid; i <= a.max_path; i += kEndThreads) a.out_tokens[(size_t)s.index * (a.max_path + 1) + i] = -1;
  if (tid == 0) {
    a.out_count[s.index] = 0;
    a.out_prob[s.index] = 0.0f;
    if (a.cu_seqlens[s.index + 1] - a.cu_seqlens[s.index] > a.max_query_len) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
  }
  for (int i = tid; i < s.n; i += kEndThreads) {
    const Node x = i < kEndThreads ? mine : node_at(a, s, i);
    if (x.parent < -1 || x.parent >= i) atomicOr(a.faults, FI_FAULT_TREE_RANGE);
    if (i > 0 && (x.token < 0 || x.token >= a.vocab)) atomicOr(a.faults, FI_FAULT_TOKEN_RANGE);
  }
}

// One launch of the walks: a workgroup a (segment, sequence), or, the first launch where all rows are summed,
// a (segment, row).  What bounds it: the rows of 64 sequences of 128k logits, 33 MB, take 16 to 18 us.  8 us of that are the
// exponentials, 1.05e12 a second in 64 bits (as many bytes of logits as 4.2 TB/s); the rest is the arrival and the
// last workgroup's way, one memory latency after the other.  16 sequences take 9 us, one 8.
template <bool VEC, bool FIRST>
__global__ __launch_bounds__(kEndThreads) void verify_pass_kernel(VerifyArgs a) {
  __shared__ VerifyShared sh;
  const bool rows = FIRST && a.all_rows;
  const int seq = rows ? blockIdx.y / a.max_query_len : blockIdx.y;
  const int node = rows ? blockIdx.y - seq * a.max_query_len : 0;
  Walk walk{node, 0, kTotal, -1, 0.0f, 0.0, 0.0};
  if (!FIRST) walk = a.walks[seq];
  const Sequence s = sequence_of(a, seq);
  const float pick_u = a.pick_u[seq];
  if (!FIRST && walk.phase == kDone) return;
  if (FIRST && node >= s.n) {
    if (node == 0 && blockIdx.x == 0) {  // no nodes at all
      begin_outputs(a, s, Node{});
      if (threadIdx.x == 0) a.walks[seq].phase = kDone;
    }
    return;
  }
  const int from = FIRST ? 0 : walk.node;
  Node mine;
  sum_segment<VEC>(a, sh, s, walk, blockIdx.x, from, mine);
  if (threadIdx.x == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums are there before the arrival
    // (the last of `of` to arrive)
    auto last_of = [&](int counter, int of) {
      unsigned* at = a.counters + (size_t)counter * a.apart;
      const bool last = __hip_atomic_fetch_add(at, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == static_cast<unsigned>(of);
      if (last) put(at, 0u);
      return last;
    };
    sh.last = rows ? last_of(gridDim.y / a.max_query_len + blockIdx.y, a.segments) && last_of(seq, s.n) : last_of(seq, a.segments);
  }
  __syncthreads();
  if (!sh.last) return;
  if (FIRST) begin_outputs(a, s, mine);
  walk.node = from;
  advance<VEC>(a, sh, s, walk, mine, pick_u);
  if (threadIdx.x == 0) a.walks[seq] = walk;
}

// The walks that are left, a workgroup each: 40 us a row of 128k logits (48 with two groups, 72 with one).
template <bool VEC>
__global__ __launch_bounds__(kGroups * kEndThreads) void verify_finish_kernel(VerifyArgs a) {
  __shared__ VerifyShared sh;
  Walk walk = a.walks[blockIdx.x];
  if (walk.phase == kDone) return;
  const Sequence s = sequence_of(a, blockIdx.x);
  while (walk.phase != kDone) {  // each round tries a child, goes to one, or ends the walk
    Node mine;
    for (int i = 0; i < a.segments; i += kGroups) sum_segment<VEC>(a, sh, s, walk, i + group_of(), walk.node, mine);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    advance<VEC>(a, sh, s, walk, mine, a.pick_u[blockIdx.x]);
    __syncthreads();
  }
}

}  // namespace

extern "C" {

int32_t fi_verify_drafts(fi_context* ctx, const float* d_logits, int32_t ld, int32_t vocab, const int32_t* d_tokens,
                         const int32_t* d_parents, const int32_t* d_cu_seqlens, int32_t num_seqs, int32_t max_query_len,
                         const float* d_temperature, const float* d_draft_probs, int32_t draft_ld, int32_t distinct,
                         const float* d_accept_u, const float* d_pick_u, int32_t max_path, int32_t* d_out_tokens,
                         int32_t* d_out_path, int32_t* d_out_count, float* d_out_prob) {
  FI_TRY(fi::enter(ctx));
  FI_REQUIRE(num_seqs >= 0 && max_query_len >= 0 && max_path >= 0, FI_ERR_INVALID_SHAPE, "fi_verify_drafts: negative sizes");
  FI_REQUIRE(vocab > 0 && ld >= vocab && (!d_draft_probs || draft_ld >= vocab), FI_ERR_INVALID_SHAPE,
             "fi_verify_drafts: requires non-empty rows (vocab > 0, ld >= vocab, draft_ld >= vocab)");
  FI_REQUIRE(vocab <= kMaxVocab, FI_ERR_UNSUPPORTED,
             "fi_verify_drafts: vocabularies of more than " + std::to_string(kMaxVocab) + " logits");
  FI_REQUIRE(max_query_len <= fi::kMaxTreeNodes, FI_ERR_UNSUPPORTED,
             "fi_verify_drafts: trees of more than " + std::to_string(fi::kMaxTreeNodes) + " nodes");
  FI_REQUIRE(max_path < fi::kMaxTreeNodes, FI_ERR_INVALID_SHAPE, "fi_verify_drafts: max_path is more than a tree can be deep");
  FI_REQUIRE(num_seqs <= 65535, FI_ERR_INVALID_SHAPE, "fi_verify_drafts: at most 65535 sequences per call");
  if (num_seqs == 0) return FI_OK;
  FI_REQUIRE(((d_logits && d_tokens && d_parents && d_accept_u) || max_query_len == 0) && d_cu_seqlens && d_temperature && d_pick_u &&
                 d_out_tokens && (d_out_path || max_path == 0) && d_out_count && d_out_prob,
             FI_ERR_INVALID_CONFIG, "fi_verify_drafts: null pointer");
  VerifyArgs a{};
  a.logits = d_logits;
  a.tokens = d_tokens;
  a.parents = d_parents;
  a.cu_seqlens = d_cu_seqlens;
  a.temperature = d_temperature;
  a.probs = d_draft_probs;
  a.accept_u = d_accept_u;
  a.pick_u = d_pick_u;
  a.out_tokens = d_out_tokens;
  a.out_path = d_out_path;
  a.out_count = d_out_count;
  a.out_prob = d_out_prob;
  a.faults = ctx->d_faults;
  a.ld = ld;
  a.ld_probs = draft_ld;
  a.vocab = vocab;
  a.distinct = distinct != 0;
  a.max_path = max_path;
  a.max_query_len = max_query_len;
  a.segments = (vocab + kSegment - 1) / kSegment;
  const int64_t rows = static_cast<int64_t>(num_seqs) * max_query_len;
  // Few rows are all summed in the first launch, so that a walk goes through accepted tokens without further ones: one
  // sequence of 8 rows of 152k logits 22 us, 38 with a launch a row; 24 sequences of 5 rows of 128k, drawn, 51 and 58; 32 of
  // them 62 and 64; 24 of 8 rows of 152k, given, 61 and 56, drawn 77 and 91; 64 of 5 rows of 128k 98 and 89.
  a.all_rows = max_path > 0 && max_query_len > 1 && rows <= 65535 && rows + num_seqs <= FI_MERGE_COUNTERS && rows * vocab <= kAllRows;
  // Arrivals at one line follow each other at 11 ns: counters a line each, as far as there are lines (64 sequences of five rows,
  // all rows summed: 63 us, 117 with the counters side by side).
  for (a.apart = 32; (num_seqs + (a.all_rows ? rows : 0)) * a.apart > FI_MERGE_COUNTERS;) a.apart /= 2;
  const size_t sums = static_cast<size_t>(a.all_rows ? rows : num_seqs) * a.segments * sizeof(RowSums);
  const size_t rests = static_cast<size_t>(num_seqs) * a.segments * sizeof(double);
  FI_TRY(fi::ensure_workspace(ctx, sums + rests + static_cast<size_t>(num_seqs) * sizeof(Walk)));
  a.sums = static_cast<RowSums*>(ctx->workspace);
  a.rests = reinterpret_cast<double*>(static_cast<char*>(ctx->workspace) + sums);
  a.walks = reinterpret_cast<Walk*>(static_cast<char*>(ctx->workspace) + sums + rests);
  a.counters = ctx->d_merge_counters;
  const bool vec = vocab % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(d_logits) % 16 == 0 &&
                   (!d_draft_probs || (draft_ld % 4 == 0 && reinterpret_cast<uintptr_t>(d_draft_probs) % 16 == 0));
  // The launches behind the first.  A walk visits depth + 1 rows at most; a node all of whose given children are
  // rejected costs a pass and ends the walk, so that it never needs more than that.  Each drawn child that is
  // rejected costs a pass; a walk has nodes - 1 children to try in all.
  const int depth = std::min(max_path, std::max(max_query_len - 1, 0));
  const int needed = a.all_rows ? (d_draft_probs ? max_query_len - 1 : 1)
                                : (d_draft_probs && depth > 0 ? max_query_len - 1 : depth);
  // Launches for four rejections, then one that takes what is left, a workgroup a walk: 16 trees of up to 32 nodes, drawn, 99 us
  // in the mean of twelve (112 with launches for two, 99 for six, 103 for eight), 64 of them 173 (198, 170, 172).  max_path may be a loose bound, and a launch that finds nothing to do costs
  // 1 to 3 us: rows behind the first kDepth are left to that as well.
  const int passes = std::min(needed, (a.all_rows ? 0 : std::min(depth, kDepth)) + kRejections);
  auto launch = [&](auto vec_rows) {
    constexpr bool VEC = decltype(vec_rows)::value;
    const unsigned segments = static_cast<unsigned>(a.segments);
    hipLaunchKernelGGL((verify_pass_kernel<VEC, true>), dim3(segments, static_cast<unsigned>(a.all_rows ? rows : num_seqs)),
                       dim3(kEndThreads), 0, ctx->stream, a);
    for (int i = 0; i < passes; ++i)
      hipLaunchKernelGGL((verify_pass_kernel<VEC, false>), dim3(segments, num_seqs), dim3(kEndThreads), 0, ctx->stream, a);
    if (passes < needed) hipLaunchKernelGGL((verify_finish_kernel<VEC>), dim3(num_seqs), dim3(kGroups * kEndThreads), 0, ctx->stream, a);
  };
  if (vec)
    launch(std::true_type{});
  else
    launch(std::false_type{});
  FI_CHECK_LAUNCH("verify_pass_kernel");
  return FI_OK;
}

}  // extern "C"
