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
// max(p - a q, 0) with a number a, and each rejection that a further child follows costs one pass over the
// two rows.  (A rejected child's rho is 0 from then on: it was below c q.  So taking it out of q as well
// changes nothing.)  The token at the end is the first index at which the running sum of rho passes u Z.
//
// Tokens are compared with u at borders that lie 1e-7 and less apart in a flat row, so what decides is in 64
// bits: exponentials and sums to 1e-14.  The walk itself takes sums of f32 exponentials, with a bound on
// their error, and repeats a node in 64 bits where a comparison falls within it (one in 30000).
//
// verify_walk_kernel walks, one workgroup a sequence: it reads the rows of the path's nodes that have
// children.  verify_end_kernel draws the last token, one workgroup a (segment of a row, sequence): the
// segments' sums, then the last workgroup of a sequence to finish finds the segment and the token in it.
// The numbers a that the walk took rho by are off as its sums are, so the segments also sum what rho changes by
// with a: f(a) = sum(max(w - a q, 0)) = f(a') - (a - a') sum(q where w > a' q) but for the elements whose w / q lies
// between a' and a, 1e-7 apart, each of which is off by 1e-7 of a q.  From the exact sum of w the exact a's follow one
// by one.
#include <algorithm>

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
  struct EndState* ends;     // [B]
  struct SegmentSums* sums;  // [B, segments]
  unsigned* counters;        // [B], zero between launches
  uint32_t* faults;
  int64_t ld, ld_probs;
  int vocab, distinct, max_path, max_query_len, segments;
};

constexpr int kMaxSteps = 4;  // values of a that the end follows; past them the walk's are of 64 bits

// The values of a at a node (times the sum of the weights w): a_1 = sum(w), a_(i + 1) = a_i + f(a_i) / room_(i + 1),
// one each time a drawn token was rejected; only the last where they are exact.
struct Offs {
  int steps, exact;
  double off[kMaxSteps], room[kMaxSteps];
};

// Where a sequence's walk ended.
struct EndState {
  int node;   // -1: nothing to draw
  int count;  // tokens accepted
  int tried;  // its children were tried and rejected
  float ref;  // the reference point of the row's weights
  Offs offs;
};

// A row's weights are 2^(k (l - ref)): k = log2(e) / temperature, l the logit.
struct Weights {
  double k, ref;
};

constexpr double kLog2E = 1.4426950408889634;
constexpr float kMinTemperature = 1.1920929e-7f;  // as sampling has it (f32::EPSILON)

__device__ __forceinline__ double row_scale(float temperature) {
  return kLog2E / static_cast<double>(fmaxf(temperature, kMinTemperature));
}

// 2^x for x in [-1100, 1000]: 2^n times the series of e^(f ln 2), |f| <= 1/2; its twelfth term is 6e-15.
__device__ __forceinline__ double exp2_64(double x) {
  constexpr double L = 0.69314718055994530942;
  const double n = __builtin_rint(x), f = (x - n) * L;
  double s = 1.0 / 39916800;
  s = __builtin_fma(s, f, 1.0 / 3628800);
  s = __builtin_fma(s, f, 1.0 / 362880);
  s = __builtin_fma(s, f, 1.0 / 40320);
  s = __builtin_fma(s, f, 1.0 / 5040);
  s = __builtin_fma(s, f, 1.0 / 720);
  s = __builtin_fma(s, f, 1.0 / 120);
  s = __builtin_fma(s, f, 1.0 / 24);
  s = __builtin_fma(s, f, 1.0 / 6);
  s = __builtin_fma(s, f, 0.5);
  s = __builtin_fma(s, f, 1.0);
  s = __builtin_fma(s, f, 1.0);
  return __builtin_ldexp(s, static_cast<int>(n));
}

// A logit's weight; one of -inf (and, where k is 0, NaN from it) weighs nothing.
__device__ __forceinline__ double weight(double l, const Weights& w) {
  return exp2_64(__builtin_fmin(__builtin_fmax((l - w.ref) * w.k, -1100.0), 1000.0));
}

// What weights by `from` are multiplied with to be weights by `to`.
__device__ __forceinline__ double change_of_ref(double k, float from, float to) {
  return exp2_64(__builtin_fmin(__builtin_fmax((static_cast<double>(from) - to) * k, -1100.0), 1000.0));
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.0f; }

__device__ __forceinline__ bool unusable(float l) { return !(l <= 3.402823466e38f); }  // NaN or +inf

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
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

// ---------------------------------------------------------------- the walk

constexpr int kWalkThreads = 512;
constexpr int kWalkWaves = kWalkThreads / 64;
constexpr int kAhead = 4;  // quads of a row that a lane has in flight

// What a wave finds in its part of a row.
struct PartStats {
  double sum;  // of the weights by the point k * ref
  float ref, top;
  int first;  // the index of the first logit of value top
  int bad;    // a logit that is NaN or +inf, or (fast sums) nothing that can be relied on
};

struct WalkShared {
  int tokens[fi::kMaxTreeNodes];
  int parents[fi::kMaxTreeNodes];
  float accept[fi::kMaxTreeNodes];
  uint64_t kids[fi::kMaxTreeNodes / 64];  // the node's children, as bits
  PartStats parts[kWalkWaves];
  double rest[kWalkWaves];
};

// The fast sums' error, relative to the sum.  A term's exponent t = (l - ref) k is off by three roundings, its value
// by ln 2 * 3 * 2^-24 |t| + 2^-23 of itself.  The maximum lies within 40 of the reference point, so that |t| <= 80 (1.0e-5)
// for all but terms below 2^-40 of the largest, a million of which are worth 1e-6.  A lane adds 16 terms in f32
// (2^-20), the rest in f64.  Together below 2^-16.
constexpr double kFastError = 1.52587890625e-5;

// One pass of a wave over row[begin, end): maximum, its first index and, unless GREEDY, the weights' sum by a reference
// point from the first quads of the part.  That serves as long as the maximum lies within 900 (fast: 40) binary
// orders of it; a part where it does not is summed again by its maximum.
template <bool VEC, bool FAST, bool GREEDY>
__device__ __forceinline__ PartStats part_stats(const float* __restrict__ row, int begin, int end, double k, int lane) {
  PartStats r{0.0, 0.0f, -INFINITY, 0x7fffffff, 0};
  const float k32 = static_cast<float>(k);
  for (int round = 0; round < 2; ++round) {
    float ref = r.top, top = -INFINITY;
    int first = 0x7fffffff;
    double sum = 0.0;
    bool bad = false;
    for (int at0 = begin + 4 * lane; at0 - 4 * lane < end; at0 += 256 * kAhead) {  // wave-uniform
      float4 x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) x[j] = quad_at<VEC>(row, at0 + 256 * j < end ? at0 + 256 * j : 0x7ffffff0, end, -INFINITY);
      if (!GREEDY && round == 0 && at0 - 4 * lane == begin) {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) m = fmaxf(m, fmaxf(fmaxf(x[j].x, x[j].y), fmaxf(x[j].z, x[j].w)));
        ref = fi::wave_max(m);
        if (!(fabsf(ref) <= 3.402823466e38f)) ref = 0.0f;
      }
      const Weights w{k, ref};
      float quick = 0.0f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float v[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (v[e] > top) {
            top = v[e];
            first = at0 + 256 * j + e;
          }
          if constexpr (!GREEDY) {
            if constexpr (FAST) {
              quick += __builtin_amdgcn_exp2f((v[e] - ref) * k32);
            } else {
              bad |= unusable(v[e]);
              sum += weight(v[e], w);
            }
          }
        }
      }
      if constexpr (FAST && !GREEDY) sum += quick;
    }
    const float wave_top = fi::wave_max(top);
    int at = top == wave_top ? first : 0x7fffffff;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, 64));
    r.top = wave_top;
    r.first = at;
    r.ref = ref;
    if constexpr (GREEDY) return r;
    r.sum = wave_sum64(sum);
    const bool over = wave_top != -INFINITY && __builtin_fabs((static_cast<double>(wave_top) - ref) * k) > (FAST ? 40.0 : 900.0);
    r.bad = __builtin_amdgcn_ballot_w64(bad) != 0 || !(r.sum <= 1.7976931348623157e308);
    if (!over || unusable(wave_top)) return r;
  }
  return r;
}

// sum of max(weight - off * q, 0) over a wave's part of the rows
template <bool VEC, bool FAST>
__device__ __forceinline__ double part_rest(const float* __restrict__ row, const float* __restrict__ probs, int begin, int end,
                                            const Weights& w, double off, int lane) {
  double sum = 0.0;
  const float k32 = static_cast<float>(w.k), off32 = static_cast<float>(off), ref32 = static_cast<float>(w.ref);
  for (int at0 = begin + 4 * lane; at0 - 4 * lane < end; at0 += 256 * kAhead) {
    float4 x[kAhead], q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int at = at0 + 256 * j < end ? at0 + 256 * j : 0x7ffffff0;
      x[j] = quad_at<VEC>(row, at, end, -INFINITY);
      q[j] = quad_at<VEC>(probs, at, end, 0.0f);
    }
    float quick = 0.0f;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float v[4] = {x[j].x, x[j].y, x[j].z, x[j].w}, p[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (FAST)
          quick += fmaxf(__builtin_amdgcn_exp2f((v[e] - ref32) * k32) - off32 * p[e], 0.0f);
        else
          sum += __builtin_fmax(weight(v[e], w) - off * p[e], 0.0);
      }
    }
    if constexpr (FAST) sum += quick;
  }
  return wave_sum64(sum);
}

// What a node's trial gives.
struct Trial {
  int child;    // the accepted child, or -1
  int unsure;   // a comparison within the fast sums' error, or a row that they do not serve
  int failed;   // no distribution: a logit that is NaN or +inf, or none that is finite
  float ref;
  Offs offs;
};

// The first child (a bit of sh.kids) behind node j, or -1.
__device__ __forceinline__ int next_child(const WalkShared& sh, int n, int j) {
  ++j;
  for (int word = j >> 6; word < (n + 63) >> 6; ++word) {
    const uint64_t bits = sh.kids[word] & (word == j >> 6 ? ~0ull << (j & 63) : ~0ull);
    if (bits != 0) return 64 * word + __builtin_ctzll(bits);
  }
  return -1;
}

// Tries the children of `node`, sh.kids, of which there is one.  Every thread of the workgroup takes the same way.
template <bool VEC, bool FAST>
__device__ __forceinline__ Trial try_node(const VerifyArgs& a, WalkShared& sh, const fi::TreeSpan& t, int n, int node,
                                          float temperature) {
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int part = ((a.vocab + kWalkWaves - 1) / kWalkWaves + 255) & ~255;
  const int begin = min(w * part, a.vocab), end = min(begin + part, a.vocab);
  const float* row = a.logits + (int64_t)(t.first + node) * a.ld;
  const bool greedy = temperature <= 0.0f;
  const double k = row_scale(temperature);
  const PartStats mine = greedy ? part_stats<VEC, true, true>(row, begin, end, k, lane)
                                : part_stats<VEC, FAST, false>(row, begin, end, k, lane);
  __syncthreads();  // the last trial's readers are done
  if (lane == 0) sh.parts[w] = mine;
  __syncthreads();
  Trial r{};
  r.child = -1;
  float top = -INFINITY;
  int first = 0x7fffffff, bad = 0;
  for (int i = 0; i < kWalkWaves; ++i) {
    const PartStats p = sh.parts[i];
    if (p.top > top) {
      top = p.top;
      first = p.first;
    }
    bad |= p.bad;
  }
  if (greedy) {
    r.child = next_child(sh, n, node);
    while (r.child >= 0 && (sh.tokens[r.child] != first || first >= a.vocab)) r.child = next_child(sh, n, r.child);
    return r;
  }
  r.unsure = FAST && bad;
  r.failed = !FAST && (bad || top == -INFINITY);
  if (bad || top == -INFINITY) {
    r.unsure = FAST;
    return r;
  }
  const Weights by{k, top};
  r.ref = top;
  double total = 0.0;  // 1 at least: the largest logit's
  for (int i = 0; i < kWalkWaves; ++i) {
    const PartStats p = sh.parts[i];
    if (p.sum > 0.0) total += p.sum * change_of_ref(k, p.ref, top);
  }
  const float* probs = a.probs ? a.probs + (int64_t)(t.first + node) * a.ld_probs : nullptr;
  double rest = total, rest_error = FAST ? kFastError * total : 0.0;  // Z
  double off = 0.0, off_error = 0.0, taken = 0.0;
  int next = next_child(sh, n, node);
  while (next >= 0) {
    const int j = next, x = sh.tokens[j];
    next = next_child(sh, n, j);
    if (x < 0 || x >= a.vocab || !(taken < 1.0)) continue;
    const double mass = weight(row[x], by), u = sh.accept[j];
    if (!probs) {
      // an earlier child of the same token has been taken out
      bool out = false;
      for (int i = next_child(sh, n, node); i < j; i = next_child(sh, n, i)) out |= sh.tokens[i] == x;
      const double left = out ? 0.0 : mass;
      if (FAST && __builtin_fabs(u * rest - left) <= u * rest_error + 1e-9 * left) r.unsure = 1;
      if (u * rest < left) {
        r.child = j;
        break;
      }
      rest -= left;
    } else {
      const double q = probs[x], c = rest / (1.0 - taken), c_error = rest_error / (1.0 - taken);
      const double left = __builtin_fmax(mass - off * q, 0.0);
      if (FAST && __builtin_fabs(u * c * q - left) <= (u * c_error + off_error) * q + 1e-9 * (left + off * q)) r.unsure = 1;
      if (u * c * q < left) {
        r.child = j;
        break;
      }
      off += c;
      off_error += c_error;
      if constexpr (FAST) {
        // the end takes it from here; more steps than it follows: the node once more, in 64 bits
        if (r.offs.steps == kMaxSteps) r.unsure = 1;
#pragma unroll
        for (int i = 0; i < kMaxSteps; ++i)
          if (i == r.offs.steps) {
            r.offs.off[i] = off;
            r.offs.room[i] = 1.0 - taken;
          }
        ++r.offs.steps;
      } else {
        r.offs.steps = r.offs.exact = 1;
        r.offs.off[0] = off;
      }
      if (a.distinct) taken += q;
      if (next >= 0 && !r.unsure) {
        const double wave = part_rest<VEC, FAST>(row, probs, begin, end, by, off, lane);
        __syncthreads();
        if (lane == 0) sh.rest[w] = wave;
        __syncthreads();
        rest = 0.0;
        for (int i = 0; i < kWalkWaves; ++i) rest += sh.rest[i];
        rest_error = FAST ? kFastError * total + off_error + 1e-6 * off : 0.0;
      }
    }
    if (r.unsure) return r;
  }
  return r;
}

template <bool VEC>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyArgs a) {
  __shared__ WalkShared sh;
  const int seq = blockIdx.x, tid = threadIdx.x;
  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, nullptr, seq);
  const int n = min(t.nodes, a.max_query_len);
  if (tid == 0 && t.nodes > a.max_query_len) atomicOr(a.faults, FI_FAULT_QUERY_RANGE);
  for (int i = tid; i < n; i += kWalkThreads) {
    const int p = a.parents[t.first + i], x = a.tokens[t.first + i];
    if (p < -1 || p >= i) atomicOr(a.faults, FI_FAULT_TREE_RANGE);
    if (i > 0 && (x < 0 || x >= a.vocab)) atomicOr(a.faults, FI_FAULT_TOKEN_RANGE);
    sh.parents[i] = p >= i ? -1 : p;
    sh.tokens[i] = x;
    sh.accept[i] = a.accept_u[t.first + i];
  }
  int* tokens = a.out_tokens + (size_t)seq * (a.max_path + 1);
  int* path = a.out_path + (size_t)seq * a.max_path;
  __syncthreads();
  const float temperature = a.temperature[seq];
  EndState end{};
  end.node = n > 0 ? 0 : -1;
  while (end.node >= 0 && end.count < a.max_path) {
    for (int i = tid; i < (n + 63) / 64 * 64; i += kWalkThreads) {  // whole waves
      const uint64_t bits = __builtin_amdgcn_ballot_w64(i < n && sh.parents[i] == end.node);
      if ((tid & 63) == 0) sh.kids[i >> 6] = bits;
    }
    __syncthreads();
    if (next_child(sh, n, end.node) < 0) break;
    Trial r = try_node<VEC, true>(a, sh, t, n, end.node, temperature);
    if (r.unsure) r = try_node<VEC, false>(a, sh, t, n, end.node, temperature);
    if (r.failed) {
      if (tid == 0) atomicOr(a.faults, FI_FAULT_SAMPLE_NONFINITE);
      end.node = -1;
    } else if (r.child < 0) {
      end.tried = 1;
      end.offs = r.offs;
      end.ref = r.ref;
      break;
    } else {
      if (tid == 0) {
        path[end.count] = r.child;
        tokens[end.count] = sh.tokens[r.child];
      }
      end.node = r.child;
      ++end.count;
    }
    __syncthreads();  // sh.kids is read no more
  }
  for (int i = end.count + tid; i < a.max_path; i += kWalkThreads) path[i] = -1;
  for (int i = end.count + tid; i <= a.max_path; i += kWalkThreads) tokens[i] = -1;
  if (tid == 0) {
    a.out_count[seq] = end.count;
    a.out_prob[seq] = 0.0f;
    a.ends[seq] = end;
  }
}

// ---------------------------------------------------------------- the token at the end

constexpr int kEndThreads = 256;
constexpr int kEndElems = 16;                          // consecutive elements a thread
constexpr int kSegment = kEndThreads * kEndElems;      // 4096
constexpr int kMaxSegments = 256;                      // a thread each when they are joined
constexpr int kMaxVocab = kSegment * kMaxSegments;     // 1048576

struct SegmentSums {
  double sum;              // of the weights
  double rest[kMaxSteps];  // of what is left of them, at each a
  double part[kMaxSteps];  // of q where something is left
  float top;               // the reference point of the weights (0 where it is not finite)
  int first, bad, pad;
};

struct EndShared {
  uint32_t out[kSegment / 32];  // tokens given and rejected
  double scan[kEndThreads / 64];
  float tops[kEndThreads / 64];
  int firsts[kEndThreads / 64], bads[kEndThreads / 64];
  double total;
  int last, pick, segment;
};

// The 16 elements of a thread.
template <bool VEC>
__device__ __forceinline__ void end_load(const float* __restrict__ row, int begin, int vocab, float pad, float (&v)[kEndElems]) {
#pragma unroll
  for (int j = 0; j < kEndElems / 4; ++j) {
    const float4 x = quad_at<VEC>(row, begin + 4 * j, vocab, pad);
    v[4 * j] = x.x;
    v[4 * j + 1] = x.y;
    v[4 * j + 2] = x.z;
    v[4 * j + 3] = x.w;
  }
}

template <bool VEC>
__global__ __launch_bounds__(kEndThreads) void verify_end_kernel(VerifyArgs a) {
  __shared__ EndShared sh;
  const int seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const EndState end = a.ends[seq];
  if (end.node < 0) return;  // every segment of the sequence
  const fi::TreeSpan t = fi::tree_span(a.cu_seqlens, nullptr, seq);
  const int n = min(t.nodes, a.max_query_len);
  const float* row = a.logits + (int64_t)(t.first + end.node) * a.ld;
  const float* probs = a.probs ? a.probs + (int64_t)(t.first + end.node) * a.ld_probs : nullptr;
  const float temperature = a.temperature[seq];
  const bool greedy = temperature <= 0.0f;
  const double k = greedy ? kLog2E : row_scale(temperature);
  const bool less = end.tried && !greedy && probs && end.offs.steps > 0;  // max(w - a q, 0)
  const bool without = end.tried && !greedy && !probs;                    // w, but for the tokens tried
  const int steps = less ? end.offs.steps : 1;

  // marks the segment's tokens that were tried, and loads it
  auto open = [&](int segment, float (&v)[kEndElems], float (&q)[kEndElems]) {
    const int begin = segment * kSegment;
    end_load<VEC>(row, begin + tid * kEndElems, a.vocab, -INFINITY, v);
    if (less) end_load<VEC>(probs, begin + tid * kEndElems, a.vocab, 0.0f, q);
    if (without) {  // workgroup-uniform
      for (int i = tid; i < kSegment / 32; i += kEndThreads) sh.out[i] = 0;
      __syncthreads();
      for (int j = end.node + 1 + tid; j < n; j += kEndThreads) {
        const int x = a.tokens[t.first + j];
        if (a.parents[t.first + j] == end.node && x >= begin && x < min(begin + kSegment, a.vocab))
          atomicOr(&sh.out[(x - begin) >> 5], 1u << ((x - begin) & 31));
      }
      __syncthreads();
    }
  };

  auto tried = [&](int e) { return ((sh.out[e >> 5] >> (e & 31)) & 1) != 0; };

  float v[kEndElems], q[kEndElems];
  const int segment = blockIdx.x;
  open(segment, v, q);
  float top = -INFINITY;
  int first = 0x7fffffff;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    bad |= unusable(v[e]);
    if (v[e] > top) {
      top = v[e];
      first = segment * kSegment + tid * kEndElems + e;
    }
  }
  {
    const float wave_top = fi::wave_max(top);
    int at = top == wave_top ? first : 0x7fffffff;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, 64));
    const bool any = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) {
      sh.tops[w] = wave_top;
      sh.firsts[w] = at;
      sh.bads[w] = any;
    }
  }
  __syncthreads();
  top = -INFINITY;
  bad = false;
  for (int i = 0; i < kEndThreads / 64; ++i) {
    if (sh.tops[i] > top) {
      top = sh.tops[i];
      first = sh.firsts[i];
    }
    bad |= sh.bads[i] != 0;
  }
  const Weights by{k, finite_or_zero(top)};
  double sum = 0.0, rest[kMaxSteps] = {}, in_part[kMaxSteps] = {}, off[kMaxSteps];
  {
    const double change = less ? change_of_ref(k, end.ref, finite_or_zero(top)) : 0.0;
#pragma unroll
    for (int i = 0; i < kMaxSteps; ++i) off[i] = less && i < steps ? end.offs.off[i] * change : 0.0;
  }
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    const double x = weight(v[e], by);
    sum += x;
    if (less) {
#pragma unroll
      for (int i = 0; i < kMaxSteps; ++i)
        if (i < steps) {
          const double left = x - off[i] * q[e];
          rest[i] += __builtin_fmax(left, 0.0);
          in_part[i] += left > 0.0 ? static_cast<double>(q[e]) : 0.0;
        }
    } else {
      rest[0] += without && tried(tid * kEndElems + e) ? 0.0 : x;
    }
  }
  // the workgroup's sum of x, in thread 0
  auto gather = [&](double x) {
    x = wave_sum64(x);
    __syncthreads();  // the last use of sh.scan is over
    if (lane == 0) sh.scan[w] = x;
    __syncthreads();
    double all = 0.0;
    for (int i = 0; i < kEndThreads / 64; ++i) all += sh.scan[i];
    return all;
  };
  sum = gather(sum);
#pragma unroll
  for (int i = 0; i < kMaxSteps; ++i)
    if (i < steps) {
      rest[i] = gather(rest[i]);
      if (less) in_part[i] = gather(in_part[i]);
    }
  if (tid == 0) {
    SegmentSums* to = a.sums + (size_t)seq * a.segments + segment;
    // read by another workgroup of this launch: device-coherent stores, complete before the arrival
    __hip_atomic_store(&to->sum, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < kMaxSteps; ++i)
      if (i < steps) {
        __hip_atomic_store(&to->rest[i], rest[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&to->part[i], in_part[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    __hip_atomic_store(&to->top, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&to->first, first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&to->bad, bad ? 1 : 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    const unsigned arrived = __hip_atomic_fetch_add(&a.counters[seq], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    sh.last = arrived == static_cast<unsigned>(a.segments);
    if (sh.last) __hip_atomic_store(&a.counters[seq], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sh.last) return;

  // ---- the last workgroup of the sequence: a thread a segment ----
  SegmentSums mine{};
  mine.top = -INFINITY;
  mine.first = 0x7fffffff;
  if (tid < a.segments) {
    SegmentSums* from = a.sums + (size_t)seq * a.segments + tid;
    mine.sum = __hip_atomic_load(&from->sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < kMaxSteps; ++i)
      if (i < steps) {
        mine.rest[i] = __hip_atomic_load(&from->rest[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        mine.part[i] = __hip_atomic_load(&from->part[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    mine.top = __hip_atomic_load(&from->top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    mine.first = __hip_atomic_load(&from->first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    mine.bad = __hip_atomic_load(&from->bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  {
    const float wave_top = fi::wave_max(mine.top);
    int at = mine.top == wave_top ? mine.first : 0x7fffffff;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, 64));
    const bool any = __builtin_amdgcn_ballot_w64(mine.bad != 0) != 0;
    if (lane == 0) {
      sh.tops[w] = wave_top;
      sh.firsts[w] = at;
      sh.bads[w] = any;
    }
  }
  __syncthreads();
  top = -INFINITY;
  bad = false;
  for (int i = 0; i < kEndThreads / 64; ++i) {
    if (sh.tops[i] > top) {
      top = sh.tops[i];
      first = sh.firsts[i];
    }
    bad |= sh.bads[i] != 0;
  }
  int* token = a.out_tokens + (size_t)seq * (a.max_path + 1) + end.count;
  if ((bad && !greedy) || top == -INFINITY) {
    if (tid == 0) atomicOr(a.faults, FI_FAULT_SAMPLE_NONFINITE);
    return;  // the token stays -1
  }
  // the segments' sums by one reference point
  const float ref = finite_or_zero(top);
  const double scale = tid < a.segments ? change_of_ref(k, finite_or_zero(mine.top), ref) : 0.0;
  // running sums of `x` over the threads, in order; the total in sh.total
  auto running = [&](double x) {
    double run = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const double y = __shfl_up(run, m, 64);
      if (lane >= m) run += y;
    }
    __syncthreads();  // the last use of sh.scan is over
    if (lane == 63) sh.scan[w] = run;
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int i = 0; i < kEndThreads / 64; ++i) {
      if (i < w) before += sh.scan[i];
      all += sh.scan[i];
    }
    if (tid == 0) sh.total = all;
    return before + run;
  };
  if (greedy) {
    running(mine.sum * scale);
    if (tid == 0) {
      *token = first;
      a.out_prob[seq] = bad ? NAN : static_cast<float>(1.0 / sh.total);
    }
    return;
  }
  // the exact a, step by step, and what is left of the segment's weights there
  double exact = 0.0, left_here = mine.rest[0] * scale;
  if (less) {
    const double change = change_of_ref(k, end.ref, ref);
    if (end.offs.exact) {
      exact = end.offs.off[0] * change;
    } else {
      const double all = gather(mine.sum * scale);
#pragma unroll
      for (int i = 0; i < kMaxSteps; ++i)
        if (i < steps) {
          exact = i == 0 ? all : exact + gather(left_here) / end.offs.room[i];
          left_here = __builtin_fmax(mine.rest[i] * scale - (exact - end.offs.off[i] * change) * mine.part[i], 0.0);
        }
    }
  }
  // nothing left (p = a q but for rounding): the draw is from the distribution itself
  double run = running(left_here);
  __syncthreads();
  const bool whole = !(sh.total > 0.0);
  if (whole) run = running(mine.sum * scale);
  if (tid == 0) {
    sh.segment = a.segments;
    sh.pick = 0x7fffffff;
  }
  __syncthreads();
  const double total = sh.total, target = static_cast<double>(a.pick_u[seq]) * total;
  const double share = whole ? mine.sum * scale : left_here;
  if (tid < a.segments && share > 0.0 && run > target) atomicMin(&sh.segment, tid);
  __syncthreads();
  int chosen = sh.segment;
  __syncthreads();             // every wave has read it
  if (chosen >= a.segments) {  // u of 1 and more (or NaN): the last segment that has anything
    if (tid == 0) sh.segment = -1;
    __syncthreads();
    if (tid < a.segments && share > 0.0) atomicMax(&sh.segment, tid);
    __syncthreads();
    chosen = sh.segment;
  }
  __shared__ double s_before;
  __shared__ float s_top;
  if (tid == chosen) {
    s_before = run - share;
    s_top = mine.top;
  }
  __syncthreads();
  // ---- the token in the segment ----
  open(chosen, v, q);
  const Weights in{k, finite_or_zero(s_top)};
  const double to_ref = change_of_ref(k, finite_or_zero(s_top), ref);
  const double off_in = less ? exact * change_of_ref(k, ref, finite_or_zero(s_top)) : 0.0;
  double left[kEndElems], here = 0.0;
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    const double x = weight(v[e], in);
    left[e] = to_ref * (whole  ? x
                        : less ? __builtin_fmax(x - off_in * q[e], 0.0)
                               : (without && tried(tid * kEndElems + e) ? 0.0 : x));
    here += left[e];
  }
  const double before = s_before;
  double at = before + running(here) - here;
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for (int e = 0; e < kEndElems; ++e) {
    at += left[e];
    if (left[e] > 0.0) {
      last = e;
      if (at > target && found == 0x7fffffff) found = e;
    }
  }
  if (found != 0x7fffffff) atomicMin(&sh.pick, tid * kEndElems + found);
  __syncthreads();
  if (sh.pick == 0x7fffffff) {  // the sums' roundings, or u of 1 and more: the last that has anything
    if (tid == 0) sh.segment = -1;
    __syncthreads();
    if (last >= 0) atomicMax(&sh.segment, tid * kEndElems + last);
    __syncthreads();
    if (tid == 0) sh.pick = sh.segment;
    __syncthreads();
  }
  const int pick = sh.pick;
  if (pick >= 0 && pick / kEndElems == tid) {
    double mass = 0.0;
#pragma unroll
    for (int e = 0; e < kEndElems; ++e)
      if (e == pick % kEndElems) mass = left[e];
    *token = chosen * kSegment + pick;
    a.out_prob[seq] = static_cast<float>(mass / total);
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
  FI_REQUIRE(d_logits && d_tokens && d_parents && d_cu_seqlens && d_temperature && d_accept_u && d_pick_u && d_out_tokens &&
                 (d_out_path || max_path == 0) && d_out_count && d_out_prob,
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
  const size_t sums = static_cast<size_t>(num_seqs) * a.segments * sizeof(SegmentSums);
  FI_TRY(fi::ensure_workspace(ctx, sums + static_cast<size_t>(num_seqs) * sizeof(EndState)));
  a.sums = static_cast<SegmentSums*>(ctx->workspace);
  a.ends = reinterpret_cast<EndState*>(static_cast<char*>(ctx->workspace) + sums);
  a.counters = ctx->d_merge_counters;
  const bool vec = vocab % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(d_logits) % 16 == 0 &&
                   (!d_draft_probs || (draft_ld % 4 == 0 && reinterpret_cast<uintptr_t>(d_draft_probs) % 16 == 0));
  const dim3 ends(static_cast<unsigned>(a.segments), static_cast<unsigned>(num_seqs));
  if (vec) {
    hipLaunchKernelGGL((verify_walk_kernel<true>), dim3(num_seqs), dim3(kWalkThreads), 0, ctx->stream, a);
    FI_CHECK_LAUNCH("verify_walk_kernel");
    hipLaunchKernelGGL((verify_end_kernel<true>), ends, dim3(kEndThreads), 0, ctx->stream, a);
  } else {
    hipLaunchKernelGGL((verify_walk_kernel<false>), dim3(num_seqs), dim3(kWalkThreads), 0, ctx->stream, a);
    FI_CHECK_LAUNCH("verify_walk_kernel");
    hipLaunchKernelGGL((verify_end_kernel<false>), ends, dim3(kEndThreads), 0, ctx->stream, a);
  }
  FI_CHECK_LAUNCH("verify_end_kernel");
  return FI_OK;
}

}  // extern "C"
