// Trees of drafted tokens: what the kernels over them share.  Sequence b's tree is the rows
// [cu_seqlens[b], cu_seqlens[b + 1]) of the step, node i of it row cu_seqlens[b] + i, and node i's K/V row
// lies at position prefix + i of the sequence, prefix = context_lens[b] - nodes.
#pragma once

#include "fi_common.h"

namespace fi {

constexpr int kMaxTreeNodes = 1024;  // nodes of one tree (plan and verification keep a tree in LDS)

// The tree of a sequence: its first row, its nodes, and the cached positions before it (below 0 where
// context_lens is short; lengths below 0 count as 0, for the difference to stay in 32 bits).
struct TreeSpan {
  int first, nodes, prefix;
};

__device__ __forceinline__ TreeSpan tree_span(const int* cu_seqlens, const int* context_lens, int seq) {
  TreeSpan t;
  t.first = cu_seqlens[seq];
  t.nodes = max(cu_seqlens[seq + 1] - t.first, 0);
  t.prefix = (context_lens ? max(context_lens[seq], 0) : 0) - t.nodes;
  return t;
}

// The 64 bits [at, at + 64) of a mask row of `words` words.  Bits before the row (at below 0) are the
// prefix's, all set; bits behind it are not.
__device__ __forceinline__ uint64_t mask_window(const uint64_t* __restrict__ row, int words, int at) {
  if (at <= -64) return ~0ull;
  if (at <= 0) return at == 0 ? row[0] : (row[0] << -at) | ((1ull << -at) - 1);
  const int w = at >> 6, s = at & 63;
  uint64_t bits = w < words ? row[w] >> s : 0;
  if (s != 0 && w + 1 < words) bits |= row[w + 1] << (64 - s);
  return bits;
}

// Which of the 64 keys k0 .. k0 + 63 lie before kend, as bits.
__host__ __device__ inline uint64_t keys_before(int kend, int k0) {
  return kend - k0 >= 64 ? ~0ull : kend <= k0 ? 0 : (1ull << (kend - k0)) - 1;
}

}  // namespace fi
