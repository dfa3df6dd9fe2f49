// The paged KV cache of a batch: argument checks and device lookups shared by
// the kernels that append to it and attend over it.
#pragma once

#include "bmx_device.h"

namespace bmx {

constexpr int kPagedDim = 128;       // head_dim
constexpr int kPagedMaxSeqs = 4096;  // (a wave finds a token's sequence in two loads of 64)
constexpr int kPagedMaxRows = 1 << 24;  // of a sequence

// Checks of the structs themselves; `what` names the entry point.
int check_paged(const char* what, const bmx_paged_kv* c, const bmx_batch* b, int n_heads, int head_dim);

// Whether a bytes from x and b bytes from y have any in common
inline bool paged_overlap(const void* x, size_t a, const void* y, size_t b) {
  const uintptr_t i = reinterpret_cast<uintptr_t>(x), j = reinterpret_cast<uintptr_t>(y);
  return i < j + b && j < i + a;
}

inline int log2_of(int n) { return 31 - __builtin_clz(static_cast<unsigned>(n)); }

// A sequence as its entries of the batch's arrays say, brought into range:
// `tokens` packed rows from `row0` on, the first of them at position `pos`.
struct PagedSeq {
  int row0, tokens, pos;
};
__device__ __forceinline__ PagedSeq paged_seq(int s0, int s1, int len, int T) {
  s0 = min(max(s0, 0), T);
  s1 = min(max(s1, s0), T);
  // (positions below -T, and from the largest table's end on, are all the same: of no row)
  return PagedSeq{s0, s1 - s0, min(max(len, 0), kPagedMaxRows + T) - (s1 - s0)};
}

}  // namespace bmx
