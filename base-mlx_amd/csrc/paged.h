// The paged KV cache of a batch: argument checks and device lookups shared by
// the kernels that append to it and attend over it.
#pragma once

#include <initializer_list>

#include "bmx_device.h"

namespace bmx {

constexpr int kPagedDim = 128;       // head_dim
constexpr int kPagedMaxSeqs = 4096;  // (a wave finds a token's sequence in two loads of 64)
constexpr int kPagedMaxRows = 1 << 24;  // of a sequence

// Checks of the structs themselves; `what` names the entry point.
int check_paged(const char* what, const bmx_paged_kv* c, const bmx_batch* b, int n_heads, int head_dim);

// Some bytes of memory
struct Span {
  const void* at;
  size_t bytes;
};
// Whether `s` has a byte in common with any of the others
inline bool overlaps(const Span& s, std::initializer_list<Span> others) {
  const uintptr_t i = reinterpret_cast<uintptr_t>(s.at);
  for (const Span& o : others) {
    const uintptr_t j = reinterpret_cast<uintptr_t>(o.at);
    if (i < j + o.bytes && j < i + s.bytes) return true;
  }
  return false;
}
inline Span span_of_pages(const bmx_paged_kv& c, const void* at) {
  return {at, static_cast<size_t>(c.n_pages) * c.n_kv_heads * c.page_size * kPagedDim * sizeof(uint16_t)};
}
// Whether `s` lies over the cache, or over the batch's arrays
inline bool over_cache(const Span& s, const bmx_paged_kv& c) {
  return overlaps(s, {span_of_pages(c, c.k), span_of_pages(c, c.v)});
}
inline bool over_batch(const Span& s, const bmx_batch& b) {
  const size_t n = b.n_seqs;
  return overlaps(s, {{b.starts, (n + 1) * 4}, {b.lens, n * 4}, {b.pages, n * b.max_pages * 4}});
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
