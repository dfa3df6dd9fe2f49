// Eviction from the 4-bit KV cache by accumulated attention weight (gfx950).
//
// Selection, per kv head: the n = budget - sink - recent largest weights of
// rows [sink, length - recent), ties to the lower row, by radix selection over
// order-preserving integer keys in digits of 11, 11 and 10 bits; then every
// kept row's number in order.  Heads of up to 8192 rows: one workgroup each,
// the keys in registers.  Longer ones: up to 64 slices of a head and three
// launches.  The first leaves every slice's histogram of the first digit (the
// next adds them up, so nothing has to be cleared and the order is fixed); the
// second, knowing where that digit ends, each slice's keys of that digit, the
// ends of their range and how many lie above; the third finds the other digits among those few, in
// every slice again, and writes the numbers of its own rows.
// Compaction: rows kept[i] to rows i, kept[i] >= i; into another cache by the
// workgroup that found the numbers, where it has few, else and in place by a
// launch of its own.
#include <math.h>

#include <algorithm>

#include "kv4.h"

namespace bmx {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kCopies = 2;  // of a histogram in LDS: equal digits of a wave collide less
// Rows of a head that one workgroup selects from.  Above, slices are faster (8
// heads out of place, us: 12000 rows to 2000 16.8 against 19.8 with 16 rows a
// thread, 16000 to 4000 18.3 / 27.6).
constexpr int kOneWorkgroup = 8 * kThreads;
constexpr int kMaxSlices = 64;
constexpr int kShift[3] = {21, 10, 0};

// Unsigned keys in the order of the weights: -0 and +0 alike, every NaN
// above +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 -> +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct MoveParams {
  const uint32_t* src[6];  // k, v words; k, v scales and biases as one word per row
  uint32_t* dst[6];
  const float* w;
  float* w_out;
  int32_t* kept;
  int cap, cap_into, budget;
};

struct SelectParams {
  MoveParams m;
  uint32_t* hist;   // [heads, slices, kBins] of the first digit
  uint32_t* found;  // [heads, 2]: the first digit's place in the key, the count left
  uint32_t* count;  // [heads, slices, 4]: keys above the first digit, keys of it, the largest of these, of their complements
  uint32_t* cand;   // [heads, slices, slice_rows]: the keys of it
  int length, sink, recent;
  int slices, slice_rows;  // rows per slice, a multiple of 8
  int moves;               // rows are copied, too
};

typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

struct SelectLds {
  alignas(16) uint32_t hist[3][kCopies][kBins];
  alignas(16) uint32_t tmp[2][kWaves];
  uint32_t sel[3][2];
  uint32_t first[kMaxSlices + 1];  // candidates before each slice
};

// The sum over a wave's lanes up to this one, by DPP: within 16-lane rows
// (row_shr 1, 2, 4, 8), then the rows' ends across (row_bcast 15, 31).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);
  return dpp_add<0x143, 0xC>(v);
}
// Lane 63: the largest of a wave's v, the same way.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  v = dpp_max<0x111, 0xF>(v);
  v = dpp_max<0x112, 0xF>(v);
  v = dpp_max<0x114, 0xF>(v);
  v = dpp_max<0x118, 0xF>(v);
  v = dpp_max<0x142, 0xA>(v);
  return dpp_max<0x143, 0xC>(v);
}
// Sum of v over the workgroup's earlier threads; *total over all.  Calls take
// the buffers `turn` = 0, 1, 0, 1, ..: the barrier of the one between keeps a
// buffer from being written while it is read.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, SelectLds& s, int turn, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t x = wave_scan(v);
  if (lane == 63) s.tmp[turn][wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i += 4) {
    const u32x4_t t = *reinterpret_cast<const u32x4_t*>(&s.tmp[turn][i]);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      before += i + k < wave ? t[k] : 0u;
      all += t[k];
    }
  }
  *total = all;
  return before + x - v;
}

// This thread's E rows from `first` on: their keys; a row outside the middle
// (or outside the head) counts for nothing.
template <int E>
struct Rows {
  uint32_t key[E];
  uint32_t mid;  // bit e: row first + e takes part in the selection
};
template <int E>
__device__ __forceinline__ void load_rows(const SelectParams& p, const float* w, int first, Rows<E>& r) {
  typedef __attribute__((ext_vector_type(4))) float f4;
  typedef f4 __attribute__((aligned(4))) f4u;
  float v[E];
  if (first + E <= p.length) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<f4*>(&v[i]) = *reinterpret_cast<const f4u*>(w + first + i);
  } else {
#pragma unroll
    for (int i = 0; i < E; i++) v[i] = first + i < p.length ? w[first + i] : 0.0f;
  }
  r.mid = 0;
#pragma unroll
  for (int i = 0; i < E; i++) {
    r.key[i] = weight_key(v[i]);
    if (first + i >= p.sink && first + i < p.length - p.recent) r.mid |= 1u << i;
  }
}

__device__ __forceinline__ uint32_t digit_of(uint32_t key, int d) { return (key >> kShift[d]) & (d == 2 ? 1023u : 2047u); }

// Adds digit d of every key that agrees with `prefix` above it.
template <int E>
__device__ __forceinline__ void count_digits(const Rows<E>& r, int d, uint32_t prefix, SelectLds& s) {
  const int copy = threadIdx.x & (kCopies - 1);
  const uint32_t above = d == 0 ? 0u : ~0u << kShift[d - 1];
  uint32_t in = 0, same = 0;
  const uint32_t one = __builtin_amdgcn_readfirstlane(digit_of(r.key[0], d));
#pragma unroll
  for (int i = 0; i < E; i++) {
    if ((r.mid >> i & 1u) && (r.key[i] & above) == prefix) {
      in |= 1u << i;
      if (digit_of(r.key[i], d) == one) same |= 1u << i;
    }
  }
  if (__all(in == same)) {
    // equal digits all through the wave (a fresh cache's zeros): one addition
    const uint32_t n = wave_scan(static_cast<uint32_t>(__popc(in)));
    if ((threadIdx.x & 63) == 63 && n) atomicAdd(&s.hist[d][0][one], n);
    return;
  }
#pragma unroll
  for (int i = 0; i < E; i++)
    if (in >> i & 1u) atomicAdd(&s.hist[d][copy][digit_of(r.key[i], d)], 1u);
}

// The digit at which the `left` largest end, and how many of it are among
// them, from the counts of this thread's two bins kBins - 1 - 2 tid (c0) and
// the one below (c1).
__device__ __forceinline__ void find_digit(SelectLds& s, int d, uint32_t c0, uint32_t c1, uint32_t* digit,
                                           uint32_t* left) {
  const uint32_t b = kBins - 1 - 2 * threadIdx.x;
  uint32_t total;
  const uint32_t above = block_scan(c0 + c1, s, d & 1, &total);
  if (above < *left && *left <= above + c0) {
    s.sel[d][0] = b;
    s.sel[d][1] = *left - above;
  } else if (above + c0 < *left && *left <= above + c0 + c1) {
    s.sel[d][0] = b - 1;
    s.sel[d][1] = *left - above - c0;
  }
  __syncthreads();
  *digit = s.sel[d][0];
  *left = s.sel[d][1];
}
// ... with the histogram in LDS
__device__ __forceinline__ void find_own_digit(SelectLds& s, int d, uint32_t* T, uint32_t* left) {
  const int b = kBins - 2 - 2 * static_cast<int>(threadIdx.x);
  uint32_t c0 = 0, c1 = 0, digit;
#pragma unroll
  for (int c = 0; c < kCopies; c++) {
    const uint2 v = *reinterpret_cast<const uint2*>(&s.hist[d][c][b]);
    c0 += v.y;
    c1 += v.x;
  }
  find_digit(s, d, c0, c1, &digit, left);
  *T |= digit << kShift[d];
}

__device__ __forceinline__ void clear_hists(SelectLds& s) {
  u32x4_t* h = reinterpret_cast<u32x4_t*>(&s.hist[0][0][0]);
  for (int i = threadIdx.x; i < 3 * kCopies * kBins / 4; i += kThreads) h[i] = u32x4_t{0u, 0u, 0u, 0u};
}

// Numbers of the kept among this thread's E rows below `end`.  T: the smallest
// kept key, of which `left` may still be kept; `at`: rows kept before the
// workgroup's rows.  Both move on past them.
template <int E>
__device__ __forceinline__ void emit_rows(const Rows<E>& r, int first, int end, uint32_t T, bool none, uint32_t& left,
                                          uint32_t& at, int32_t* kept, SelectLds& s, int turn) {
  uint32_t keep = 0, eq = 0;
#pragma unroll
  for (int i = 0; i < E; i++) {
    if (first + i >= end) continue;
    const bool mid = r.mid >> i & 1u;
    if (!mid || (!none && r.key[i] > T)) keep |= 1u << i;
    if (mid && !none && r.key[i] == T) eq |= 1u << i;
  }
  uint32_t total;
  const uint32_t scan = block_scan(static_cast<uint32_t>(__popc(keep)) << 16 | static_cast<uint32_t>(__popc(eq)), s, turn, &total);
  uint32_t equal = scan & 0xffffu, pos = at + (scan >> 16) + min(equal, left);
#pragma unroll
  for (int i = 0; i < E; i++) {
    bool k = keep >> i & 1u;
    if (eq >> i & 1u) k = equal++ < left;
    if (k) kept[pos++] = first + i;
  }
  const uint32_t took = min(total & 0xffffu, left);
  at += (total >> 16) + took;
  left -= took;
}

// Rows kept[r0 .. r1) of head h to rows r0 .. r1 of the other cache, and this
// workgroup's share of the zeros behind the weights.
__device__ __forceinline__ void copy_rows(const MoveParams& m, int64_t h, int r0, int r1, int part, int parts) {
  constexpr int N = 8;
  const int32_t* kept = m.kept + h * m.budget;
  const u32x4_t* ws[2];
  u32x4_t* wd[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    ws[k] = reinterpret_cast<const u32x4_t*>(m.src[k] + h * m.cap * kKv4Words);
    wd[k] = reinterpret_cast<u32x4_t*>(m.dst[k] + h * m.cap_into * kKv4Words);
  }
  // one word of each small array and the weight per row; the first rows' are
  // read ahead of the pieces
  uint32_t v4[4] = {0u, 0u, 0u, 0u};
  float w1 = 0.0f;
  auto read_row = [&](int r) {
    const int64_t from = h * m.cap + kept[r];
#pragma unroll
    for (int k = 0; k < 4; k++) v4[k] = m.src[2 + k][from];
    w1 = m.w[from];
  };
  int r = r0 + static_cast<int>(threadIdx.x);
  if (r < r1) read_row(r);
  // 16-byte pieces: 4 of k, 4 of v per row
  for (int64_t i0 = static_cast<int64_t>(r0) * 8 + threadIdx.x; i0 < static_cast<int64_t>(r1) * 8; i0 += N * kThreads) {
    u32x4_t v[N];
    int32_t from[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int64_t i = i0 + k * kThreads;
      from[k] = i < static_cast<int64_t>(r1) * 8 ? kept[i >> 3] : -1;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int64_t i = i0 + k * kThreads;
      if (from[k] >= 0) v[k] = (i & 4 ? ws[1] : ws[0])[static_cast<int64_t>(from[k]) * 4 + (i & 3)];
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int64_t i = i0 + k * kThreads;
      if (from[k] >= 0) (i & 4 ? wd[1] : wd[0])[(i >> 3) * 4 + (i & 3)] = v[k];
    }
  }
  while (r < r1) {
    const int64_t to = h * m.cap_into + r;
#pragma unroll
    for (int k = 0; k < 4; k++) m.dst[2 + k][to] = v4[k];
    m.w_out[to] = w1;
    r += kThreads;
    if (r < r1) read_row(r);
  }
  for (int64_t i = m.budget + static_cast<int64_t>(part) * kThreads + threadIdx.x; i < m.cap_into;
       i += static_cast<int64_t>(parts) * kThreads)
    m.w_out[h * m.cap_into + i] = 0.0f;
}

// The rows of a head by several workgroups (see own_copy).
constexpr int kCopyRows = 256;
__global__ void __launch_bounds__(kThreads) kv4_copy_kernel(const MoveParams m) {
  const int r0 = blockIdx.y * kCopyRows;
  copy_rows(m, blockIdx.x, r0, min(m.budget, r0 + kCopyRows), blockIdx.y, gridDim.y);
}

// A head in one workgroup: up to kThreads * E rows, in registers.
template <int E>
__global__ void __launch_bounds__(kThreads) kv4_select_kernel(const SelectParams p) {
  __shared__ SelectLds s;
  const int h = blockIdx.x, first = threadIdx.x * E;
  Rows<E> r;
  load_rows<E>(p, p.m.w + static_cast<int64_t>(h) * p.m.cap, first, r);
  uint32_t left = static_cast<uint32_t>(p.m.budget - p.sink - p.recent), T = 0;
  const bool none = left == 0;  // uniform
  if (!none) {
    clear_hists(s);
    __syncthreads();
    for (int d = 0; d < 3; d++) {
      count_digits<E>(r, d, T, s);
      __syncthreads();
      find_own_digit(s, d, &T, &left);
    }
  }
  uint32_t at = 0;
  emit_rows<E>(r, first, p.length, T, none, left, at, p.m.kept + static_cast<int64_t>(h) * p.m.budget, s, 1);
  if (!p.moves) return;
  __syncthreads();  // (the numbers are written: the workgroup reads its own)
  copy_rows(p.m, h, 0, p.m.budget, 0, 1);
}

// Long heads, first launch: the histogram of a slice's first digit.
template <int E>
__global__ void __launch_bounds__(kThreads) kv4_hist_kernel(const SelectParams p) {
  __shared__ SelectLds s;
  const int h = blockIdx.x, slice = blockIdx.y, start = slice * p.slice_rows, end = min(p.length, start + p.slice_rows);
  const float* w = p.m.w + static_cast<int64_t>(h) * p.m.cap;
  for (int i = threadIdx.x; i < kCopies * kBins; i += kThreads) (&s.hist[0][0][0])[i] = 0;
  __syncthreads();
  for (int j0 = start; j0 < end; j0 += kThreads * E) {
    const int first = j0 + static_cast<int>(threadIdx.x) * E;
    Rows<E> r;
    load_rows<E>(p, w, first, r);
    if (first >= end) r.mid = 0;
    count_digits<E>(r, 0, 0u, s);
  }
  __syncthreads();
  uint32_t* out = p.hist + (static_cast<int64_t>(h) * p.slices + slice) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    uint32_t n = 0;
#pragma unroll
    for (int c = 0; c < kCopies; c++) n += s.hist[0][c][i];
    out[i] = n;
  }
}

// Second launch: where the first digit ends, and a slice's keys of it.
template <int E>
__global__ void __launch_bounds__(kThreads) kv4_pick_kernel(const SelectParams p) {
  __shared__ SelectLds s;
  const int h = blockIdx.x, slice = blockIdx.y, start = slice * p.slice_rows, end = min(p.length, start + p.slice_rows);
  const float* w = p.m.w + static_cast<int64_t>(h) * p.m.cap;
  uint32_t left = static_cast<uint32_t>(p.m.budget - p.sink - p.recent), digit;
  if (left == 0) return;  // uniform: nothing to select
  if (threadIdx.x == 0) s.sel[1][0] = s.sel[1][1] = 0;
  Rows<E> r;
  load_rows<E>(p, w, start + static_cast<int>(threadIdx.x) * E, r);
  const uint32_t* hist = p.hist + static_cast<int64_t>(h) * p.slices * kBins + (kBins - 2 - 2 * static_cast<int>(threadIdx.x));
  uint32_t c0 = 0, c1 = 0;
#pragma unroll 8
  for (int i = 0; i < p.slices; i++) {
    const uint2 v = *reinterpret_cast<const uint2*>(hist + i * kBins);
    c0 += v.y;
    c1 += v.x;
  }
  find_digit(s, 0, c0, c1, &digit, &left);
  if (slice == 0 && threadIdx.x == 0) {
    p.found[2 * h] = digit << kShift[0];
    p.found[2 * h + 1] = left;
  }
  const int64_t at = static_cast<int64_t>(h) * p.slices + slice;
  uint32_t* cand = p.cand + at * p.slice_rows;
  uint32_t above = 0, mine = 0;        // keys so far
  uint32_t largest = 0, smallest = 0;  // of this thread's, the smallest as its complement
  int turn = 1;
  for (int j0 = start; j0 < end; j0 += kThreads * E, turn ^= 1) {
    const int first = j0 + static_cast<int>(threadIdx.x) * E;
    if (j0 > start) load_rows<E>(p, w, first, r);
    if (first >= end) r.mid = 0;
    uint32_t over = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
      const uint32_t d = digit_of(r.key[i], 0);
      if ((r.mid >> i & 1u) && d > digit) over++;
      if ((r.mid >> i & 1u) && d == digit) eq |= 1u << i;
    }
    uint32_t total;
    uint32_t pos = mine + (block_scan(over << 16 | static_cast<uint32_t>(__popc(eq)), s, turn, &total) & 0xffffu);
#pragma unroll
    for (int i = 0; i < E; i++)
      if (eq >> i & 1u) {
        cand[pos++] = r.key[i];
        largest = max(largest, r.key[i]);
        smallest = max(smallest, ~r.key[i]);
      }
    above += total >> 16;
    mine += total & 0xffffu;
  }
  largest = wave_largest(largest);
  smallest = wave_largest(smallest);
  if ((threadIdx.x & 63) == 63) {
    atomicMax(&s.sel[1][0], largest);
    atomicMax(&s.sel[1][1], smallest);
  }
  __syncthreads();
  if (threadIdx.x == 0) *reinterpret_cast<u32x4_t*>(&p.count[4 * at]) = u32x4_t{above, mine, s.sel[1][0], s.sel[1][1]};
}

// Third launch: the smallest kept key, and the numbers of a slice's kept rows.
template <int E>
__global__ void __launch_bounds__(kThreads) kv4_emit_kernel(const SelectParams p) {
  __shared__ SelectLds s;
  const int h = blockIdx.x, slice = blockIdx.y, start = slice * p.slice_rows, end = min(p.length, start + p.slice_rows);
  const float* w = p.m.w + static_cast<int64_t>(h) * p.m.cap;
  Rows<E> r;
  load_rows<E>(p, w, start + static_cast<int>(threadIdx.x) * E, r);
  const bool none = p.m.budget - p.sink - p.recent == 0;
  uint32_t T = 0, left = 0;
  // rows kept in the slices before: of the ends, above T, and equal to it
  uint32_t at = static_cast<uint32_t>(min(start, p.sink) + max(0, start - (p.length - p.recent)));
  if (!none) {
    T = p.found[2 * h];
    left = p.found[2 * h + 1];
    const u32x4_t* count = reinterpret_cast<const u32x4_t*>(p.count) + static_cast<int64_t>(h) * p.slices;
    const uint32_t* cand = p.cand + static_cast<int64_t>(h) * p.slices * p.slice_rows;
    if (threadIdx.x < 64) {
      const int i = threadIdx.x;
      const u32x4_t c = i < p.slices ? count[i] : u32x4_t{0u, 0u, 0u, 0u};
      const uint32_t n = c.y, scan = wave_scan(n);
      s.first[i] = scan - n;
      if (i == 63) s.first[64] = scan;
      const uint32_t over = wave_scan(i < slice ? c.x : 0u);
      const uint32_t largest = wave_largest(c.z), smallest = ~wave_largest(c.w);
      if (i == 63) {
        s.sel[0][0] = over;
        s.sel[0][1] = largest;
        s.sel[1][1] = smallest;
      }
    }
    clear_hists(s);
    __syncthreads();
    at += s.sel[0][0];
    const uint32_t all = s.first[kMaxSlices];
    uint32_t equal = s.first[slice];  // keys T in the slices before
    if (s.sel[0][1] == s.sel[1][1]) {  // all alike (a fresh cache's zeros): nothing left to find
      T = s.sel[0][1];
    } else {
      // every candidate of the head, 4 per thread at a time: f(key, slice, or -1
      // where there is none).  The first 4096 stay in registers.
      auto fetch = [&](uint32_t g0, uint32_t (&key)[4], int (&from)[4]) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t g = g0 + k * kThreads;
          from[k] = -1;
          key[k] = 0;
          if (g < all) {
            int lo = 0, hi = p.slices - 1;  // the last slice that starts at or before g
            while (lo < hi) {
              const int mid = (lo + hi + 1) >> 1;
              if (s.first[mid] <= g) lo = mid;
              else hi = mid - 1;
            }
            from[k] = lo;
            key[k] = cand[static_cast<int64_t>(lo) * p.slice_rows + (g - s.first[lo])];
          }
        }
      };
      uint32_t held[4];
      int held_from[4];
      fetch(threadIdx.x, held, held_from);
      auto each = [&](auto f) {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (static_cast<uint32_t>(k) * kThreads < all) f(held[k], held_from[k]);
        for (uint32_t g0 = 4 * kThreads + threadIdx.x; g0 - threadIdx.x < all; g0 += 4 * kThreads) {
          uint32_t key[4];
          int from[4];
          fetch(g0, key, from);
#pragma unroll
          for (int k = 0; k < 4; k++) f(key[k], from[k]);
        }
      };
      for (int d = 1; d < 3; d++) {
        const uint32_t prefix = T;
        each([&](uint32_t key, int from) {
          Rows<1> one;
          one.key[0] = key;
          one.mid = from >= 0;
          count_digits<1>(one, d, prefix, s);
        });
        __syncthreads();
        find_own_digit(s, d, &T, &left);
      }
      uint32_t above = 0, total;
      equal = 0;
      each([&](uint32_t key, int from) {
        above += from >= 0 && from < slice && key > T;
        equal += from >= 0 && from < slice && key == T;
      });
      block_scan(above, s, 1, &total);
      at += total;
      block_scan(equal, s, 0, &equal);
    }
    const uint32_t took = min(equal, left);
    at += took;
    left -= took;
  }
  const uint32_t at0 = at;
  int turn = 1;
  for (int j0 = start; j0 < end; j0 += kThreads * E, turn ^= 1) {
    const int first = j0 + static_cast<int>(threadIdx.x) * E;
    if (j0 > start) load_rows<E>(p, w, first, r);
    emit_rows<E>(r, first, end, T, none, left, at, p.m.kept + static_cast<int64_t>(h) * p.m.budget, s, turn);
  }
  if (!p.moves) return;
  __syncthreads();  // (the numbers are written: the workgroup reads its own)
  copy_rows(p.m, h, static_cast<int>(at0), static_cast<int>(at), slice, p.slices);
}

// Items kept[i] to items i, `per` apart.  A block of 8 items per thread is
// read, and after a barrier written: the items that later blocks read,
// kept[i] >= i, are not among those written until then.
template <class T>
__device__ __forceinline__ void move_rows(const T* src, T* dst, const int32_t* kept, int n, int64_t per) {
  constexpr int N = 8;
  for (int64_t i0 = threadIdx.x; i0 - threadIdx.x < n; i0 += N * kThreads) {
    T v[N];
    int32_t from[N];
#pragma unroll
    for (int k = 0; k < N; k++) from[k] = i0 + k * kThreads < n ? kept[i0 + k * kThreads] : -1;
#pragma unroll
    for (int k = 0; k < N; k++)
      if (from[k] >= 0) v[k] = src[from[k] * per];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++)
      if (from[k] >= 0) dst[(i0 + k * kThreads) * per] = v[k];
  }
}

// In place: a workgroup takes one 16-byte column of all the rows of a head
// (so up to 8192 rows are one block), or an array of one word per row.
__global__ void __launch_bounds__(kThreads) kv4_move_kernel(const MoveParams p) {
  const int64_t h = blockIdx.x;
  const int32_t* kept = p.kept + h * p.budget;
  const int y = blockIdx.y;
  if (y < 8) {
    move_rows(reinterpret_cast<const u32x4_t*>(p.src[y >> 2] + h * p.cap * kKv4Words) + (y & 3),
              reinterpret_cast<u32x4_t*>(p.dst[y >> 2] + h * p.cap_into * kKv4Words) + (y & 3), kept, p.budget, 4);
  } else if (y < 12) {
    move_rows(p.src[y - 6] + h * p.cap, p.dst[y - 6] + h * p.cap_into, kept, p.budget, 1);
  } else {
    float* out = p.w_out + h * p.cap_into;
    move_rows(p.w + h * p.cap, out, kept, p.budget, 1);
    // (every weight has been read)
    for (int i = p.budget + threadIdx.x; i < p.cap_into; i += kThreads) out[i] = 0.0f;
  }
}

bool same_pointers(const bmx_kv4& a, const bmx_kv4& b) {
  return a.k == b.k && a.k_scales == b.k_scales && a.k_biases == b.k_biases && a.v == b.v &&
         a.v_scales == b.v_scales && a.v_biases == b.v_biases;
}

// Whether any array of one cache (its weights among them) reaches into one of the other
bool caches_overlap(const bmx_kv4& a, const float* aw, const bmx_kv4& b, const float* bw) {
  const void* x[7] = {a.k, a.v, aw, a.k_scales, a.k_biases, a.v_scales, a.v_biases};
  const void* y[7] = {b.k, b.v, bw, b.k_scales, b.k_biases, b.v_scales, b.v_biases};
  const size_t rows_a = static_cast<size_t>(a.n_kv_heads) * a.capacity;
  const size_t rows_b = static_cast<size_t>(b.n_kv_heads) * b.capacity;
  auto bytes = [](int i, size_t rows) { return rows * (i < 2 ? kKv4Words * 4 : 4); };
  for (int i = 0; i < 7; i++)
    for (int j = 0; j < 7; j++)
      if (kv4_overlap(x[i], bytes(i, rows_a), y[j], bytes(j, rows_b))) return true;
  return false;
}

// Slices of a head (0: one workgroup holds the head), the rows of each and how
// many a thread takes at a time.  4096 rows a slice while that is no more
// workgroups than CUs, else 8192 and up (out of place, us, 4096 / 8192: 8
// heads of 20001 rows to 4000 17.9 / 21.7, of 131001 to 4096 31.5 / 32.9; but
// 32 heads 63 / 46).
int select_slices(int heads, int length, int* rows, int* per_thread) {
  if (length <= kOneWorkgroup) return 0;
  auto slices = [&](int e) { return (length + kThreads * e - 1) / (kThreads * e); };
  *per_thread = slices(4) <= kMaxSlices && static_cast<int64_t>(heads) * slices(4) <= 256 ? 4 : 8;
  const int n = std::min(kMaxSlices, slices(*per_thread));
  *rows = ((length + n - 1) / n + 7) / 8 * 8;
  return (length + *rows - 1) / *rows;
}
// Whether the kept rows are copied by a launch of its own, not by the
// workgroups that find them: where one of these has many of them, so that the
// card gains the 2 us that another launch costs the host.  Out of place, us,
// own launch / not: one workgroup a head, 8 heads of 4352 rows to 512 10.7 /
// 10.4, to 1024 10.8 / 12.1, to 1536 10.8 / 13.6, to 4000 11.4 / 21.3; slices,
// 16000 to 1000 16.6 / 15.7, to 4000 17.0 / 18.3, to 12000 20.5 / 27.5, 131001
// to 4096 22.9 / 21.3.  The first and the last rows are all in one slice.
bool own_copy(int slices, int budget, int end) {
  return slices == 0 ? budget > 1536 : end > 1024 || budget > 768 * slices;
}
// Words of a head's workspace, as many as any shorter head's
size_t select_words(int length) {
  const size_t slices = std::min(kMaxSlices, (length + 4 * kThreads - 1) / (4 * kThreads));
  return slices * (kBins + 4 + 8) + length + 2;
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_kv4_evict_workspace_bytes(int n_kv_heads, int length) {
  if (n_kv_heads <= 0 || length <= 0 || length > kKv4MaxCapacity) return 0;
  return length > kOneWorkgroup ? n_kv_heads * select_words(length) * sizeof(uint32_t) : 0;
}

extern "C" int bmx_kv4_evict(const bmx_kv4* cache, const float* weights, const bmx_kv4* into, float* weights_into,
                             int32_t* kept, int length, int budget, int sink, int recent, int head_dim,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_kv4("kv4_evict", cache, head_dim)) return rc;
  if (int rc = check_kv4("kv4_evict: into", into, head_dim)) return rc;
  if (!weights || !weights_into || !kept) return set_error(BMX_E_ARG, "kv4_evict: null pointer");
  if (!aligned(weights, 16) || !aligned(weights_into, 16) || !aligned(kept, 16) || !aligned(workspace, 16))
    return set_error(BMX_E_ALIGN, "kv4_evict: weights, kept and workspace must be 16-byte aligned");
  if (into->n_kv_heads != cache->n_kv_heads)
    return set_error(BMX_E_SHAPE, "kv4_evict: %d kv heads into %d", cache->n_kv_heads, into->n_kv_heads);
  if (length > cache->capacity || budget > into->capacity)
    return set_error(BMX_E_KV_CAPACITY, "kv4_evict: length %d of capacity %d, budget %d of capacity %d", length,
                     cache->capacity, budget, into->capacity);
  if (budget < 1 || budget > length || sink < 0 || recent < 0 || static_cast<int64_t>(sink) + recent > budget)
    return set_error(BMX_E_SHAPE, "kv4_evict: length=%d budget=%d sink=%d recent=%d", length, budget, sink, recent);
  const bool in_place = same_pointers(*cache, *into);
  if (in_place != (weights == weights_into) || (in_place && into->capacity != cache->capacity))
    return set_error(BMX_E_ARG, "kv4_evict: cache and weights must both be in place, or neither");
  if (!in_place && caches_overlap(*cache, weights, *into, weights_into))
    return set_error(BMX_E_ARG, "kv4_evict: into overlaps the cache");
  const size_t need = bmx_kv4_evict_workspace_bytes(cache->n_kv_heads, length);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(BMX_E_ARG, "kv4_evict: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  const hipStream_t st = as_stream(stream);
  const int heads = cache->n_kv_heads;
  SelectParams s{};
  const bmx_kv4* c[2] = {cache, into};
  for (int i = 0; i < 2; i++) {
    uint32_t* a[6] = {c[i]->k,
                      c[i]->v,
                      reinterpret_cast<uint32_t*>(c[i]->k_scales),
                      reinterpret_cast<uint32_t*>(c[i]->k_biases),
                      reinterpret_cast<uint32_t*>(c[i]->v_scales),
                      reinterpret_cast<uint32_t*>(c[i]->v_biases)};
    for (int k = 0; k < 6; k++) {
      if (i) s.m.dst[k] = a[k];
      else s.m.src[k] = a[k];
    }
  }
  s.m.w = weights;
  s.m.w_out = weights_into;
  s.m.kept = kept;
  s.m.cap = cache->capacity;
  s.m.cap_into = into->capacity;
  s.m.budget = budget;
  s.length = length;
  s.sink = sink;
  s.recent = recent;
  int per_thread = 0;
  s.slices = select_slices(heads, length, &s.slice_rows, &per_thread);
  s.hist = static_cast<uint32_t*>(workspace);
  s.count = s.hist + static_cast<size_t>(heads) * s.slices * kBins;
  s.cand = s.count + static_cast<size_t>(heads) * s.slices * 4;
  s.found = s.cand + static_cast<size_t>(heads) * s.slices * s.slice_rows;
  const bool copies = !in_place && own_copy(s.slices, budget, std::max(sink, recent));
  s.moves = !in_place && !copies;
  if (s.slices == 0) {
    if (length <= 4 * kThreads) hipLaunchKernelGGL(kv4_select_kernel<4>, dim3(heads), dim3(kThreads), 0, st, s);
    else hipLaunchKernelGGL(kv4_select_kernel<8>, dim3(heads), dim3(kThreads), 0, st, s);
  } else {
    const dim3 grid(heads, s.slices), block(kThreads);
    if (per_thread == 4) {
      hipLaunchKernelGGL(kv4_hist_kernel<4>, grid, block, 0, st, s);
      hipLaunchKernelGGL(kv4_pick_kernel<4>, grid, block, 0, st, s);
      hipLaunchKernelGGL(kv4_emit_kernel<4>, grid, block, 0, st, s);
    } else {
      hipLaunchKernelGGL(kv4_hist_kernel<8>, grid, block, 0, st, s);
      hipLaunchKernelGGL(kv4_pick_kernel<8>, grid, block, 0, st, s);
      hipLaunchKernelGGL(kv4_emit_kernel<8>, grid, block, 0, st, s);
    }
  }
  if (int rc = check_launch("kv4_evict select")) return rc;
  if (copies) {
    hipLaunchKernelGGL(kv4_copy_kernel, dim3(heads, (budget + kCopyRows - 1) / kCopyRows), dim3(kThreads), 0, st, s.m);
    return check_launch("kv4_evict copy");
  }
  if (!in_place) return BMX_OK;
  hipLaunchKernelGGL(kv4_move_kernel, dim3(heads, 13), dim3(kThreads), 0, st, s.m);
  return check_launch("kv4_evict move");
}
