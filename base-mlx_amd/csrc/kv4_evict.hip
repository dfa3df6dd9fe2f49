// Eviction from the 4-bit KV cache by accumulated attention weight (gfx950).
//
// Selection, per kv head: the n = budget - sink - recent largest weights of
// rows [sink, length - recent) by radix selection over order-preserving
// integer keys, ties to the lower row; then every kept row's number in
// order.  Compaction: rows kept[i] to rows i, with kept[i] >= i.
#include <math.h>

#include "kv4.h"

namespace bmx {
namespace {

constexpr int kThreads = 1024;

// Unsigned keys in the order of the weights: -0 and +0 alike, every NaN
// above +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 -> +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of v over the workgroup and the total; `tmp` holds
// one word per wave.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* tmp, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int i = 0; i < kThreads / 64; i++) {
    if (i < wave) before += tmp[i];
    all += tmp[i];
  }
  *total = all;
  return before + x - v;
}

struct SelectParams {
  const float* weights;
  int32_t* kept;
  int cap, length, budget, sink, recent;
};

__global__ void __launch_bounds__(kThreads) kv4_select_kernel(const SelectParams p) {
  __shared__ uint32_t hist[256], tmp[kThreads / 64], sel[2];
  const int h = blockIdx.x, tid = threadIdx.x;
  const float* w = p.weights + static_cast<int64_t>(h) * p.cap;
  const int lo = p.sink, hi = p.length - p.recent;
  // the n largest of [lo, hi): key prefix by key prefix
  uint32_t prefix = 0, left = static_cast<uint32_t>(p.budget - p.sink - p.recent);
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int j = lo + tid; j < hi; j += kThreads) {
      const uint32_t k = weight_key(w[j]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int b = 255;
      for (; b > 0 && above + hist[b] < left; b--) above += hist[b];
      sel[0] = static_cast<uint32_t>(b);
      sel[1] = left - above;
    }
    __syncthreads();
    prefix |= sel[0] << shift;
    left = sel[1];
    __syncthreads();
  }
  // keys above `prefix` are kept, and the first `left` of those equal to it
  int32_t* kept = p.kept + static_cast<int64_t>(h) * p.budget;
  uint32_t at = 0, equal = 0;
  for (int j0 = 0; j0 < p.length; j0 += kThreads) {
    const int j = j0 + tid;
    const bool mid = j >= lo && j < hi;
    const uint32_t k = mid ? weight_key(w[j]) : 0u;
    const bool eq = mid && k == prefix;
    uint32_t n = 0;
    const uint32_t rank = equal + block_scan(eq, tmp, &n);
    equal += n;
    const bool keep = j < p.length && (!mid || k > prefix || (eq && rank < left));
    const uint32_t pos = at + block_scan(keep, tmp, &n);
    at += n;
    if (keep) kept[pos] = j;
  }
}

struct MoveParams {
  const uint32_t* src[6];  // k, v words; k, v scales and biases as one word per row
  uint32_t* dst[6];
  const float* w;
  float* w_out;
  const int32_t* kept;
  int cap, cap_into, budget;
};

// One workgroup per (kv head, array).  A block of rows is read, and after a
// barrier written: later rows are read from kept[i] >= i, which no earlier
// block has written, so the move may be in place.
template <int WORDS>
__device__ __forceinline__ void move_rows(const uint32_t* src, uint32_t* dst, const int32_t* kept, int budget) {
  for (int i0 = 0; i0 < budget * WORDS; i0 += kThreads) {
    const int i = i0 + threadIdx.x, r = i / WORDS;
    uint32_t v = 0;
    if (r < budget) v = src[static_cast<int64_t>(kept[r]) * WORDS + i % WORDS];
    __syncthreads();
    if (r < budget) dst[i] = v;
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) kv4_move_kernel(const MoveParams p) {
  const int64_t h = blockIdx.x;
  const int32_t* kept = p.kept + h * p.budget;
  if (blockIdx.y < 2) {
    move_rows<kKv4Words>(p.src[blockIdx.y] + h * p.cap * kKv4Words, p.dst[blockIdx.y] + h * p.cap_into * kKv4Words, kept,
                         p.budget);
  } else if (blockIdx.y < 6) {
    move_rows<1>(p.src[blockIdx.y] + h * p.cap, p.dst[blockIdx.y] + h * p.cap_into, kept, p.budget);
  } else {
    float* out = p.w_out + h * p.cap_into;
    move_rows<1>(reinterpret_cast<const uint32_t*>(p.w) + h * p.cap, reinterpret_cast<uint32_t*>(out), kept, p.budget);
    for (int i = p.budget + threadIdx.x; i < p.cap_into; i += kThreads) out[i] = 0.0f;
  }
}

bool same_pointers(const bmx_kv4& a, const bmx_kv4& b) {
  return a.k == b.k && a.k_scales == b.k_scales && a.k_biases == b.k_biases && a.v == b.v &&
         a.v_scales == b.v_scales && a.v_biases == b.v_biases;
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" int bmx_kv4_evict(const bmx_kv4* cache, const float* weights, const bmx_kv4* into, float* weights_into,
                             int32_t* kept, int length, int budget, int sink, int recent, int head_dim,
                             void* stream) {
  if (int rc = check_kv4("kv4_evict", cache, head_dim)) return rc;
  if (int rc = check_kv4("kv4_evict: into", into, head_dim)) return rc;
  if (!weights || !weights_into || !kept) return set_error(BMX_E_ARG, "kv4_evict: null pointer");
  if (!aligned(weights, 16) || !aligned(weights_into, 16) || !aligned(kept, 16))
    return set_error(BMX_E_ALIGN, "kv4_evict: weights and kept must be 16-byte aligned");
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
  const SelectParams s{weights, kept, cache->capacity, length, budget, sink, recent};
  hipLaunchKernelGGL(kv4_select_kernel, dim3(cache->n_kv_heads), dim3(kThreads), 0, as_stream(stream), s);
  if (int rc = check_launch("kv4_evict select")) return rc;
  MoveParams m{};
  const bmx_kv4* c[2] = {cache, into};
  for (int i = 0; i < 2; i++) {
    uint32_t* a[6] = {c[i]->k,
                      c[i]->v,
                      reinterpret_cast<uint32_t*>(c[i]->k_scales),
                      reinterpret_cast<uint32_t*>(c[i]->k_biases),
                      reinterpret_cast<uint32_t*>(c[i]->v_scales),
                      reinterpret_cast<uint32_t*>(c[i]->v_biases)};
    for (int k = 0; k < 6; k++) {
      if (i) m.dst[k] = a[k];
      else m.src[k] = a[k];
    }
  }
  m.w = weights;
  m.w_out = weights_into;
  m.kept = kept;
  m.cap = cache->capacity;
  m.cap_into = into->capacity;
  m.budget = budget;
  hipLaunchKernelGGL(kv4_move_kernel, dim3(cache->n_kv_heads, 7), dim3(kThreads), 0, as_stream(stream), m);
  return check_launch("kv4_evict move");
}
