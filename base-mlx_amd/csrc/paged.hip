// Appending a batch's packed rows to a paged KV cache (gfx950): per-head
// RMSNorm and rotary positions of queries and keys, queries to [heads, tokens,
// 128], keys and values to their sequences' pages.
//
//   y = x / sqrt(mean x^2 + eps) * w,
//   (y_i, y_{i+64}) -> (y_i cos a - y_{i+64} sin a, y_{i+64} cos a + y_i sin a),
//   a = p theta^(-i/64)
#include <math.h>

#include <algorithm>

#include "paged.h"

namespace bmx {

int check_paged(const char* what, const bmx_paged_kv* c, const bmx_batch* b, int n_heads, int head_dim) {
  if (!c || !b || !c->k || !c->v || !b->starts || !b->lens || !b->pages)
    return set_error(BMX_E_ARG, "%s: null pointer", what);
  if (head_dim != kPagedDim)
    return set_error(BMX_E_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", what, head_dim);
  if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return set_error(BMX_E_UNSUPPORTED, "%s: page_size=%d must be a power of two, 16 .. 4096", what, c->page_size);
  if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 1024 || n_heads <= 0 || n_heads > 65535 ||
      n_heads % c->n_kv_heads)
    return set_error(BMX_E_SHAPE, "%s: n_pages=%d, %d heads over %d kv heads", what, c->n_pages, n_heads,
                     c->n_kv_heads);
  if (b->n_seqs < 0 || b->n_seqs > kPagedMaxSeqs || b->max_pages <= 0 ||
      b->max_pages > kPagedMaxRows / c->page_size)
    return set_error(BMX_E_SHAPE, "%s: n_seqs=%d (0..%d), max_pages=%d (1..%d)", what, b->n_seqs, kPagedMaxSeqs,
                     b->max_pages, kPagedMaxRows / c->page_size);
  if (b->tokens < 0 || static_cast<int64_t>(b->tokens) * n_heads > (1 << 28) ||
      (b->tokens > 0 && (b->max_new < 1 || b->max_new > b->tokens)))
    return set_error(BMX_E_SHAPE, "%s: tokens=%d, max_new=%d", what, b->tokens, b->max_new);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(b->starts, 4) || !aligned(b->lens, 4) ||
      !aligned(b->pages, 4))
    return set_error(BMX_E_ALIGN, "%s: k and v must be 16-byte aligned, the batch's arrays 4-byte", what);
  return BMX_OK;
}

namespace {

struct AppendParams {
  const uint16_t* q;  // [T, Hq*128]
  const uint16_t* k;  // [T, Hkv*128]
  const uint16_t* v;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  uint16_t* q_out;  // [Hq, T, 128]
  bmx_paged_kv c;
  bmx_batch b;
  int Hq, shift;     // 2^shift = page_size
  float eps;
  double turns[64];  // theta^(-i/64) / 2 pi: turns per position
};

constexpr int kGridRow = 1 << 20;  // workgroups: a grid's row holds fewer than 2^32 threads, 2^24 tokens of this kernel

// A workgroup of 4 waves takes a token.  Its rows -- the q heads, the k heads,
// the v heads -- go 16 lanes to a row, lane li holding values 4 li .. + 3 and
// 64 + 4 li .. + 3, the two halves of four rotated pairs.  The sequence's search
// and the angles, in double, are a workgroup's once, not a row's.  Bound by memory:
// 8540 tokens of 32 + 2 x 8 heads 42 us, 210 MB at 5.0 TB/s (a large copy moves 4.9); one
// token 3.7 us, the latency of the starts, the table, the cosine and the row one
// after another.
__global__ void __launch_bounds__(256) qk_norm_rope_paged_kernel(const AppendParams p) {
  __shared__ __align__(16) float cs[2][64];
  const int t = blockIdx.y * kGridRow + blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int T = p.b.tokens, B = p.b.n_seqs, Hkv = p.c.n_kv_heads;
  if (t >= T) return;  // uniform, as every return up to the barrier
  // ---- the token's sequence: the last whose rows start at t or before.  64
  // samples of the starts, then the 64 (or fewer) from the last sample on ----
  const int step = (B + 63) >> 6;
  int seg = 0;
  if (step > 1) {
    const int at = lane * step;
    const uint64_t m = __ballot(at < B && p.b.starts[min(at, B - 1)] <= t);
    if (m == 0) return;
    seg = (__popcll(m) - 1) * step;
  }
  const int at = min(seg + lane, B - 1);
  const int s0 = p.b.starts[at], s1 = p.b.starts[at + 1], ln = p.b.lens[at];
  const uint64_t m = __ballot(seg + lane < B && s0 <= t);
  if (m == 0) return;
  const int own = __popcll(m) - 1, b = seg + own;
  const PagedSeq sq = paged_seq(__builtin_amdgcn_readlane(s0, own), __builtin_amdgcn_readlane(s1, own),
                                __builtin_amdgcn_readlane(ln, own), T);
  if (t >= sq.row0 + sq.tokens) return;  // past the last sequence
  const int pos = sq.pos + t - sq.row0;
  // its cache row (none: `page` -1)
  int page = -1;
  if (pos >= 0 && (pos >> p.shift) < p.b.max_pages) {
    page = p.b.pages[static_cast<int64_t>(b) * p.b.max_pages + (pos >> p.shift)];
    if (page >= p.c.n_pages) page = -1;
  }
  // ---- the rotation, once per workgroup: the angle in turns, reduced in
  // double (at position 2^24 an fp32 angle would be off by a radian) ----
  if (wave == 0) {
    const double a = static_cast<double>(pos) * p.turns[lane];
    float c, s;
    sincospif(2.0f * static_cast<float>(a - rint(a)), &s, &c);
    cs[0][lane] = c;
    cs[1][lane] = s;
  }
  __syncthreads();
  const int li = lane & 15, grp = threadIdx.x >> 4;
  const float4 c4 = *reinterpret_cast<const float4*>(&cs[0][4 * li]), s4 = *reinterpret_cast<const float4*>(&cs[1][4 * li]);
  const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
  const int rows = p.Hq + 2 * Hkv;
  for (int r = grp; r < rows; r += 16) {
    const bool is_q = r < p.Hq, is_v = r >= p.Hq + Hkv;
    const int h = is_q ? r : is_v ? r - p.Hq - Hkv : r - p.Hq;
    if (!is_q && page < 0) continue;
    const uint16_t* src = is_q ? p.q + (static_cast<int64_t>(t) * p.Hq + h) * 128
                               : (is_v ? p.v : p.k) + (static_cast<int64_t>(t) * Hkv + h) * 128;
    uint16_t* dst = is_q ? p.q_out + (static_cast<int64_t>(h) * T + t) * 128
                         : (is_v ? p.c.v : p.c.k) +
                               ((((static_cast<int64_t>(page) * Hkv + h) << p.shift) + (pos & ((1 << p.shift) - 1))) << 7);
    uint2 lo = *reinterpret_cast<const uint2*>(src + 4 * li), hi = *reinterpret_cast<const uint2*>(src + 64 + 4 * li);
    if (!is_v) {
      const uint16_t* nw = is_q ? p.q_norm : p.k_norm;
      const uint2 wl = *reinterpret_cast<const uint2*>(nw + 4 * li), wh = *reinterpret_cast<const uint2*>(nw + 64 + 4 * li);
      float a[4] = {bf2f(lo.x & 0xffffu), bf2f(lo.x >> 16), bf2f(lo.y & 0xffffu), bf2f(lo.y >> 16)};
      float b4[4] = {bf2f(hi.x & 0xffffu), bf2f(hi.x >> 16), bf2f(hi.y & 0xffffu), bf2f(hi.y >> 16)};
      const float wa[4] = {bf2f(wl.x & 0xffffu), bf2f(wl.x >> 16), bf2f(wl.y & 0xffffu), bf2f(wl.y >> 16)};
      const float wb[4] = {bf2f(wh.x & 0xffffu), bf2f(wh.x >> 16), bf2f(wh.y & 0xffffu), bf2f(wh.y >> 16)};
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; i++) ss += a[i] * a[i] + b4[i] * b4[i];
      ss = row16_sum(ss);
      const float inv = 1.0f / sqrtf(ss / 128.0f + p.eps);
      uint16_t o1[4], o2[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = a[i] * inv * wa[i], y = b4[i] * inv * wb[i];
        o1[i] = f2bf(x * c[i] - y * s[i]);
        o2[i] = f2bf(y * c[i] + x * s[i]);
      }
      lo = make_uint2(o1[0] | (static_cast<uint32_t>(o1[1]) << 16), o1[2] | (static_cast<uint32_t>(o1[3]) << 16));
      hi = make_uint2(o2[0] | (static_cast<uint32_t>(o2[1]) << 16), o2[2] | (static_cast<uint32_t>(o2[3]) << 16));
    }
    *reinterpret_cast<uint2*>(dst + 4 * li) = lo;
    *reinterpret_cast<uint2*>(dst + 64 + 4 * li) = hi;
  }
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" int bmx_qk_norm_rope_paged(const bmx_bf16* q, const bmx_bf16* k, const bmx_bf16* v, const bmx_bf16* q_norm,
                                      const bmx_bf16* k_norm, bmx_bf16* q_out, const bmx_paged_kv* cache,
                                      const bmx_batch* batch, int n_heads, int head_dim, float eps, float theta,
                                      void* stream) {
  if (int rc = check_paged("qk_norm_rope_paged", cache, batch, n_heads, head_dim)) return rc;
  if (!q || !k || !v || !q_norm || !k_norm || !q_out) return set_error(BMX_E_ARG, "qk_norm_rope_paged: null pointer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) ||
      !aligned(q_out, 16))
    return set_error(BMX_E_ALIGN, "qk_norm_rope_paged: pointers must be 16-byte aligned");
  const int T = batch->tokens;
  if (T == 0 || batch->n_seqs == 0) return BMX_OK;
  if (overlaps(span_of_pages(*cache, cache->k), {span_of_pages(*cache, cache->v)}))
    return set_error(BMX_E_ARG, "qk_norm_rope_paged: k and v of the cache overlap");
  const size_t qb = static_cast<size_t>(T) * n_heads * 256, kb = static_cast<size_t>(T) * cache->n_kv_heads * 256;
  const Span to{q_out, qb}, from[] = {{q, qb}, {k, kb}, {v, kb}, {q_norm, 256}, {k_norm, 256}};
  if (over_batch(to, *batch)) return set_error(BMX_E_ARG, "qk_norm_rope_paged: q_out overlaps the batch's arrays");
  if (over_cache(to, *cache)) return set_error(BMX_E_ARG, "qk_norm_rope_paged: q_out overlaps the cache");
  for (const Span& s : from) {
    if (overlaps(to, {s})) return set_error(BMX_E_ARG, "qk_norm_rope_paged: q_out overlaps an input");
    if (over_cache(s, *cache)) return set_error(BMX_E_ARG, "qk_norm_rope_paged: an input overlaps the cache");
  }
  for (const void* pages : {cache->k, cache->v})
    if (over_batch(span_of_pages(*cache, pages), *batch))
      return set_error(BMX_E_ARG, "qk_norm_rope_paged: the batch's arrays overlap the cache");
  AppendParams p{q, k, v, q_norm, k_norm, q_out, *cache, *batch, n_heads, log2_of(cache->page_size), eps, {}};
  // (64 pow calls are most of a small call's host time: a thread keeps the last)
  thread_local float last = NAN;  // (unequal to anything)
  thread_local double turns[64];
  if (theta != last) {
    for (int i = 0; i < 64; i++) turns[i] = pow(static_cast<double>(theta), -i / 64.0) / 6.283185307179586476925;
    last = theta;
  }
  for (int i = 0; i < 64; i++) p.turns[i] = turns[i];
  hipLaunchKernelGGL(qk_norm_rope_paged_kernel, dim3(std::min(T, kGridRow), (T + kGridRow - 1) / kGridRow), dim3(256), 0, as_stream(stream), p);
  return check_launch("qk_norm_rope_paged");
}
