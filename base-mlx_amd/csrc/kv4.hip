// Rows of the 4-bit KV cache: quantizing write, write fused with QK-norm and
// RoPE, and read-back (gfx950).
//
// Write, per row and group of 64 values (fp32):
//   b = min x, s = bf16((max x - min x) / 15), n = min(rne((x - b) / s), 15)
// b is one of the bf16 inputs, so storing it rounds nothing; the nibbles are
// taken against the rounded s, which is what a reader multiplies by.
#include <math.h>

#include "kv4.h"

namespace bmx {

int check_kv4(const char* what, const bmx_kv4* c, int head_dim) {
  if (!c || !c->k || !c->k_scales || !c->k_biases || !c->v || !c->v_scales || !c->v_biases)
    return set_error(BMX_E_ARG, "%s: null pointer", what);
  if (c->bits != 4 || c->group_size != 64)
    return set_error(BMX_E_UNSUPPORTED, "%s: only bits=4, group_size=64 (got %d, %d)", what, c->bits, c->group_size);
  if (head_dim != kKv4Dim)
    return set_error(BMX_E_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", what, head_dim);
  if (c->n_kv_heads <= 0 || c->n_kv_heads > 65535 || c->capacity <= 0 || c->capacity > kKv4MaxCapacity)
    return set_error(BMX_E_SHAPE, "%s: n_kv_heads=%d (1..65535), capacity=%d (1..%d)", what, c->n_kv_heads,
                     c->capacity, kKv4MaxCapacity);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scales, 16) || !aligned(c->k_biases, 16) ||
      !aligned(c->v_scales, 16) || !aligned(c->v_biases, 16))
    return set_error(BMX_E_ALIGN, "%s: cache pointers must be 16-byte aligned", what);
  return BMX_OK;
}

int check_kv4_rows(const char* what, const bmx_kv4* c, int M, int offset) {
  if (M < 0) return set_error(BMX_E_SHAPE, "%s: M=%d", what, M);
  if (offset < 0 || static_cast<int64_t>(offset) + M > c->capacity)
    return set_error(BMX_E_KV_CAPACITY, "%s: rows %d .. %lld, capacity %d", what, offset,
                     static_cast<long long>(offset) + M - 1, c->capacity);
  return BMX_OK;
}

namespace {

constexpr int kMaxPosition = 1 << 24;  // the largest up to which every position is an fp32 number

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
template <int CTRL>
__device__ __forceinline__ u16x2_t dpp_u16x2(u16x2_t v) {
  return __builtin_bit_cast(u16x2_t, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

struct Kv4Tensor {
  const uint16_t* x;  // bf16 rows (write: in, read: out)
  int64_t head_stride, row_stride;
  uint32_t* w;
  uint32_t* s;  // the row's two scales as one word
  uint32_t* b;
};

struct Kv4RowsParams {
  Kv4Tensor t[2];  // k, v
  int M, cap, offset;
};

// 16 lanes per row, 8 values (one word) per lane: lanes 0-7 hold group 0,
// lanes 8-15 group 1.  blockIdx.y: the kv head, blockIdx.z: k or v (and so no
// division by M: 15.4 us with one, 8191 rows of 8 heads).
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4RowsParams p) {
  const int m = blockIdx.x * 16 + (threadIdx.x >> 4), li = threadIdx.x & 15;
  if (m >= p.M) return;
  const Kv4Tensor& t = p.t[blockIdx.z];
  const int64_t h = blockIdx.y;
  const uint4 d = *reinterpret_cast<const uint4*>(t.x + h * t.head_stride + m * t.row_stride + 8 * li);
  const uint32_t v[4] = {d.x, d.y, d.z, d.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = bf2f(v[i] & 0xffffu);
    x[2 * i + 1] = bf2f(v[i] >> 16);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; i++) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  // a NaN, which min and max pass over, by the largest magnitude's bits
  auto mag = [](uint32_t w) { return __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu); };
  u16x2_t top = __builtin_elementwise_max(__builtin_elementwise_max(mag(v[0]), mag(v[1])),
                                          __builtin_elementwise_max(mag(v[2]), mag(v[3])));
  // over the group's 8 lanes: lane ^ 1, lane ^ 2, 7 - lane (quad_perm twice, row_half_mirror)
  lo = fminf(lo, dpp_f32<0xB1>(lo));
  hi = fmaxf(hi, dpp_f32<0xB1>(hi));
  top = __builtin_elementwise_max(top, dpp_u16x2<0xB1>(top));
  lo = fminf(lo, dpp_f32<0x4E>(lo));
  hi = fmaxf(hi, dpp_f32<0x4E>(hi));
  top = __builtin_elementwise_max(top, dpp_u16x2<0x4E>(top));
  lo = fminf(lo, dpp_f32<0x141>(lo));
  hi = fmaxf(hi, dpp_f32<0x141>(hi));
  top = __builtin_elementwise_max(top, dpp_u16x2<0x141>(top));
  const uint16_t sb = kv4_scale(lo, hi, max(top.x, top.y) > 0x7f80u);
  const float s = bf2f(sb), rs = 1.0f / s;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) word |= kv4_nibble(x[i], lo, s, rs) << (4 * i);
  const int64_t slot = h * p.cap + p.offset + m;
  t.w[slot * kKv4Words + li] = word;
  const uint16_t bb = s != s ? 0x7fc0u : f2bf(lo);
  const uint32_t so = __shfl_xor(static_cast<uint32_t>(sb), 8, 64);
  const uint32_t bo = __shfl_xor(static_cast<uint32_t>(bb), 8, 64);
  if (li == 0) {
    t.s[slot] = sb | (so << 16);
    t.b[slot] = bb | (bo << 16);
  }
}

// The inverse: one word per thread, 16 bytes out.
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4RowsParams p) {
  const int m = blockIdx.x * 16 + (threadIdx.x >> 4), li = threadIdx.x & 15;
  if (m >= p.M) return;
  const Kv4Tensor& t = p.t[blockIdx.z];
  const int64_t h = blockIdx.y;
  const int64_t slot = h * p.cap + p.offset + m;
  const uint32_t wd = t.w[slot * kKv4Words + li];
  const int sh = li < 8 ? 0 : 16;
  const float s = bf2f((t.s[slot] >> sh) & 0xffffu), b = bf2f((t.b[slot] >> sh) & 0xffffu);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    // s * n is exact, so the fused multiply-add rounds as the two operations do
    const float lo = __builtin_fmaf(s, static_cast<float>((wd >> (8 * i)) & 0xfu), b);
    const float hi = __builtin_fmaf(s, static_cast<float>((wd >> (8 * i + 4)) & 0xfu), b);
    o[i] = static_cast<uint32_t>(f2bf(lo)) | (static_cast<uint32_t>(f2bf(hi)) << 16);
  }
  *reinterpret_cast<uint4*>(const_cast<uint16_t*>(t.x) + (h * p.M + m) * kKv4Dim + 8 * li) = make_uint4(o[0], o[1], o[2], o[3]);
}

struct QkKv4Params {
  const uint16_t* q;  // [M, Hq*128]
  const uint16_t* k;  // [M, Hkv*128]
  const uint16_t* v;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  uint16_t* q_out;  // [Hq, M, 128]
  bmx_kv4 c;
  int M, Hq, offset;
  int64_t position;
  float eps;
  RopeTable tab;
};

// Quantizes one row held by a wave (lane: values lane and lane + 64, that
// is, one of each group) and writes it.
__device__ __forceinline__ void kv4_store_row(float a, float b, int lane, uint32_t* w, uint32_t* s, uint32_t* bias) {
  const float x[2] = {a, b};
  uint32_t sw = 0, bw = 0;
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const float lo = kv4_min64(x[g]), hi = kv4_max64(x[g]);
    const uint16_t sb = kv4_scale(lo, hi, __any(x[g] != x[g]));
    const float sf = bf2f(sb);
    uint32_t n = kv4_nibble(x[g], lo, sf, 1.0f / sf) << (4 * (lane & 7));
    n |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(n), 0xB1, 0xF, 0xF, false));
    n |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(n), 0x4E, 0xF, 0xF, false));
    n |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(n), 0x141, 0xF, 0xF, false));
    if ((lane & 7) == 0) w[8 * g + (lane >> 3)] = n;
    sw |= static_cast<uint32_t>(sb) << (16 * g);
    bw |= static_cast<uint32_t>(sf != sf ? 0x7fc0u : f2bf(lo)) << (16 * g);
  }
  if (lane == 0) {
    *s = sw;
    *bias = bw;
  }
}

// One wave per (token, q head or kv head); lane i holds the rotate-half pair
// (i, i + 64), with the norm and rotation of qk_norm_rope_kv.
__global__ void __launch_bounds__(256) qk_norm_rope_kv4_kernel(const QkKv4Params p) {
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int Hkv = p.c.n_kv_heads, H = p.Hq + Hkv;
  if (wid >= static_cast<int64_t>(p.M) * H) return;
  const int t = static_cast<int>(wid / H), g = static_cast<int>(wid - static_cast<int64_t>(t) * H);
  const bool is_q = g < p.Hq;
  const int h = is_q ? g : g - p.Hq;
  const uint16_t* src = (is_q ? p.q + static_cast<int64_t>(t) * p.Hq * 128 : p.k + static_cast<int64_t>(t) * Hkv * 128) +
                        static_cast<int64_t>(h) * 128;
  const uint16_t* nw = is_q ? p.q_norm : p.k_norm;
  float c, s;
  rope_cs(p.tab.inv_freq[lane], static_cast<float>(p.position + t), c, s);
  uint16_t o1, o2;
  qk_norm_rope_lane_cs(bf2f(src[lane]), bf2f(src[lane + 64]), bf2f(nw[lane]), bf2f(nw[lane + 64]), c, s, p.eps, o1, o2);
  if (is_q) {
    uint16_t* dst = p.q_out + (static_cast<int64_t>(h) * p.M + t) * 128;
    dst[lane] = o1;
    dst[lane + 64] = o2;
    return;
  }
  const int64_t slot = static_cast<int64_t>(h) * p.c.capacity + p.offset + t;
  kv4_store_row(bf2f(o1), bf2f(o2), lane, p.c.k + slot * kKv4Words, reinterpret_cast<uint32_t*>(p.c.k_scales) + slot,
                reinterpret_cast<uint32_t*>(p.c.k_biases) + slot);
  const uint16_t* vs = p.v + (static_cast<int64_t>(t) * Hkv + h) * 128;
  kv4_store_row(bf2f(vs[lane]), bf2f(vs[lane + 64]), lane, p.c.v + slot * kKv4Words,
                reinterpret_cast<uint32_t*>(p.c.v_scales) + slot, reinterpret_cast<uint32_t*>(p.c.v_biases) + slot);
}

Kv4RowsParams rows_params(const bmx_kv4& c, int M, int offset) {
  Kv4RowsParams p{};
  p.t[0].w = c.k;
  p.t[0].s = reinterpret_cast<uint32_t*>(c.k_scales);
  p.t[0].b = reinterpret_cast<uint32_t*>(c.k_biases);
  p.t[1].w = c.v;
  p.t[1].s = reinterpret_cast<uint32_t*>(c.v_scales);
  p.t[1].b = reinterpret_cast<uint32_t*>(c.v_biases);
  p.M = M;
  p.cap = c.capacity;
  p.offset = offset;
  return p;
}

// 16 rows of a head and array per workgroup
dim3 rows_grid(const bmx_kv4& c, int M) {
  return dim3(static_cast<unsigned>((M + 15) / 16), static_cast<unsigned>(c.n_kv_heads), 2);
}

}  // namespace

int launch_kv4_read(const bmx_kv4& c, uint16_t* k, uint16_t* v, int M, int start, hipStream_t stream) {
  Kv4RowsParams p = rows_params(c, M, start);
  p.t[0].x = k;
  p.t[1].x = v;
  hipLaunchKernelGGL(kv4_read_kernel, rows_grid(c, M), dim3(256), 0, stream, p);
  return check_launch("kv4_read");
}

}  // namespace bmx

using namespace bmx;

extern "C" int bmx_kv4_write(const bmx_bf16* k, int64_t k_head_stride, int64_t k_row_stride, const bmx_bf16* v,
                             int64_t v_head_stride, int64_t v_row_stride, const bmx_kv4* cache, int M, int head_dim,
                             int offset, void* stream) {
  if (int rc = check_kv4("kv4_write", cache, head_dim)) return rc;
  if (!k || !v) return set_error(BMX_E_ARG, "kv4_write: null pointer");
  if (int rc = check_kv4_rows("kv4_write", cache, M, offset)) return rc;
  if (k_head_stride < 0 || k_row_stride < 0 || v_head_stride < 0 || v_row_stride < 0)
    return set_error(BMX_E_SHAPE, "kv4_write: negative stride");
  if ((k_head_stride | k_row_stride | v_head_stride | v_row_stride) % 8 || !aligned(k, 16) || !aligned(v, 16))
    return set_error(BMX_E_ALIGN, "kv4_write: k and v must be 16-byte aligned, strides multiples of 8");
  if (M == 0) return BMX_OK;
  Kv4RowsParams p = rows_params(*cache, M, offset);
  p.t[0].x = k;
  p.t[0].head_stride = k_head_stride;
  p.t[0].row_stride = k_row_stride;
  p.t[1].x = v;
  p.t[1].head_stride = v_head_stride;
  p.t[1].row_stride = v_row_stride;
  hipLaunchKernelGGL(kv4_write_kernel, rows_grid(*cache, M), dim3(256), 0, as_stream(stream), p);
  return check_launch("kv4_write");
}

extern "C" int bmx_kv4_read(const bmx_kv4* cache, bmx_bf16* k, bmx_bf16* v, int M, int head_dim, int start,
                            void* stream) {
  if (int rc = check_kv4("kv4_read", cache, head_dim)) return rc;
  if (!k || !v) return set_error(BMX_E_ARG, "kv4_read: null pointer");
  if (int rc = check_kv4_rows("kv4_read", cache, M, start)) return rc;
  if (!aligned(k, 16) || !aligned(v, 16)) return set_error(BMX_E_ALIGN, "kv4_read: k and v must be 16-byte aligned");
  if (M == 0) return BMX_OK;
  return launch_kv4_read(*cache, k, v, M, start, as_stream(stream));
}

extern "C" int bmx_qk_norm_rope_kv4(const bmx_bf16* q, const bmx_bf16* k, const bmx_bf16* v, const bmx_bf16* q_norm,
                                    const bmx_bf16* k_norm, bmx_bf16* q_out, const bmx_kv4* cache, int M, int n_heads,
                                    int head_dim, int offset, int64_t position, float eps, float theta,
                                    void* stream) {
  if (int rc = check_kv4("qk_norm_rope_kv4", cache, head_dim)) return rc;
  if (!q || !k || !v || !q_norm || !k_norm || !q_out) return set_error(BMX_E_ARG, "qk_norm_rope_kv4: null pointer");
  if (n_heads <= 0) return set_error(BMX_E_SHAPE, "qk_norm_rope_kv4: n_heads=%d", n_heads);
  if (int rc = check_kv4_rows("qk_norm_rope_kv4", cache, M, offset)) return rc;
  if (position < 0 || position > kMaxPosition - (M - 1))
    return set_error(BMX_E_ARG, "qk_norm_rope_kv4: position=%lld, M=%d (up to position %d)",
                     static_cast<long long>(position), M, kMaxPosition);
  if (M == 0) return BMX_OK;
  const int64_t waves = static_cast<int64_t>(M) * (n_heads + cache->n_kv_heads);
  if (waves > INT32_MAX) return set_error(BMX_E_SHAPE, "qk_norm_rope_kv4: M=%d too large for one launch", M);
  QkKv4Params p{q, k, v, q_norm, k_norm, q_out, *cache, M, n_heads, offset, position, eps,
                make_rope_table(head_dim, theta)};
  hipLaunchKernelGGL(qk_norm_rope_kv4_kernel, dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0,
                     as_stream(stream), p);
  return check_launch("qk_norm_rope_kv4");
}
