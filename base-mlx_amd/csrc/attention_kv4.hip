// Attention over the 4-bit KV cache, and the weight each cached position
// drew (gfx950).
//
//   S[t, j] = scale * sum_d q[t, d] (s n + b)[j, d],  j <= offset + t
//   P = softmax(S),  out = bf16(P (s n + b)),  weights[h, j] += sum P[., j]
//
// Nibbles go to the matrix cores without a conversion: (w shifted) & 0x78 |
// 0x4180 per half is the bf16 number 16 + n, exactly, one shift and one
// and-or for two values.  With Q_g the sum of q over group g and scores
// computed transposed (rows: keys, columns: queries),
//   S / scale = sum_g s_g (sum_d q_d (16 + n_d) - 16 Q_g) + b_g Q_g,
// where -16 Q_g is the accumulator's start and b_g Q_g one more product over
// k = (group, piece) with Q_g in three bf16 pieces (24 bits); the scales
// multiply fp32 results.  So a score is fp32 arithmetic on the stored values:
// nothing of K is rounded.  For the values, with p' = bf16(p s_g),
//   sum_j p_j (s n + b)_j = sum_j p'_j (16 + n_j) - 23.5 sum_j p'_j
//                         + 7.5 sum_j p~_j s_j + sum_j p~_j b_j,  p~ = bf16(p):
// the roundings of p' then act on n - 7.5, the centred nibble, and so weigh
// no more than rounding P does in a bf16 attention.  The last three sums are
// products with constant or raw scale / bias rows.
#include <math.h>

#include <algorithm>

#include "kv4.h"

namespace bmx {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBufferConfig = 0x00020000;  // raw buffer, range checked per dword against num_records
constexpr int kRows = 16;                  // query rows per wave
constexpr int kKeys = 32;                  // keys per step of a wave
constexpr int kMaxSplits = 64;             // (a lane per split in the merge)
constexpr int kOs = kKv4Dim + 4;           // LDS stride of an output row

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

struct Kv4AttnParams {
  const uint16_t* q;  // [Hq, M, 128]
  bmx_kv4 c;
  uint16_t* out;      // [M, Hq*128]
  float* weights;     // [Hkv, cap], or null
  unsigned* cnt;      // arrival counters, cnt_stride words apart, zero between calls
  float2* lse;        // [Hq, M] (max * c2, log2 of the sum), or null
  uint4* qp;          // [Hq, M] the three pieces of Q_0 and Q_1, with lse
  float* part_o;      // [Hq, M, ns, 128]
  float* part_ml;     // [Hq, M, ns, 2]
  int Hq, M, offset;
  float c2;           // |scale| log2(e)
  uint32_t flip;      // sign bits of a bf16 pair where scale < 0
  int ns;             // key splits
  int bps;            // steps of all waves per split
  int cnt_stride;
  int rw;             // weigh: waves of a workgroup that share keys
};

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}

// The masks of the nibble pairs, held in registers (a gfx9 and-or takes no
// literal)
struct PairK {
  uint32_t mask, one;
  __device__ __forceinline__ PairK() : mask(0x00780078u), one(0x41804180u) { asm volatile("" : "+v"(mask), "+v"(one)); }
};
// Nibbles i and i + 4 of w as the bf16 pair (16 + n_i, 16 + n_(i+4))
template <int I>
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, const PairK& k) {
  return ((I == 0 ? w << 3 : w >> (4 * I - 3)) & k.mask) | k.one;
}
__device__ __forceinline__ u32x4_t word_pairs(uint32_t w, const PairK& k) {
  return u32x4_t{nibble_pair<0>(w, k), nibble_pair<1>(w, k), nibble_pair<2>(w, k), nibble_pair<3>(w, k)};
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
  return static_cast<uint32_t>(f2bf(a)) | (static_cast<uint32_t>(f2bf(b)) << 16);
}
__device__ __forceinline__ uint32_t dpp_ror8(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xF, 0xF, false));
}
// A head's array as a buffer that ends after `bytes`: reads past it give
// zeros without a memory access
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const uint32_t* base, int64_t words, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(base) + words, static_cast<short>(0), bytes,
                                           kBufferConfig);
}
__device__ __forceinline__ u32x4_t load4(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ u32x2_t load2(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
}
__device__ __forceinline__ uint32_t load1(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}

// Partials travel between workgroups (and XCDs) through agent-scope
// accesses: written through to memory, complete before the arrival, read
// after it.
__device__ __forceinline__ void store_part(float* p, float x, float y) {
  const uint64_t v = static_cast<uint64_t>(__float_as_uint(x)) | (static_cast<uint64_t>(__float_as_uint(y)) << 32);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_part(const float* p) {
  const uint64_t v =
      __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// One output row's 4 dims, and the row's softmax statistics for the weights.
__device__ __forceinline__ void finish_row(const Kv4AttnParams& p, int kvh, int r, int d, float4 o, float m, float l) {
  const int rep = p.Hq / p.c.n_kv_heads, t = r % p.M, h = kvh * rep + r / p.M;
  const float inv = 1.0f / l;
  *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(t) * p.Hq + h) * kKv4Dim + d) =
      make_uint2(pack_bf(o.x * inv, o.y * inv), pack_bf(o.z * inv, o.w * inv));
  if (p.lse && d == 0) p.lse[static_cast<int64_t>(kvh) * rep * p.M + r] = make_float2(m * p.c2, log2f(l));
}

// A workgroup of NW waves: one kv head, 16 query rows (row r = j * M + t:
// head kvh * rep + j, token t), one split of the keys; a wave takes 32 keys
// a step, with its own running maximum and sums.
//   Lanes: li = lane % 16, g = lane / 16.
//   K (A operand): keys li of two 16-key tiles, words 2g, 2g+1 (group 0) and
//     8 + 2g, 9 + 2g (group 1) of their rows.
//   Scores (D): query li, keys 4g .. 4g+3 of each tile -- which is the B
//     operand of P V when its k index runs over keys 4g..4g+3, 16+4g..+3, so
//     P never leaves the lane.
//   V (A operand): rows are the 16 (word, half) pairs of 8 words of a group,
//     with nibble i of the half in product i: dims 64 y + 8 (li % 8) +
//     4 (li / 8) + i.  Lane li < 8 loads a word of the even key of a pair,
//     lane li + 8 the same word of the odd key, and they swap halves.
// The next step's K is loaded once the scores are done, its V once P V is.
template <int NW>
__global__ void __launch_bounds__(64 * NW) kv4_split_kernel(const Kv4AttnParams p) {
  __shared__ __align__(16) float os[NW][kRows][kOs];
  __shared__ float ms[NW][kRows], ls[NW][kRows], wt[kRows][kMaxSplits], fin[kRows][2];
  __shared__ int last;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, split = blockIdx.y, r0 = blockIdx.z * kRows;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, RT = min(kRows, R - r0), L = p.offset + M;
  const int64_t row0 = static_cast<int64_t>(kvh) * R + r0;
  // rows' tokens: query li sees keys < lim; the tile's first and last token
  const int lim = p.offset + (r0 + min(li, RT - 1)) % M + 1;
  const int t0 = r0 % M, tmin = t0 + RT > M ? 0 : t0, tmax = t0 + RT > M ? M - 1 : t0 + RT - 1;
  const int all_see = p.offset + tmin + 1, kend = p.offset + tmax + 1;
  const PairK nk;

  const int64_t slot = static_cast<int64_t>(kvh) * p.c.capacity;
  const __amdgpu_buffer_rsrc_t kwr = rsrc(p.c.k, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t vwr = rsrc(p.c.v, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t ksr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t kbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_biases), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vsr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_biases), slot, L * 4);

  u32x2_t kw[2][2];  // [tile][group]
  uint32_t kb[2];
  u32x4_t ks[2];
  uint32_t vw[2][4];  // [group][key pair]
  u32x4_t vs[2], vb[2];
  auto load_k = [&](int b) {
    const int w = (b * kKeys + li) * 64 + 8 * g, s = b * kKeys * 4;
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (int y = 0; y < 2; y++) kw[t][y] = load2(kwr, w + t * 1024 + y * 32);
      kb[t] = load1(kbr, s + (16 * t + li) * 4);
      ks[t] = load4(ksr, s + (16 * t + 4 * g) * 4);
    }
  };
  auto load_v = [&](int b) {
    const int w = (b * kKeys + 4 * g + (li >> 3)) * 64 + 4 * (li & 7), s = (b * kKeys + 4 * g) * 4;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int y = 0; y < 2; y++) vw[y][j] = load1(vwr, w + ((j & 1) * 2 + (j >> 1) * 16) * 64 + y * 32);
#pragma unroll
    for (int t = 0; t < 2; t++) {
      vs[t] = load4(vsr, s + t * 64);
      vb[t] = load4(vbr, li < 2 ? s + t * 64 : 0x7ffffff0);  // only lanes li < 2 use it (edge steps load the rest)
    }
  };

  const int blocks = (kend + kKeys - 1) / kKeys;
  const int b_end = min(blocks, (split + 1) * p.bps * NW);
  int b = split * p.bps * NW + wave;
  load_k(b);
  load_v(b);

  // ---- the query fragments, in the pair order of a word, and their sums ----
  u32x4_t qf[2][2];
  f32x4_t start[2];  // -16 Q_y of query li
  u32x4_t qp;        // lanes g = 0: Q_0, Q_1 in three bf16 pieces each
  {
    const uint16_t* qr = p.q + (row0 + min(li, RT - 1)) * kKv4Dim + 16 * g;
    float qs[2];
#pragma unroll
    for (int y = 0; y < 2; y++) {
      qs[y] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        uint4 d = *reinterpret_cast<const uint4*>(qr + 64 * y + 8 * e);
        d.x ^= p.flip;
        d.y ^= p.flip;
        d.z ^= p.flip;
        d.w ^= p.flip;
        qs[y] += gemv_unit_sum(d);
        d = permute_pairs(d);
        qf[y][e] = u32x4_t{d.x, d.y, d.z, d.w};
      }
      qs[y] = add_xor32(add_xor16(qs[y]));
      start[y] = f32x4_t{-16.0f, -16.0f, -16.0f, -16.0f} * qs[y];
    }
    const float h0 = round_bf(qs[0]), h1 = round_bf(qs[1]);
    const float m0 = round_bf(qs[0] - h0), m1 = round_bf(qs[1] - h1);
    qp = u32x4_t{pack_bf(h0, h1), pack_bf(m0, m1), pack_bf(qs[0] - h0 - m0, qs[1] - h1 - m1), 0u};
    if (p.qp && split == 0 && wave == 0 && g == 0 && li < RT) p.qp[row0 + li] = make_uint4(qp.x, qp.y, qp.z, 0u);
    if (g != 0) qp = u32x4_t{0u, 0u, 0u, 0u};
  }

  const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x4_t acc[2][4], ones[2], edge = zero;
#pragma unroll
  for (int y = 0; y < 2; y++) {
    ones[y] = zero;
#pragma unroll
    for (int i = 0; i < 4; i++) acc[y][i] = zero;
  }
  float m = -INFINITY, l = 0.0f, slow[2] = {0.0f, 0.0f};
  constexpr uint32_t kCentre = 0xC1BCC1BCu;  // bf16 -23.5 twice
  const uint32_t half_sel = li < 8 ? 0x01000504u : 0x07060302u;
  const uint32_t odd_sel = li & 1 ? 0x07060302u : 0x05040100u;

  for (; b < b_end; b += NW) {
    // ---- scores ----
    float sc[8];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f32x4_t d0 = start[0], d1 = start[1];
      d0 = mfma(word_pairs(kw[t][0].x, nk), qf[0][0], d0);
      d1 = mfma(word_pairs(kw[t][1].x, nk), qf[1][0], d1);
      d0 = mfma(word_pairs(kw[t][0].y, nk), qf[0][1], d0);
      d1 = mfma(word_pairs(kw[t][1].y, nk), qf[1][1], d1);
      const f32x4_t db = mfma(u32x4_t{kb[t], kb[t], kb[t], kb[t]}, qp, zero);
#pragma unroll
      for (int i = 0; i < 4; i++)
        sc[4 * t + i] =
            __builtin_fmaf(lo_f(ks[t][i]), d0[i], __builtin_fmaf(hi_f(ks[t][i]), d1[i], db[i]));
    }
    load_k(b + NW);
    // ---- running softmax: the maximum over all keys of query li ----
    const int key0 = b * kKeys + 4 * g;
    const bool cut = b * kKeys + kKeys > all_see;  // uniform: some row does not see some key
    if (cut) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (key0 + (e & 3) + 16 * (e >> 2) >= lim) sc[e] = -INFINITY;
    }
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < 8; e++) bm = fmaxf(bm, sc[e]);
    bm = max_xor32(max_xor16(bm));
    if (__any(bm > m)) {
      const float mn = fmaxf(m, bm);
      const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * p.c2);
      m = mn;
      l *= a;
      edge *= a;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        slow[y] *= a;
        ones[y] *= a;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[y][i] *= a;
      }
    }
    const float mc = m == -INFINITY ? 0.0f : m * p.c2;
    float pr[8];
#pragma unroll
    for (int e = 0; e < 8; e++) pr[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], p.c2, -mc));
    if (cut) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (key0 + (e & 3) + 16 * (e >> 2) >= lim) pr[e] = 0.0f;
    }
    l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
    // ---- P V ----
    float ps[2][8];
    uint32_t sw[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      sw[e] = vs[e >> 2][e & 3];
      ps[0][e] = pr[e] * lo_f(sw[e]);
      ps[1][e] = pr[e] * hi_f(sw[e]);
    }
    bool odd = false;
    if (cut) {
      // rows that a query does not see weigh nothing in it, whatever their
      // scales and biases are: its P V column has zeros for them, and biases
      // that are not finite go to the lanes' own sums of the rows that see
      // them, not into the product that every query shares
      u32x4_t bw[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        bw[t] = load4(vbr, key0 * 4 + t * 64);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float f = (lo_f(bw[t][i]) + lo_f(vs[t][i])) * 0.0f + (hi_f(bw[t][i]) + hi_f(vs[t][i])) * 0.0f;
          odd |= f != 0.0f;  // NaN
        }
      }
      odd = __any(odd);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool seen = key0 + (e & 3) + 16 * (e >> 2) < lim;
        if (!seen) ps[0][e] = ps[1][e] = 0.0f;
        if (odd && seen) {
          slow[0] += lo_f(bw[e >> 2][e & 3]) * 0.0f;  // 0 or NaN
          slow[1] += hi_f(bw[e >> 2][e & 3]) * 0.0f;
        }
      }
    }
    u32x4_t pb[2], pt;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      pb[0][j] = pack_bf(ps[0][2 * j], ps[0][2 * j + 1]);
      pb[1][j] = pack_bf(ps[1][2 * j], ps[1][2 * j + 1]);
      pt[j] = pack_bf(pr[2 * j], pr[2 * j + 1]);
    }
#pragma unroll
    for (int y = 0; y < 2; y++) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = __builtin_amdgcn_perm(vw[y][j], dpp_ror8(vw[y][j]), half_sel);
      acc[y][0] = mfma(u32x4_t{nibble_pair<0>(v[0], nk), nibble_pair<0>(v[1], nk), nibble_pair<0>(v[2], nk),
                               nibble_pair<0>(v[3], nk)}, pb[y], acc[y][0]);
      acc[y][1] = mfma(u32x4_t{nibble_pair<1>(v[0], nk), nibble_pair<1>(v[1], nk), nibble_pair<1>(v[2], nk),
                               nibble_pair<1>(v[3], nk)}, pb[y], acc[y][1]);
      acc[y][2] = mfma(u32x4_t{nibble_pair<2>(v[0], nk), nibble_pair<2>(v[1], nk), nibble_pair<2>(v[2], nk),
                               nibble_pair<2>(v[3], nk)}, pb[y], acc[y][2]);
      acc[y][3] = mfma(u32x4_t{nibble_pair<3>(v[0], nk), nibble_pair<3>(v[1], nk), nibble_pair<3>(v[2], nk),
                               nibble_pair<3>(v[3], nk)}, pb[y], acc[y][3]);
      ones[y] = mfma(u32x4_t{kCentre, kCentre, kCentre, kCentre}, pb[y], ones[y]);
    }
    {
      // rows 0..3 of A: b_0, b_1, s_0, s_1 of the step's keys (the other
      // rows' results are not used)
      u32x4_t a;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t x = li < 2 ? vb[j >> 1][2 * (j & 1)] : vs[j >> 1][2 * (j & 1)];
        const uint32_t z = li < 2 ? vb[j >> 1][2 * (j & 1) + 1] : vs[j >> 1][2 * (j & 1) + 1];
        a[j] = __builtin_amdgcn_perm(z, x, odd_sel);
        if (odd) {
          if ((a[j] & 0x7f80u) == 0x7f80u) a[j] &= 0xffff0000u;
          if ((a[j] & 0x7f800000u) == 0x7f800000u) a[j] &= 0xffffu;
        }
      }
      edge = mfma(a, pt, edge);
    }
    load_v(b + NW);
  }

  // ---- the waves' sums joined: weights exp2((m_w - m) c2) ----
  l = add_xor32(add_xor16(l));
  if (l != l) m = l;  // a NaN score: the row stays NaN
  if (g == 0) {
    ms[wave][li] = m;
    ls[wave][li] = l;
  }
  __syncthreads();
  {
    float mm = ms[0][li];
#pragma unroll
    for (int w = 1; w < NW; w++) mm = fmaxf(mm, ms[w][li]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mm) * p.c2);
    float x[2];
#pragma unroll
    for (int y = 0; y < 2; y++)
      x[y] = ones[y][0] + __builtin_fmaf(7.5f, __shfl(edge[2 + y], li, 64), __shfl(edge[y], li, 64)) +
             add_xor32(add_xor16(slow[y]));
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int a = 4 * g + i;  // row of A: word a % 8, half a / 8
        *reinterpret_cast<float4*>(&os[wave][li][64 * y + 8 * (a & 7) + 4 * (a >> 3)]) =
            make_float4((acc[y][0][i] + x[y]) * f, (acc[y][1][i] + x[y]) * f, (acc[y][2][i] + x[y]) * f,
                        (acc[y][3][i] + x[y]) * f);
      }
  }
  __syncthreads();
  for (int it = tid; it < RT * 32; it += 64 * NW) {
    const int r = it >> 5, d = 4 * (it & 31);
    float mm = ms[0][r];
#pragma unroll
    for (int w = 1; w < NW; w++) mm = fmaxf(mm, ms[w][r]);
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = ms[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ms[w][r] - mm) * p.c2);
      sum = __builtin_fmaf(f, ls[w][r], sum);
      const float4 v = *reinterpret_cast<const float4*>(&os[w][r][d]);
      o.x += v.x;
      o.y += v.y;
      o.z += v.z;
      o.w += v.w;
    }
    if (sum != sum) mm = sum;
    if (p.ns == 1) {
      finish_row(p, kvh, r0 + r, d, o, mm, sum);
    } else {
      const int64_t at = (row0 + r) * p.ns + split;
      store_part(p.part_o + at * kKv4Dim + d, o.x, o.y);
      store_part(p.part_o + at * kKv4Dim + d + 2, o.z, o.w);
      if (d == 0) store_part(p.part_ml + at * 2, mm, sum);
    }
  }
  if (p.ns == 1) return;

  // ---- the last workgroup of a (kv head, row tile) merges its splits ----
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    unsigned* c = p.cnt + (static_cast<int64_t>(blockIdx.z) * gridDim.x + kvh) * p.cnt_stride;
    const unsigned n = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = n == static_cast<unsigned>(p.ns - 1);
    if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  // a wave per row, a lane per split: the splits' weights
  for (int r = wave; r < RT; r += NW) {
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < p.ns) ml = load_part(p.part_ml + ((row0 + r) * p.ns + lane) * 2);
    const float mm = max_xor32(max_xor16(row16_max(ml.x)));
    const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml.x - mm) * p.c2);
    const float sum = lanes_sum(f * ml.y, 64);
    wt[r][lane] = f;
    if (lane == 0) {
      fin[r][0] = mm;
      fin[r][1] = sum;
    }
  }
  __syncthreads();
  // (row, 4 dims) per thread, and the splits over as many threads as there are
  constexpr int kThreads = 64 * NW;
  const int items = RT * 32, groups = max(1, kThreads / items);
  const int n = tid / items;  // this thread's group; those past the last have none
  float* red = &os[0][0][0];
  for (int it = tid - n * items; it < items && n < groups; it += kThreads) {
    const int r = it >> 5, d = 4 * (it & 31);
    const float* src = p.part_o + (row0 + r) * p.ns * kKv4Dim + d;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int s = n; s < p.ns; s += groups) {
      const float2 u = load_part(src + static_cast<int64_t>(s) * kKv4Dim);
      const float2 v = load_part(src + static_cast<int64_t>(s) * kKv4Dim + 2);
      const float f = wt[r][s];
      if (f != 0.0f) {
        o.x = __builtin_fmaf(f, u.x, o.x);
        o.y = __builtin_fmaf(f, u.y, o.y);
        o.z = __builtin_fmaf(f, v.x, o.z);
        o.w = __builtin_fmaf(f, v.y, o.w);
      }
    }
    if (groups == 1)
      finish_row(p, kvh, r0 + r, d, o, fin[r][0], fin[r][1]);
    else
      *reinterpret_cast<float4*>(&red[(n * items + it) * 4]) = o;
  }
  if (groups == 1) return;
  __syncthreads();
  for (int it = tid; it < items; it += kThreads) {
    float4 o = *reinterpret_cast<const float4*>(&red[it * 4]);
    for (int k = 1; k < groups; k++) {
      const float4 v = *reinterpret_cast<const float4*>(&red[(k * items + it) * 4]);
      o.x += v.x;
      o.y += v.y;
      o.z += v.z;
      o.w += v.w;
    }
    finish_row(p, kvh, r0 + (it >> 5), 4 * (it & 31), o, fin[it >> 5][0], fin[it >> 5][1]);
  }
}

// weights[h][j] += sum over the query rows of exp2(S c2 - max c2 - log2 sum).
// A wave holds 32 keys unpacked and walks the query rows 16 at a time; rw
// waves of a workgroup share keys and take every rw-th row tile.
constexpr int kWeighWaves = 8;
__global__ void __launch_bounds__(64 * kWeighWaves) kv4_weigh_kernel(const Kv4AttnParams p) {
  __shared__ float red[kWeighWaves][kKeys];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, kg = kWeighWaves / p.rw;  // key blocks per workgroup
  const int b = blockIdx.y * kg + wave / p.rw, rs = wave % p.rw;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, L = p.offset + M;
  const int tiles = (R + kRows - 1) / kRows;
  const int64_t slot = static_cast<int64_t>(kvh) * p.c.capacity, row0 = static_cast<int64_t>(kvh) * R;
  const PairK nk;
  float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (b * kKeys < L) {
    const __amdgpu_buffer_rsrc_t kwr = rsrc(p.c.k, slot * kKv4Words, L * 64);
    const __amdgpu_buffer_rsrc_t ksr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_scales), slot, L * 4);
    const __amdgpu_buffer_rsrc_t kbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_biases), slot, L * 4);
    u32x4_t ka[2][2][2];  // [tile][group][word]
    u32x4_t kb[2];
    float ks[2][8];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const int key = b * kKeys + 16 * t;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const u32x2_t w = load2(kwr, (key + li) * 64 + 8 * g + 32 * y);
        ka[t][y][0] = word_pairs(w.x, nk);
        ka[t][y][1] = word_pairs(w.y, nk);
      }
      const uint32_t bw = load1(kbr, (key + li) * 4);
      kb[t] = u32x4_t{bw, bw, bw, bw};
      const u32x4_t s = load4(ksr, (key + 4 * g) * 4);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ks[0][4 * t + i] = lo_f(s[i]);
        ks[1][4 * t + i] = hi_f(s[i]);
      }
    }
    for (int rt = rs; rt < tiles; rt += p.rw) {
      const int r = rt * kRows + li, rc = min(r, R - 1);
      const int t0 = rt * kRows % M, n = min(kRows, R - rt * kRows);
      const int tmax = t0 + n > M ? M - 1 : t0 + n - 1, tmin = t0 + n > M ? 0 : t0;
      if (b * kKeys > p.offset + tmax) continue;  // uniform: none of these rows sees any of these keys
      const uint16_t* qr = p.q + (row0 + rc) * kKv4Dim + 16 * g;
      u32x4_t qf[2][2];
#pragma unroll
      for (int y = 0; y < 2; y++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          uint4 d = *reinterpret_cast<const uint4*>(qr + 64 * y + 8 * e);
          d = permute_pairs(d);
          qf[y][e] = u32x4_t{d.x ^ p.flip, d.y ^ p.flip, d.z ^ p.flip, d.w ^ p.flip};
        }
      const uint4 pieces = p.qp[row0 + rc];
      const float2 st = p.lse[row0 + rc];
      const u32x4_t qp = g ? u32x4_t{0u, 0u, 0u, 0u} : u32x4_t{pieces.x, pieces.y, pieces.z, 0u};
      const float q0 = lo_f(pieces.x) + lo_f(pieces.y) + lo_f(pieces.z);
      const float q1 = hi_f(pieces.x) + hi_f(pieces.y) + hi_f(pieces.z);
      const f32x4_t one = {-16.0f, -16.0f, -16.0f, -16.0f};
      const bool cut = n < kRows || b * kKeys + kKeys > p.offset + tmin + 1;
      const int lim = r < R ? p.offset + r % M + 1 : 0;
#pragma unroll
      for (int t = 0; t < 2; t++) {
        f32x4_t d0 = one * q0, d1 = one * q1;
        d0 = mfma(ka[t][0][0], qf[0][0], d0);
        d1 = mfma(ka[t][1][0], qf[1][0], d1);
        d0 = mfma(ka[t][0][1], qf[0][1], d0);
        d1 = mfma(ka[t][1][1], qf[1][1], d1);
        const f32x4_t db = mfma(kb[t], qp, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int e = 4 * t + i;
          const float s = __builtin_fmaf(ks[0][e], d0[i], __builtin_fmaf(ks[1][e], d1[i], db[i]));
          float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c2, -st.x) - st.y);
          if (cut && b * kKeys + 16 * t + 4 * g + i >= lim) w = 0.0f;
          acc[e] += w;
        }
      }
    }
  }
  // over the 16 queries of a lane row, then over the waves that share keys
#pragma unroll
  for (int e = 0; e < 8; e++) {
    acc[e] = row16_sum(acc[e]);
    if (li == 0) red[wave][16 * (e >> 2) + 4 * g + (e & 3)] = acc[e];
  }
  __syncthreads();
  const int k = tid >> 5;  // key block of the workgroup
  if (k >= kg) return;
  const int key = (blockIdx.y * kg + k) * kKeys + (tid & 31);
  if (key >= L) return;
  float s = red[k * p.rw][tid & 31];
  for (int i = 1; i < p.rw; i++) s += red[k * p.rw + i][tid & 31];
  p.weights[slot + key] += s;
}

constexpr int64_t kMaxQueryRows = 1 << 28;  // Hq * M of a call

bool attn_shape_ok(int Hq, int Hkv, int M, int64_t L) {
  if (Hkv <= 0 || Hkv > 65535 || Hq <= 0 || Hq > 65535 || Hq % Hkv || M <= 0 || L < M || L > kKv4MaxCapacity ||
      static_cast<int64_t>(Hq) * M > kMaxQueryRows)
    return false;
  return (static_cast<int64_t>(Hq / Hkv) * M + kRows - 1) / kRows <= 65535;  // row tiles: grid z
}

constexpr int kSplitWaves = 8;
constexpr int kSplitGrid = 512;  // workgroups that a call's splits aim at

// Where the keys of a call are split, and where its workspace's parts are.
struct Kv4Plan {
  int tiles, ns, bps, cnt_stride;
  size_t lse, qp, part_o, part_ml, bytes;  // byte offsets; the counters come first
};

Kv4Plan make_plan(int Hq, int Hkv, int M, int L, bool weigh) {
  Kv4Plan a{};
  const int64_t R = static_cast<int64_t>(Hq / Hkv) * M;
  a.tiles = static_cast<int>((R + kRows - 1) / kRows);
  const int64_t pairs = static_cast<int64_t>(Hkv) * a.tiles;
  const int steps = (L + kKeys * kSplitWaves - 1) / (kKeys * kSplitWaves);
  const int64_t want = std::max<int64_t>(1, kSplitGrid / pairs);
  int ns = static_cast<int>(std::min<int64_t>({want, steps, kMaxSplits}));
  a.cnt_stride = pairs <= 128 ? 128 : 16;
  if (pairs * a.cnt_stride * 4 > BMX_KV4_COUNTER_BYTES) ns = 1;
  a.bps = (steps + ns - 1) / ns;
  a.ns = (steps + a.bps - 1) / a.bps;
  const size_t rows = static_cast<size_t>(Hq) * M;
  size_t at = BMX_KV4_COUNTER_BYTES;
  a.lse = at;
  if (weigh) at += rows * sizeof(float2);
  at = (at + 15) & ~static_cast<size_t>(15);
  a.qp = at;
  if (weigh) at += rows * sizeof(uint4);
  a.part_o = at;
  if (a.ns > 1) at += rows * a.ns * kKv4Dim * sizeof(float);
  a.part_ml = at;
  if (a.ns > 1) at += rows * a.ns * 2 * sizeof(float);
  a.bytes = at;
  return a;
}

// What any call of up to M queries that ends at up to row L needs: with at
// most kSplitGrid workgroups of kRows rows where keys are split at all, the
// partials have a bound that grows with M and L, as the rest does.
size_t plan_bound(int Hq, int M, int L, bool weigh) {
  const size_t rows = static_cast<size_t>(Hq) * M;
  const size_t steps = (static_cast<size_t>(L) + kKeys * kSplitWaves - 1) / (kKeys * kSplitWaves);
  const size_t parts = std::min<size_t>(rows * std::min<size_t>(steps, kMaxSplits), kSplitGrid * kRows);
  return BMX_KV4_COUNTER_BYTES + (weigh ? rows * (sizeof(float2) + sizeof(uint4)) + 16 : 0) +
         parts * (kKv4Dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_attention_kv4_workspace_bytes(int n_heads, int n_kv_heads, int M, int L, int weigh) {
  return attn_shape_ok(n_heads, n_kv_heads, M, L) ? plan_bound(n_heads, M, L, weigh != 0) : 0;
}

extern "C" int bmx_attention_gqa_kv4(const bmx_bf16* q, const bmx_kv4* cache, bmx_bf16* out, float* weights,
                                     int n_heads, int M, int head_dim, int offset, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (int rc = check_kv4("attention_kv4", cache, head_dim)) return rc;
  if (!q || !out || !workspace) return set_error(BMX_E_ARG, "attention_kv4: null pointer");
  const int Hkv = cache->n_kv_heads, L = offset + M;
  if (M < 0 || n_heads <= 0 || n_heads % Hkv)
    return set_error(BMX_E_SHAPE, "attention_kv4: M=%d, %d heads over %d kv heads", M, n_heads, Hkv);
  if (int rc = check_kv4_rows("attention_kv4", cache, M, offset)) return rc;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(weights, 16))
    return set_error(BMX_E_ALIGN, "attention_kv4: q, out, weights and workspace must be 16-byte aligned");
  if (M == 0) return BMX_OK;
  if (!attn_shape_ok(n_heads, Hkv, M, L))
    return set_error(BMX_E_SHAPE, "attention_kv4: %d heads, M=%d too large for one call", n_heads, M);
  const Kv4Plan a = make_plan(n_heads, Hkv, M, L, weights != nullptr);
  const size_t need = plan_bound(n_heads, M, L, weights != nullptr);
  if (workspace_bytes < need || need < a.bytes)
    return set_error(BMX_E_ARG, "attention_kv4: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  char* ws = static_cast<char*>(workspace);
  Kv4AttnParams p{};
  p.q = q;
  p.c = *cache;
  p.out = out;
  p.weights = weights;
  p.cnt = reinterpret_cast<unsigned*>(ws);
  p.lse = weights ? reinterpret_cast<float2*>(ws + a.lse) : nullptr;
  p.qp = weights ? reinterpret_cast<uint4*>(ws + a.qp) : nullptr;
  p.part_o = reinterpret_cast<float*>(ws + a.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + a.part_ml);
  p.Hq = n_heads;
  p.M = M;
  p.offset = offset;
  p.c2 = fabsf(scale) * kLog2e;
  p.flip = scale < 0.0f ? 0x80008000u : 0u;
  p.ns = a.ns;
  p.bps = a.bps;
  p.cnt_stride = a.cnt_stride;
  hipLaunchKernelGGL(kv4_split_kernel<kSplitWaves>, dim3(Hkv, a.ns, a.tiles), dim3(64 * kSplitWaves), 0,
                     as_stream(stream), p);
  if (int rc = check_launch("attention_kv4")) return rc;
  if (!weights) return BMX_OK;
  p.rw = 1;
  while (p.rw < kWeighWaves && p.rw < a.tiles) p.rw *= 2;
  const int keys = kKeys * (kWeighWaves / p.rw);
  if ((L + keys - 1) / keys > 65535) {
    // (fewer key groups: waves do not share keys)
    p.rw = 1;
  }
  const int per = kKeys * (kWeighWaves / p.rw);
  hipLaunchKernelGGL(kv4_weigh_kernel, dim3(Hkv, (L + per - 1) / per), dim3(64 * kWeighWaves), 0, as_stream(stream), p);
  return check_launch("attention_kv4 weights");
}
