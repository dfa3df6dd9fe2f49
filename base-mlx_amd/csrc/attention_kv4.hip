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
// nothing of K is rounded.  For the values (of many rows: at kv4_tile_kernel),
//   sum_j p_j (s n + b)_j = sum_j (p s)_j (16 + n_j) - 16 sum_j p_j s_j + sum_j p_j b_j
// with p s_g, and p where the last two sums are products with rows of scales
// and biases, in two bf16 pieces each: 16 bits, so that the outputs are off by
// their own rounding alone.  (One piece: 0.0018 to 0.0024 of the norm, long
// contexts worst, where the rounding is 0.0017.)
#include <math.h>

#include <algorithm>
#include <type_traits>

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
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

struct Kv4AttnParams {
  const uint16_t* q;  // [Hq, M, 128]
  bmx_kv4 c;
  uint16_t* out;      // [M, Hq*128]
  float* weights;     // [Hkv, cap], or null
  unsigned* cnt;      // arrival counters, kCounterWords apart, zero between calls
  float2* lse;        // [Hq, M] (max * c2, log2 of the sum), or null
  uint4* qp;          // [Hq, M, 17] the queries as the weights' kernel takes them, with lse
  float* part_o;      // [Hq, M, ns, 128]
  float* part_ml;     // [Hq, M, ns, 2]; of kv4_tile_kernel by 32-row tiles, as part_o, and relative to powers of two (log2)
  int Hq, M, offset;
  float c2;           // |scale| log2(e)
  uint32_t flip;      // sign bits of a bf16 pair where scale < 0
  int ns;             // key splits
  int bps;            // steps of all waves per split
  int local;          // every workgroup of a kv head runs on one XCD (shares its L2)
  float* sums;        // [row ranges, Hkv, L] of the weights
};

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}

__device__ __forceinline__ f32x16_t mfma32_f16(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}

// The wave's number as a scalar, so branches on it cost no lane masks
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// All weights hold a factor 2^-28 where they are summed up, which the division
// by their sum takes out again: 2^24 rows of values of 2^120, whose sums of
// p s (16 + n) are 2^122 each, at a weight of 2^8 (see moves) stay below 2^127.
// A weight below 2^-88 of the largest loses the second of its bf16 pieces, one
// below 2^-98 is 0.
constexpr float kDown = 28.0f;

// Whether a running maximum m moves to its step's maximum bm: only where the
// weights exp2((bm - m) c2) would pass 2^8.  Until then m stays, P goes up to
// 2^8, and the products so far need no rescaling.
__device__ __forceinline__ bool moves(float bm, float m, float c2) { return bm > m && !((bm - m) * c2 <= 8.0f); }

// The masks of the nibble pairs, held in registers (a gfx9 and-or takes no
// literal)
struct PairK {
  uint32_t mask, one;
  __device__ __forceinline__ PairK() : mask(0x00780078u), one(0x41804180u) { asm volatile("" : "+v"(mask), "+v"(one)); }
};
struct PairH {  // ... of fp16 1024 + n
  uint32_t mask, one;
  __device__ __forceinline__ PairH() : mask(0x000f000fu), one(0x64006400u) { asm volatile("" : "+v"(mask), "+v"(one)); }
};
__device__ __forceinline__ f16x2_t half2(uint32_t x) { return __builtin_bit_cast(f16x2_t, x); }
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
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {  // one v_cvt_pk_bf16_f32
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}
__device__ __forceinline__ uint32_t dpp_ror8(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x128, 0xF, 0xF, true));
}
// Whether one of a row's two scales (or biases) is infinite or NaN
__device__ __forceinline__ bool not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
// Keeps what is done to x in a seldom taken branch there: without, the compiler
// does it always and selects
__device__ __forceinline__ void stay_here(float& x) { asm volatile("" : "+v"(x)); }
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

// Partials travel between workgroups, in general on different XCDs: agent-scope
// stores (written through to memory), complete before the arrival, and loads
// with sc1 after it.  Where all workgroups of a kv head share an XCD, plain
// stores and L2 increments, and loads with sc0 (past the L1) do; the counter
// is another word then, 256 bytes on, so that a line is only ever updated in
// one place.
constexpr int kAgentCoherent = 16, kL2Coherent = 1;
constexpr int kLocalCounter = 64;  // words into a counter's 512 bytes
constexpr int kCounterWords = 128, kMaxCounters = BMX_KV4_COUNTER_BYTES / (4 * kCounterWords);
__device__ __forceinline__ void store_part(float* p, float x, float y) {
  const uint64_t v = static_cast<uint64_t>(__float_as_uint(x)) | (static_cast<uint64_t>(__float_as_uint(y)) << 32);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {  // round to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}

// Q_0 and Q_1 of a query row, each in three bf16 pieces that add up to it
__device__ __forceinline__ u32x4_t q_pieces(const float (&qs)[2]) {
  const float h0 = round_bf(qs[0]), h1 = round_bf(qs[1]);
  const float m0 = round_bf(qs[0] - h0), m1 = round_bf(qs[1] - h1);
  return u32x4_t{pack_bf(h0, h1), pack_bf(m0, m1), pack_bf(qs[0] - h0 - m0, qs[1] - h1 - m1), 0u};
}
// ... kept for the weights with the row's fragments, in the order their
// lanes g take them: 64 bytes per g, then the pieces (17 words of 16 bytes)
constexpr int kQueryWords = 17;
__device__ __forceinline__ void store_query(const Kv4AttnParams& p, int64_t row, int g, const u32x4_t (&qf)[2][2],
                                            const float (&qs)[2]) {
  u32x4_t* dst = reinterpret_cast<u32x4_t*>(p.qp) + row * kQueryWords;
#pragma unroll
  for (int k = 0; k < 4; k++) dst[4 * g + k] = qf[k >> 1][k & 1];
  if (g == 0) dst[16] = q_pieces(qs);
}

// One output row's 4 dims, and the row's softmax statistics for the weights;
// o and l hold the factor 2^-28.
__device__ __forceinline__ void finish_row(const Kv4AttnParams& p, int kvh, int r, int d, float4 o, float m, float l) {
  const int rep = p.Hq / p.c.n_kv_heads, t = r % p.M, h = kvh * rep + r / p.M;
  const float inv = 1.0f / l;
  *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(t) * p.Hq + h) * kKv4Dim + d) =
      make_uint2(pack_bf(o.x * inv, o.y * inv), pack_bf(o.z * inv, o.w * inv));
  if (p.lse && d == 0) p.lse[static_cast<int64_t>(kvh) * rep * p.M + r] = make_float2(m, log2f(l) + kDown);
}

template <int NW, int ROWS>
struct JoinLds {
  alignas(16) float os[NW][ROWS][kOs];
  float ms[NW][ROWS], ls[NW][ROWS], wt[ROWS][kMaxSplits], fin[ROWS][2];
  int last;
};

// Rows r0 .. r0 + RT - 1 from their splits' partials, by one workgroup; AUX:
// the cache policy of the loads.
template <int NW, int ROWS, int AUX>
__device__ __forceinline__ void merge_splits(const Kv4AttnParams& p, JoinLds<NW, ROWS>& sm, int kvh, int r0, int RT) {
  constexpr int kThreads = 64 * NW, kAhead = 8;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63;
  const int64_t row0 = static_cast<int64_t>(kvh) * (p.Hq / p.c.n_kv_heads) * p.M + r0;
  const __amdgpu_buffer_rsrc_t rml =
      rsrc(reinterpret_cast<const uint32_t*>(p.part_ml), row0 * p.ns * 2, RT * p.ns * 8);
  const __amdgpu_buffer_rsrc_t ro =
      rsrc(reinterpret_cast<const uint32_t*>(p.part_o), row0 * p.ns * kKv4Dim, RT * p.ns * kKv4Dim * 4);
  // (row, 4 dims) per thread, the splits n, n + groups, .. over as many threads
  // as there are; this thread's first eight are on their way while the splits'
  // weights are formed
  const int items = RT * 32, groups = max(1, kThreads / items), n = tid / items;
  auto load_o = [&](int it, int s) {
    return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                           ro, (((it >> 5) * p.ns + s) * kKv4Dim + 4 * (it & 31)) * 4, 0, AUX));
  };
  // a wave per row, a lane per split
  f32x2_t ml = {-INFINITY, 0.0f};
  int r = wave;
  auto load_ml = [&]() {
    return __builtin_bit_cast(f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rml, (r * p.ns + min(lane, p.ns - 1)) * 8, 0, AUX));
  };
  if (r < RT) ml = load_ml();
  int it = tid - n * items;
  f32x4_t ahead[kAhead];
  if (it < items && n < groups) {
#pragma unroll
    for (int k = 0; k < kAhead; k++) ahead[k] = load_o(it, min(n + k * groups, p.ns - 1));
  }
  while (r < RT) {
    const float m = lane < p.ns ? ml.x : -INFINITY;
    const float mm = max_xor32(max_xor16(row16_max(m)));
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mm) * p.c2);
    const float sum = lanes_sum(lane < p.ns ? f * ml.y : 0.0f, 64);
    sm.wt[r][lane] = f;
    if (lane == 0) {
      sm.fin[r][0] = mm;
      sm.fin[r][1] = sum;
    }
    r += NW;
    if (r < RT) ml = load_ml();
  }
  __syncthreads();
  float* red = &sm.os[0][0][0];
  for (bool first = true; it < items && n < groups; it += kThreads, first = false) {
    const int row = it >> 5, d = 4 * (it & 31);
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!first) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) ahead[k] = load_o(it, min(n + k * groups, p.ns - 1));
    }
    int s = n;
#pragma unroll
    for (int k = 0; k < kAhead; k++, s += groups)
      if (s < p.ns) o += sm.wt[row][s] * ahead[k];
#pragma unroll 8
    for (; s < p.ns; s += groups) o += sm.wt[row][s] * load_o(it, s);
    if (groups == 1)
      finish_row(p, kvh, r0 + row, d, make_float4(o[0], o[1], o[2], o[3]), sm.fin[row][0] * p.c2,
                 sm.fin[row][1]);
    else
      *reinterpret_cast<f32x4_t*>(&red[(n * items + it) * 4]) = o;
  }
  if (groups == 1) return;
  __syncthreads();
  for (int k = tid; k < items; k += kThreads) {
    f32x4_t o = *reinterpret_cast<const f32x4_t*>(&red[k * 4]);
    for (int i = 1; i < groups; i++) o += *reinterpret_cast<const f32x4_t*>(&red[(i * items + k) * 4]);
    finish_row(p, kvh, r0 + (k >> 5), 4 * (k & 31), make_float4(o[0], o[1], o[2], o[3]),
               sm.fin[k >> 5][0] * p.c2, sm.fin[k >> 5][1]);
  }
}

// The end of a workgroup: each wave hands in, for row li of the tile (lanes
// li < ROWS), its maximum m and sum l over its keys, and in lane (li, g) the
// products acc[y][nibble][i] of the dims described at the kernel, to which
// x[y] adds.
template <int NW, int ROWS>
__device__ __forceinline__ void join_and_finish(const Kv4AttnParams& p, JoinLds<NW, ROWS>& sm, int kvh, int split,
                                                int r0, int RT, float m, float l, const f32x4_t (&acc)[2][4],
                                                const float (&x)[2]) {
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int64_t row0 = static_cast<int64_t>(kvh) * (p.Hq / p.c.n_kv_heads) * p.M + r0;
  // ---- the waves' sums joined: weights exp2((m_w - m) c2) ----
  if (l != l) m = l;  // a NaN score: the row stays NaN
  if (g == 0 && li < ROWS) {
    sm.ms[wave][li] = m;
    sm.ls[wave][li] = l;
  }
  __syncthreads();
  if (li < ROWS) {
    float mm = sm.ms[0][li];
#pragma unroll
    for (int w = 1; w < NW; w++) mm = fmaxf(mm, sm.ms[w][li]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mm) * p.c2);
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int a = 4 * g + i;  // row of A: word a % 8, half a / 8
        *reinterpret_cast<float4*>(&sm.os[wave][li][64 * y + 8 * (a & 7) + 4 * (a >> 3)]) =
            make_float4((acc[y][0][i] + x[y]) * f, (acc[y][1][i] + x[y]) * f, (acc[y][2][i] + x[y]) * f,
                        (acc[y][3][i] + x[y]) * f);
      }
  }
  __syncthreads();
  for (int it = tid; it < RT * 32; it += 64 * NW) {
    const int r = it >> 5, d = 4 * (it & 31);
    float mm = sm.ms[0][r];
#pragma unroll
    for (int w = 1; w < NW; w++) mm = fmaxf(mm, sm.ms[w][r]);
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = sm.ms[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((sm.ms[w][r] - mm) * p.c2);
      sum = __builtin_fmaf(f, sm.ls[w][r], sum);
      const float4 v = *reinterpret_cast<const float4*>(&sm.os[w][r][d]);
      o.x += v.x;
      o.y += v.y;
      o.z += v.z;
      o.w += v.w;
    }
    if (sum != sum) mm = sum;
    if (p.ns == 1) {
      finish_row(p, kvh, r0 + r, d, o, mm * p.c2, sum);
    } else {
      const int64_t at = (row0 + r) * p.ns + split;
      if (p.local) {
        *reinterpret_cast<float4*>(p.part_o + at * kKv4Dim + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mm, sum);
      } else {
        store_part(p.part_o + at * kKv4Dim + d, o.x, o.y);
        store_part(p.part_o + at * kKv4Dim + d + 2, o.z, o.w);
        if (d == 0) store_part(p.part_ml + at * 2, mm, sum);
      }
    }
  }
  if (p.ns == 1) return;

  // ---- the last workgroup of a (kv head, row tile) merges its splits ----
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    unsigned* c = p.cnt + (static_cast<int64_t>(blockIdx.z) * gridDim.x + kvh) * kCounterWords;
    unsigned n;
    if (p.local) {
      c += kLocalCounter;
      n = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    } else {
      n = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    sm.last = n == static_cast<unsigned>(p.ns - 1);
    if (sm.last) {
      // (subtracted rather than stored: performed where the additions are)
      if (p.local) __hip_atomic_fetch_sub(c, static_cast<unsigned>(p.ns), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      else __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (!sm.last) return;
  if (p.local) merge_splits<NW, ROWS, kL2Coherent>(p, sm, kvh, r0, RT);
  else merge_splits<NW, ROWS, kAgentCoherent>(p, sm, kvh, r0, RT);
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
// Bound by instruction issue: a step takes about 370 VALU instructions and 28
// products, which hardly overlap (64 tokens over 4064 rows, 32 heads of 8: 21
// us; with one piece of p s and p, 60 instructions and 7 products less, 19).
// Two row tiles per wave, to share the 180 that nibbles and scales take, spilled
// registers and were no faster.
template <int NW>
__global__ void __launch_bounds__(64 * NW) kv4_rows_kernel(const Kv4AttnParams p) {
  __shared__ JoinLds<NW, kRows> sm;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, split = blockIdx.y, r0 = blockIdx.z * kRows;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, RT = min(kRows, R - r0), L = p.offset + M;
  const int64_t row0 = static_cast<int64_t>(kvh) * R + r0;
  // rows' tokens: a query sees keys < lim; the tile's first and last token
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
  float start[2];  // -16 Q_y of the query
  u32x4_t qp;      // lanes g = 0: Q_0, Q_1 in three bf16 pieces each
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
      start[y] = -16.0f * qs[y];
    }
    if (p.qp && split == 0 && wave == 0 && li < RT) store_query(p, row0 + li, g, qf, qs);
    qp = q_pieces(qs);
    if (g != 0) qp = u32x4_t{0u, 0u, 0u, 0u};
  }

  const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
  // edge: rows 0, 1 sum p b, rows 2, 3 sum p s of groups 0, 1
  f32x4_t acc[2][4], edge = zero;
#pragma unroll
  for (int y = 0; y < 2; y++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[y][i] = zero;
  float m = -INFINITY, l = 0.0f, slow[2] = {0.0f, 0.0f};
  const uint32_t half_sel = li < 8 ? 0x01000504u : 0x07060302u;
  // (selector 0x0c gives a zero byte: rows from 4 on take nothing)
  const uint32_t odd_sel = li >= 4 ? 0x0c0c0c0cu : li & 1 ? 0x07060302u : 0x05040100u;

  auto step = [&](auto cut_) {
    constexpr bool cut = decltype(cut_)::value;  // some row does not see some key
    // ---- scores ----
    float sc[8];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f32x4_t d0 = {start[0], start[0], start[0], start[0]}, d1 = {start[1], start[1], start[1], start[1]};
#pragma unroll
      for (int e = 0; e < 2; e++) {
        d0 = mfma(word_pairs(kw[t][0][e], nk), qf[0][e], d0);
        d1 = mfma(word_pairs(kw[t][1][e], nk), qf[1][e], d1);
      }
      const f32x4_t db = mfma(u32x4_t{kb[t], kb[t], kb[t], kb[t]}, qp, zero);
#pragma unroll
      for (int i = 0; i < 4; i++)
        sc[4 * t + i] = __builtin_fmaf(lo_f(ks[t][i]), d0[i], __builtin_fmaf(hi_f(ks[t][i]), d1[i], db[i]));
    }
    // An infinite scale that meets a product of the other sign gives -infinity,
    // as a hidden row's score; it is NaN instead.  (An infinite bias always is:
    // it also meets the zeros of qp.)
    float least = sc[0];
#pragma unroll
    for (int e = 1; e < 8; e++) least = fminf(least, sc[e]);
    if (__any(least == -INFINITY)) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        stay_here(sc[e]);
        if (not_finite(ks[e >> 2][e & 3])) sc[e] = NAN;
      }
    }
    load_k(b + NW);
    // ---- running softmax: the maximum over all keys of a query ----
    const int key0 = b * kKeys + 4 * g;
    u32x4_t pb[2][2], pt[2];  // [group][piece], [piece]
    bool odd = false;
    u32x4_t bw[2];
    if constexpr (cut) {
      // rows that a query does not see weigh nothing in it, whatever their
      // scales and biases are: its P V column has zeros for them, and biases
      // that are not finite go to the lanes' own sums of the rows that see
      // them, not into the product that every query shares
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
    }
    if constexpr (cut) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (key0 + (e & 3) + 16 * (e >> 2) >= lim) sc[e] = -INFINITY;
    }
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < 8; e++) bm = fmaxf(bm, sc[e]);
    bm = max_xor32(max_xor16(bm));
    if (__any(moves(bm, m, p.c2))) {
      const float mn = fmaxf(m, bm);
      const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * p.c2);
      m = mn;
      l *= a;
      edge *= a;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        slow[y] *= a;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[y][i] *= a;
      }
    }
    const float mc = m == -INFINITY ? kDown : __builtin_fmaf(m, p.c2, kDown);
    float pr[8], ps[2][8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      pr[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], p.c2, -mc));
      ps[0][e] = pr[e] * lo_f(vs[e >> 2][e & 3]);
      ps[1][e] = pr[e] * hi_f(vs[e >> 2][e & 3]);
      if constexpr (cut) {
        const bool seen = key0 + (e & 3) + 16 * (e >> 2) < lim;
        if (!seen) pr[e] = ps[0][e] = ps[1][e] = 0.0f;
        if (odd && seen) {
          slow[0] += lo_f(bw[e >> 2][e & 3]) * 0.0f;  // 0 or NaN
          slow[1] += hi_f(bw[e >> 2][e & 3]) * 0.0f;
        }
      }
    }
    l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
#pragma unroll
    for (int j = 0; j < 4; j++) {
      auto pieces = [](float a, float b, uint32_t& hi, uint32_t& lo) {
        hi = pack_bf(a, b);
        lo = pack_bf(a - lo_f(hi), b - hi_f(hi));
      };
      uint32_t hi, lo;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        pieces(ps[y][2 * j], ps[y][2 * j + 1], hi, lo);
        pb[y][0][j] = hi;
        pb[y][1][j] = lo;
      }
      pieces(pr[2 * j], pr[2 * j + 1], hi, lo);
      pt[0][j] = hi;
      pt[1][j] = lo;
    }
    // ---- P V ----
#pragma unroll
    for (int y = 0; y < 2; y++) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = __builtin_amdgcn_perm(vw[y][j], dpp_ror8(vw[y][j]), half_sel);
      const u32x4_t a[4] = {
          {nibble_pair<0>(v[0], nk), nibble_pair<0>(v[1], nk), nibble_pair<0>(v[2], nk), nibble_pair<0>(v[3], nk)},
          {nibble_pair<1>(v[0], nk), nibble_pair<1>(v[1], nk), nibble_pair<1>(v[2], nk), nibble_pair<1>(v[3], nk)},
          {nibble_pair<2>(v[0], nk), nibble_pair<2>(v[1], nk), nibble_pair<2>(v[2], nk), nibble_pair<2>(v[3], nk)},
          {nibble_pair<3>(v[0], nk), nibble_pair<3>(v[1], nk), nibble_pair<3>(v[2], nk), nibble_pair<3>(v[3], nk)}};
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[y][i] = mfma(a[i], pb[y][k], acc[y][i]);
    }
    {
      // rows 0..3 of A: b_0, b_1, s_0, s_1 of the step's keys
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
#pragma unroll
      for (int k = 0; k < 2; k++) edge = mfma(a, pt[k], edge);
    }
    load_v(b + NW);
  };
  // the steps whose keys every row sees, then the others
  const int b_full = min(b_end, all_see / kKeys);
  for (; b < b_full; b += NW) step(std::false_type{});
  for (; b < b_end; b += NW) step(std::true_type{});

  float x[2];  // what every dim of a group gets besides its product
#pragma unroll
  for (int y = 0; y < 2; y++)
    x[y] = __builtin_fmaf(-16.0f, __shfl(edge[2 + y], li, 64), __shfl(edge[y], li, 64)) + add_xor32(add_xor16(slow[y]));
  join_and_finish<NW, kRows>(p, sm, kvh, split, r0, RT, m, add_xor32(add_xor16(l)), acc, x);
}

// Up to RC = 4 or 8 query rows.  The scores of T = 16 / RC key tiles share one
// 16 x 16 result: column li is query li % RC over tile li / RC, so a lane
// holds 4 scores of a step of 16 T keys, for as many keys' scales, where the
// kernel above would hold 4 T with most of them for no query.  Every tile is
// multiplied with all 16 columns (the queries RC by RC again) and each lane
// takes the result of its tile; P goes back as a B operand with zeros where a
// column's tile is not the product's, two tiles to a product.  The columns of
// a query are added at the end.  The sums over a lane's own keys that take s
// and b (see the top) are fp32 here.  The second piece of p s takes 1 % of the
// time over 4097 rows, 3 % over 131072.
// One token over 131072 rows, 32 heads of 8: 33 us, 4.6 TB/s, where the kernel
// above took 44 with one piece.
template <int RC, int NW>
__global__ void __launch_bounds__(64 * NW) kv4_few_kernel(const Kv4AttnParams p) {
  constexpr int T = 16 / RC, kStep = 16 * T;
  __shared__ JoinLds<NW, RC> sm;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int qi = li % RC, blk = li / RC;
  const int kvh = blockIdx.x, split = blockIdx.y;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, L = p.offset + M;
  const int64_t row0 = static_cast<int64_t>(kvh) * R;
  const int lim = p.offset + min(qi, R - 1) % M + 1;
  const PairK nk;

  const int64_t slot = static_cast<int64_t>(kvh) * p.c.capacity;
  const __amdgpu_buffer_rsrc_t kwr = rsrc(p.c.k, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t vwr = rsrc(p.c.v, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t ksr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t kbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_biases), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vsr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_biases), slot, L * 4);

  u32x2_t kw[T][2];        // [tile][group]: words of key li
  uint32_t vw[T / 2][2][4];  // [tile pair][group][key pair]
  u32x4_t ks, kb, vs, vb;  // the lane's 4 keys: 16 blk + 4g ..
  auto load_k = [&](int b) {
    const int w = (b * kStep + li) * 64 + 8 * g, s = (b * kStep + 16 * blk + 4 * g) * 4;
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
      for (int y = 0; y < 2; y++) kw[t][y] = load2(kwr, w + t * 1024 + y * 32);
    ks = load4(ksr, s);
    kb = load4(kbr, s);
  };
  auto load_v = [&](int b) {
    const int w = (b * kStep + 4 * g + (li >> 3)) * 64 + 4 * (li & 7), s = (b * kStep + 16 * blk + 4 * g) * 4;
#pragma unroll
    for (int u = 0; u < T / 2; u++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int y = 0; y < 2; y++)
          vw[u][y][j] = load1(vwr, w + (32 * u + (j & 1) * 2 + (j >> 1) * 16) * 64 + y * 32);
    vs = load4(vsr, s);
    vb = load4(vbr, s);
  };

  const int b_end = min((L + kStep - 1) / kStep, (split + 1) * p.bps * NW);
  int b = split * p.bps * NW + wave;
  load_k(b);
  load_v(b);

  u32x4_t qf[2][2];
  float qs[2];  // Q_y of query qi
  {
    const uint16_t* qr = p.q + (row0 + min(qi, R - 1)) * kKv4Dim + 16 * g;
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
    }
    if (p.qp && split == 0 && wave == 0 && li < R) store_query(p, row0 + li, g, qf, qs);
  }
  const float st[2] = {-16.0f * qs[0], -16.0f * qs[1]};

  f32x4_t acc[2][4];
#pragma unroll
  for (int y = 0; y < 2; y++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[y][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f, add[2] = {0.0f, 0.0f};
  const uint32_t half_sel = li < 8 ? 0x01000504u : 0x07060302u;

  auto step = [&](auto cut_) {
    constexpr bool cut = decltype(cut_)::value;
    f32x4_t d0[T], d1[T];
#pragma unroll
    for (int t = 0; t < T; t++) {
      const f32x4_t s0 = {st[0], st[0], st[0], st[0]}, s1 = {st[1], st[1], st[1], st[1]};
      d0[t] = mfma(word_pairs(kw[t][0].x, nk), qf[0][0], s0);
      d1[t] = mfma(word_pairs(kw[t][1].x, nk), qf[1][0], s1);
      d0[t] = mfma(word_pairs(kw[t][0].y, nk), qf[0][1], d0[t]);
      d1[t] = mfma(word_pairs(kw[t][1].y, nk), qf[1][1], d1[t]);
    }
#pragma unroll
    for (int n = 1; n < T; n *= 2)  // the lane's tile
#pragma unroll
      for (int t = 0; t < T; t += 2 * n)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          d0[t][i] = blk & n ? d0[t + n][i] : d0[t][i];
          d1[t][i] = blk & n ? d1[t + n][i] : d1[t][i];
        }
    float sc[4], pr[4], ps[2][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      sc[i] = __builtin_fmaf(lo_f(kb[i]), qs[0], hi_f(kb[i]) * qs[1]);
      sc[i] = __builtin_fmaf(lo_f(ks[i]), d0[0][i], __builtin_fmaf(hi_f(ks[i]), d1[0][i], sc[i]));
    }
    // an infinite scale or bias must not make its key's score -infinity, as a
    // hidden row's
    if (__any(fminf(fminf(sc[0], sc[1]), fminf(sc[2], sc[3])) == -INFINITY)) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        stay_here(sc[i]);
        if (not_finite(ks[i]) || not_finite(kb[i])) sc[i] = NAN;
      }
    }
    load_k(b + NW);
    const int key0 = b * kStep + 16 * blk + 4 * g;
    if constexpr (cut) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (key0 + i >= lim) sc[i] = -INFINITY;
    }
    float bm = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
    if constexpr (RC == 4) bm = fmaxf(bm, dpp_f32<0x124>(bm));
    bm = fmaxf(bm, dpp_f32<0x128>(bm));
    bm = max_xor32(max_xor16(bm));
    if (__any(moves(bm, m, p.c2))) {
      const float mn = fmaxf(m, bm);
      const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * p.c2);
      m = mn;
      l *= a;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        add[y] *= a;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[y][i] *= a;
      }
    }
    const float mc = m == -INFINITY ? kDown : __builtin_fmaf(m, p.c2, kDown);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      pr[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], p.c2, -mc));
      ps[0][i] = pr[i] * lo_f(vs[i]);
      ps[1][i] = pr[i] * hi_f(vs[i]);
    }
    // rows that a query does not see weigh nothing in it, whatever their
    // scales and biases are
    float mid[2][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      mid[0][i] = __builtin_fmaf(-16.0f, ps[0][i], pr[i] * lo_f(vb[i]));
      mid[1][i] = __builtin_fmaf(-16.0f, ps[1][i], pr[i] * hi_f(vb[i]));
      if constexpr (cut) {
        if (key0 + i >= lim) pr[i] = ps[0][i] = ps[1][i] = mid[0][i] = mid[1][i] = 0.0f;
      }
    }
    l += (pr[0] + pr[1]) + (pr[2] + pr[3]);
    uint32_t pb[2][2][2];  // [group][piece]
#pragma unroll
    for (int y = 0; y < 2; y++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        pb[y][0][j] = pack_bf(ps[y][2 * j], ps[y][2 * j + 1]);
        pb[y][1][j] = pack_bf(ps[y][2 * j] - lo_f(pb[y][0][j]), ps[y][2 * j + 1] - hi_f(pb[y][0][j]));
      }
      add[y] += (mid[y][0] + mid[y][1]) + (mid[y][2] + mid[y][3]);
    }
#pragma unroll
    for (int u = 0; u < T / 2; u++)
#pragma unroll
      for (int y = 0; y < 2; y++) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __builtin_amdgcn_perm(vw[u][y][j], dpp_ror8(vw[u][y][j]), half_sel);
        const u32x4_t a[4] = {
            {nibble_pair<0>(v[0], nk), nibble_pair<0>(v[1], nk), nibble_pair<0>(v[2], nk), nibble_pair<0>(v[3], nk)},
            {nibble_pair<1>(v[0], nk), nibble_pair<1>(v[1], nk), nibble_pair<1>(v[2], nk), nibble_pair<1>(v[3], nk)},
            {nibble_pair<2>(v[0], nk), nibble_pair<2>(v[1], nk), nibble_pair<2>(v[2], nk), nibble_pair<2>(v[3], nk)},
            {nibble_pair<3>(v[0], nk), nibble_pair<3>(v[1], nk), nibble_pair<3>(v[2], nk), nibble_pair<3>(v[3], nk)}};
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const u32x4_t pv = {blk == 2 * u ? pb[y][k][0] : 0u, blk == 2 * u ? pb[y][k][1] : 0u,
                              blk == 2 * u + 1 ? pb[y][k][0] : 0u, blk == 2 * u + 1 ? pb[y][k][1] : 0u};
#pragma unroll
          for (int i = 0; i < 4; i++) acc[y][i] = mfma(a[i], pv, acc[y][i]);
        }
      }
    load_v(b + NW);
  };
  const int b_full = min(b_end, (p.offset + 1) / kStep);  // every row sees keys 0 .. offset
  for (; b < b_full; b += NW) step(std::false_type{});
  for (; b < b_end; b += NW) step(std::true_type{});

  // the columns of a query together
  auto columns = [&](float v) {
    if constexpr (RC == 4) v += dpp_f32<0x124>(v);
    return v + dpp_f32<0x128>(v);
  };
  float x[2];
#pragma unroll
  for (int y = 0; y < 2; y++) {
    x[y] = add_xor32(add_xor16(columns(add[y])));
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[y][i][e] = columns(acc[y][i][e]);
  }
  join_and_finish<NW, RC>(p, sm, kvh, split, 0, R, m, add_xor32(add_xor16(columns(l))), acc, x);
}

__device__ __forceinline__ u32x4_t lds_read(const uint16_t* p) { return *reinterpret_cast<const u32x4_t*>(p); }
// Reads before it stay before it, and so ahead of the branches that follow
__device__ __forceinline__ void reads_go_out() { asm volatile("" ::: "memory"); }

constexpr float kFloatMax = 3.402823466e38f;
// The largest magnitude that values of scale s and bias b may have (not a
// finite number where the scale or bias is not)
__device__ __forceinline__ float kv4_most(float s, float b) {
  const float end = fabsf(__builtin_fmaf(15.0f, s, b));
  return end <= kFloatMax ? fmaxf(end, fabsf(b)) : end;
}
__device__ __forceinline__ bool kv4_finite(float s, float b) { return kv4_most(s, b) <= kFloatMax; }

// Many query rows: 32 RW of one kv head per workgroup of 8 waves, wave w with
// rows 32 (w % RW) ..; the waves that share rows take different key tiles of
// 32.  An iteration's keys are unpacked once, by all waves, into LDS (two
// buffers: the next iteration's while this one's are multiplied), so the
// nibbles cost a row tile 1 / RW of what they cost above.
//   K as 16 + n in the pair order of a word, [key][128], rows 272 bytes
//   apart; scores by v_mfma_f32_32x32x16_bf16, transposed: lane (query
//   l % 32, h = l / 32) holds keys 8 j + 4 h + i.  One more product adds
//   b_g Q_g - 16 s_g Q_g: its k index runs over biases (lanes h = 0) and
//   scales (h = 1), each against the three pieces of Q_0 and Q_1.
//   V as fp16 (s n + b) 2^(15 - e), 2^e the power of two above the key's
//     values, transposed: [dim][key], the keys of a half tile in the order the
//     score lanes hold them (16 k + 4 h + i, 16 k + 8 + 4 h + i), so P is its
//     own B operand.  Two iterations ahead a lane per key finds e and turns s
//     and b into fp16 (exactly: 8 bits); a pair of values is then a packed
//     subtraction and a packed multiply-add, which rounds once.
// The softmax runs over t = S c2 + e, so P = 2^(t - M) times V 2^-e needs no
// further scaling, and what a key's values weigh, not only its score, decides
// what may round away.  The product that adds the biases adds e and -M too, M
// in three bf16 pieces; M moves only where P would pass 2^15, to make the
// largest 2^7.  The sum of the weights is that of P 2^(15 - e), so e of the
// keys that weigh anything must lie within 2^80 of each other: not below -48,
// and where a key's is above 32 the rows that see it are computed again, by a
// wide pass with a sum, and a maximum, of the scores alone, and P and V of each
// group by the group's own e.  So are rows that see a key whose groups are more
// than 2^6 apart: in the smaller one P 2^-25 of the largest, which is 2^7 at
// least and belongs to the other, would vanish, a part of N 2^-26 at most with
// N keys.  (Three exponentials per score; no other row's bits change.)  A row
// leaves with its weights' exponent taken out, so that splits are joined by what
// they weigh.  With 11 bits in P and V the outputs are off by little more than
// their own rounding: 0.0017 of the norm for 2048 tokens over 4096 rows, where
// bf16 for both gave 0.0028.
// 2048 tokens over 4096 rows, 32 heads of 8: 149 us, 692 TFLOP/s, 54 % of what
// a large matrix product reaches (347 us where every row takes the wide pass,
// too).  A tile of 32 x 32 takes 17 products of 32 cycles and about 150 VALU
// instructions of 4 with its share of the unpacking, 16 of them exponentials of
// 16: the two hardly overlap, so the VALU work is half the time.  Rates of the
// counters: matrix cores busy 35 %, VALU 44 %, LDS 43 %, 1 / 9 of that in bank
// conflicts.
// A value that is not finite (its scale or bias is not) goes to LDS as 0 and
// marks the iteration, as a key's scale or bias that is not finite does; the
// rows that see it become NaN by themselves.
template <int RW>
__global__ void __launch_bounds__(512) kv4_tile_kernel(const Kv4AttnParams p) {
  constexpr int KW = 8 / RW, TPW = RW == 8 ? 2 : 1, KPI = kKeys * KW * TPW;
  constexpr int W = KPI / 32;     // words of K per thread
  constexpr int VJ = KPI / 64;    // (quad of keys, half word) jobs of V per thread
  constexpr int KS = kKv4Dim + 8;
  struct Stage {
    alignas(16) uint16_t kt[KPI][KS];
    alignas(16) uint16_t vt[kKv4Dim][KPI];
    alignas(16) uint32_t sb[2][KPI];  // K's biases, scales
    alignas(16) float sf[2][KPI];     // the scales of group 0, group 1, times c2
  };
  struct Join {
    alignas(16) float os[4][kKeys][kOs];
    float ms[4][kKeys], ls[4][kKeys];
  };
  constexpr size_t kLds = sizeof(Stage) * 2 > sizeof(Join) ? sizeof(Stage) * 2 : sizeof(Join);
  __shared__ __align__(16) char lds[kLds];
  // of four iterations in turn: whether some key or value is not finite, the
  // keys' 2^(15 - e), e (wide pass: e of group 0, of group 1)
  __shared__ int mark[4];
  __shared__ int first_wide;  // the first key whose values the plain pass does not serve
  __shared__ __align__(16) float vscale[4][KPI];
  __shared__ __align__(16) uint32_t ve[4][KPI];
  __shared__ __align__(16) uint16_t vsb[4][2][2][KPI];  // ... scales, biases of group 0, 1, times 2^(15 - e), as fp16
  Stage* const st = reinterpret_cast<Stage*>(lds);
  Join& jn = *reinterpret_cast<Join*>(lds);
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, lr = lane & 31, h = lane >> 5;
  const int rwi = wave % RW, kwi = wave / RW;
  const int kvh = blockIdx.x, split = blockIdx.y;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, L = p.offset + M;
  // the 32-row tile of wave number i: with 8, spread over the rows, so that
  // the two waves of a SIMD (and so all workgroups) see about as many keys
  // together, however the causal mask cuts them
  const int z = blockIdx.z, zs = gridDim.z;
  auto tile_of = [&](int i) {
    if constexpr (RW < 8) return z * RW + i;
    const int o = i < 4 ? i : 11 - i;
    return o * zs + (o & 1 ? zs - 1 - z : z);
  };
  // keys that any row of a tile sees
  auto end_of = [&](int first, int rows) {
    const int t0 = first % M;
    return p.offset + (t0 + rows > M ? M - 1 : t0 + rows - 1) + 1;
  };
  const int rw0 = kKeys * tile_of(rwi), n = min(kKeys, R - rw0);  // first row, rows (n <= 0: none)
  const int64_t row0 = static_cast<int64_t>(kvh) * R;
  const int row = min(rw0 + lr, R - 1);
  const int lim = p.offset + row % M + 1;
  int all_see = 0, kend = 0;  // keys that every row, any row of the wave sees
  if (n > 0) {
    const int t0 = rw0 % M;
    all_see = p.offset + (t0 + n > M ? 0 : t0) + 1;
    kend = end_of(rw0, n);
  }
  int kend_wg = 0;
  for (int i = 0; i < RW; i++) {
    const int first = kKeys * tile_of(i);
    if (first < R) kend_wg = max(kend_wg, end_of(first, min(kKeys, R - first)));
  }
  const PairK nk;
  const PairH hk;

  const int64_t slot = static_cast<int64_t>(kvh) * p.c.capacity;
  const __amdgpu_buffer_rsrc_t kwr = rsrc(p.c.k, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t vwr = rsrc(p.c.v, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t ksr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t kbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_biases), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vsr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t vbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.v_biases), slot, L * 4);

  // The 16-byte pieces of V's row d stand at their number xor this: different
  // banks for the 16 rows that a read takes together (bits 0 .. 3 of d) and
  // the rows 4 apart of a write (bits 2 .. 4)
  auto swizzle = [](int d) { return (((d >> 1) & 7) ^ ((d >> 4) & 1)) | (KPI == 128 ? (d & 1) << 3 : 0); };

  // ---- staging: this thread's part of an iteration ----
  uint32_t gk[W], gsb = 0;
  uint32_t gv[VJ][4];
  const int k_key = tid / (16 / W), k_word = W * (tid % (16 / W));
  auto fetch = [&](int it) {
    const int key0 = it * KPI;
    if constexpr (W == 2) {
      const u32x2_t w = load2(kwr, (key0 + k_key) * 64 + 4 * k_word);
      gk[0] = w.x;
      gk[1] = w.y;
    } else {
      const u32x4_t w = load4(kwr, (key0 + k_key) * 64 + 4 * k_word);
#pragma unroll
      for (int i = 0; i < W; i++) gk[i] = w[i];
    }
    if (tid < 2 * KPI) gsb = tid < KPI ? load1(kbr, (key0 + tid) * 4) : load1(ksr, (key0 + tid - KPI) * 4);
#pragma unroll
    for (int v = 0; v < VJ; v++) {
      const int job = tid + 512 * v, hw = job & 31, quad = job >> 5;
#pragma unroll
      for (int i = 0; i < 4; i++)
        gv[v][i] = __builtin_amdgcn_raw_buffer_load_b16(vwr, (key0 + 4 * quad + i) * 64 + 2 * hw, 0, 0);
    }
  };
  auto stage = [&](int it, int buf) {
    Stage& s = st[buf];
#pragma unroll
    for (int i = 0; i < W; i++)
      *reinterpret_cast<u32x4_t*>(&s.kt[k_key][8 * (k_word + i)]) = word_pairs(gk[i], nk);
    if (tid < 2 * KPI) {  // (all of a wave or none)
      (&s.sb[0][0])[tid] = gsb;
      if (__any(not_finite(gsb)) && lane == 0) mark[it & 3] = it + 1;
      if (tid >= KPI) {
        s.sf[0][tid - KPI] = lo_f(gsb) * p.c2;
        s.sf[1][tid - KPI] = hi_f(gsb) * p.c2;
      }
    }
#pragma unroll
    for (int v = 0; v < VJ; v++) {
      const int job = tid + 512 * v, hw = job & 31, quad = job >> 5;
      const int q8 = quad & 7, pair = 4 * (quad >> 3) + 2 * (q8 >> 2) + (q8 & 1);
      const uint32_t w[2] = {gv[v][0] | (gv[v][1] << 16), gv[v][2] | (gv[v][3] << 16)};
      const u32x2_t sv = *reinterpret_cast<const u32x2_t*>(&vsb[it & 3][0][hw >> 4][4 * quad]);
      const u32x2_t bv = *reinterpret_cast<const u32x2_t*>(&vsb[it & 3][1][hw >> 4][4 * quad]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        u32x2_t x;
#pragma unroll
        for (int y = 0; y < 2; y++) {
          // 1024 + n as fp16, less 1024: n exactly; then one rounding
          const f16x2_t n = half2((w[y] >> (4 * i) & hk.mask) | hk.one) - f16x2_t{1024.0f16, 1024.0f16};
          x[y] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, half2(sv[y]), half2(bv[y])));
        }
        *reinterpret_cast<u32x2_t*>(&s.vt[4 * hw + i][((pair ^ swizzle(4 * hw + i)) * 2 + ((q8 >> 1) & 1)) * 4]) = x;
      }
    }
  };

  // e of an iteration's keys, a lane each.  Not below -48: values from 2^-77 on
  // keep their 11 bits.
  constexpr int kLeastE = -48, kMostE = 32, kApart = 6;
  auto exponent = [&](float most) { return max(static_cast<int>(__float_as_uint(most) >> 23) - 126, kLeastE); };
  uint32_t bs = 0, bb = 0;
  const int ahead = wave / (KPI / 64), ke = tid - KPI * ahead;  // waves with `ahead` 0, and 1 at the start
  auto fetch_e = [&](int it) {
    bs = load1(vsr, (it * KPI + ke) * 4);
    bb = load1(vbr, (it * KPI + ke) * 4);
  };
  auto find_e = [&](int it, auto wide_) {
    constexpr bool wide = decltype(wide_)::value;
    const float m0 = kv4_most(lo_f(bs), lo_f(bb)), m1 = kv4_most(hi_f(bs), hi_f(bb));
    const bool ok0 = m0 <= kFloatMax, ok1 = m1 <= kFloatMax;
    // (a group that is not finite: as the other)
    int e0 = exponent(ok0 ? m0 : ok1 ? m1 : 0.0f), e1 = exponent(ok1 ? m1 : ok0 ? m0 : 0.0f);
    const bool apart = max(e0, e1) - min(e0, e1) > kApart;
    if constexpr (!wide) e0 = e1 = max(e0, e1);
    const float r0 = __uint_as_float(static_cast<uint32_t>(127 + 15 - e0) << 23);
    const float r1 = __uint_as_float(static_cast<uint32_t>(127 + 15 - e1) << 23);
    const uint32_t x0 = ok0 ? pack_f16(lo_f(bs) * r0, lo_f(bb) * r0) : 0u;
    const uint32_t x1 = ok1 ? pack_f16(hi_f(bs) * r1, hi_f(bb) * r1) : 0u;
    vsb[it & 3][0][0][ke] = static_cast<uint16_t>(x0);
    vsb[it & 3][1][0][ke] = static_cast<uint16_t>(x0 >> 16);
    vsb[it & 3][0][1][ke] = static_cast<uint16_t>(x1);
    vsb[it & 3][1][1][ke] = static_cast<uint16_t>(x1 >> 16);
    if constexpr (wide) {
      vscale[it & 3][ke] = static_cast<float>(e0);
      ve[it & 3][ke] = __float_as_uint(static_cast<float>(e1));
    } else {
      vscale[it & 3][ke] = r0;
      ve[it & 3][ke] = 0x3f800000u | __float_as_uint(static_cast<float>(e0)) >> 16;
      if (const uint64_t beyond = __ballot(apart || e0 > kMostE)) {
        if (lane == 0) atomicMin(&first_wide, it * KPI + ke + __builtin_ctzll(beyond));
      }
    }
    if (!__all(ok0 && ok1) && lane == 0) mark[it & 3] = it + 1;
  };

  const int iters = (kend_wg + KPI - 1) / KPI;
  const int it0 = split * p.bps, it1 = min(iters, it0 + p.bps);
  // everything that the start waits for, at once
  if (tid < 4) mark[tid] = 0;
  if (tid == 0) first_wide = INT32_MAX;
  if (ahead < 2) fetch_e(it0 + ahead);
  if (it0 < it1) fetch(it0);
  uint4 qd[8];
  {
    const uint16_t* qr = p.q + (row0 + row) * kKv4Dim + 8 * h;
#pragma unroll
    for (int k = 0; k < 8; k++) qd[k] = *reinterpret_cast<const uint4*>(qr + 16 * k);
  }
  __syncthreads();
  if (ahead < 2) find_e(it0 + ahead, std::false_type{});
  if (ahead == 0) fetch_e(it0 + 2);

  // ---- the query fragments: word 2 k + h of step k, in its pair order ----
  u32x4_t qf[8], pieces;
  {
    float qs[2];
#pragma unroll
    for (int y = 0; y < 2; y++) {
      qs[y] = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        uint4 d = qd[4 * y + k];
        d.x ^= p.flip;
        d.y ^= p.flip;
        d.z ^= p.flip;
        d.w ^= p.flip;
        qs[y] += gemv_unit_sum(d);
        d = permute_pairs(d);
        qf[4 * y + k] = u32x4_t{d.x, d.y, d.z, d.w};
      }
      qs[y] = add_xor32(qs[y]);
    }
    if (p.qp && split == 0 && kwi == 0 && lr < n) {
      u32x4_t* dst = reinterpret_cast<u32x4_t*>(p.qp) + (row0 + row) * kQueryWords;
#pragma unroll
      for (int k = 0; k < 8; k++) dst[4 * (k & 3) + 2 * (k >> 2) + h] = qf[k];
      if (h == 0) dst[16] = q_pieces(qs);
    }
    const float f = h ? -16.0f * p.c2 : p.c2, qh[2] = {f * qs[0], f * qs[1]};
    pieces = q_pieces(qh);
    pieces.w = h ? 0u : 0x3f80u;  // the factor of e; the others take -M
  }

  f32x16_t acc[4];
  // M is whole, so that the steps from one to the next are exact; `most` is the
  // largest t - M that leaves it as it is, -infinity before the first M.  Of
  // the wide pass: one for each group, and ml, at or above all scores
  float m, most, mg[2], most_g[2], ml, l, poison[2];

  // K's fragments of the tile to come: read while P V of the one before runs
  u32x4_t kf[8];
  auto read_k = [&](int buf, int tile) {
#pragma unroll
    for (int k = 0; k < 8; k++) kf[k] = lds_read(&st[buf].kt[kKeys * tile + lr][8 * (2 * k + h)]);
    reads_go_out();
  };
  auto multiply = [&](int it, int buf, int tile, bool more, auto wide_) {
    constexpr bool wide = decltype(wide_)::value;
    const Stage& s = st[buf];
    const int key0 = it * KPI + kKeys * tile, kl = kKeys * tile;
    if (key0 >= kend) return;  // uniform in the wave
    f32x16_t d0, d1, db;
#pragma unroll
    for (int i = 0; i < 16; i++) d0[i] = d1[i] = db[i] = 0.0f;
    const uint32_t w = s.sb[h][kl + lr];
    const uint32_t e1 = wide ? 0u : ve[it & 3][kl + lr], we = h ? 0x3f803f80u : e1;
    const bool marked = __builtin_amdgcn_readfirstlane(mark[it & 3]) == it + 1;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      d0 = mfma32(kf[k], qf[k], d0);
      d1 = mfma32(kf[4 + k], qf[4 + k], d1);
    }
    db = mfma32(u32x4_t{w, w, w, we}, pieces, db);
    float sc[16];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const f32x4_t s0 = *reinterpret_cast<const f32x4_t*>(&s.sf[0][kl + 8 * j + 4 * h]);
      const f32x4_t s1 = *reinterpret_cast<const f32x4_t*>(&s.sf[1][kl + 8 * j + 4 * h]);
#pragma unroll
      for (int i = 0; i < 4; i++)
        sc[4 * j + i] = __builtin_fmaf(s0[i], d0[4 * j + i], __builtin_fmaf(s1[i], d1[4 * j + i], db[4 * j + i]));
    }
    // V's fragments, on their way while the weights are computed
    u32x4_t vf[8];
#pragma unroll
    for (int k = 0; k < 8; k++)
      vf[k] = lds_read(&s.vt[32 * (k & 3) + lr][((4 * tile + 2 * (k >> 2) + h) ^ swizzle(lr)) * 8]);
    reads_go_out();
    const bool cut = key0 + kKeys > all_see;
    if (cut) {
      const int first = lim - key0 - 4 * h;  // hidden from here on
#pragma unroll
      for (int e = 0; e < 16; e++) {
        stay_here(sc[e]);
        if (8 * (e >> 2) + (e & 3) >= first) sc[e] = -INFINITY;
      }
    }
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < 16; e++) bm = fmaxf(bm, sc[e]);
    bm = max_xor32(bm);
    if constexpr (wide) {
      // the scores' own maximum and sum, then per group the products
      const float top = fmaxf(ml, ceilf(bm));
      if (__any(top > ml)) {
        if (ml != -INFINITY) l *= __builtin_amdgcn_exp2f(ml - top);
        ml = top;
      }
      const float base = ml == -INFINITY ? 0.0f : ml;
#pragma unroll
      for (int e = 0; e < 16; e++) l += __builtin_amdgcn_exp2f(sc[e] - base);
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const float* ey = y ? reinterpret_cast<const float*>(ve[it & 3]) : vscale[it & 3];
        float t[16];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const f32x4_t e = *reinterpret_cast<const f32x4_t*>(&ey[kl + 8 * j + 4 * h]);
#pragma unroll
          for (int i = 0; i < 4; i++) t[4 * j + i] = e[i];
        }
        float bt = sc[0] + t[0];
#pragma unroll
        for (int e = 1; e < 16; e++) bt = fmaxf(bt, sc[e] + t[e]);
        bt = max_xor32(bt);
        if (__any(bt - mg[y] > most_g[y])) {
          const bool up = bt - mg[y] > most_g[y];
          const float to = up ? ceilf(bt) - 7.0f : mg[y];
          const float a = most_g[y] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mg[y] - to);
          if (up) most_g[y] = 15.0f;
          mg[y] = to;
          acc[2 * y] *= a;
          acc[2 * y + 1] *= a;
        }
        u32x4_t pb[2];
#pragma unroll
        for (int e = 0; e < 16; e++) t[e] = __builtin_amdgcn_exp2f(sc[e] + (t[e] - mg[y]));
#pragma unroll
        for (int j = 0; j < 8; j++) pb[j >> 2][j & 3] = pack_f16(t[2 * j], t[2 * j + 1]);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          acc[2 * y] = mfma32_f16(vf[4 * k + 2 * y], pb[k], acc[2 * y]);
          acc[2 * y + 1] = mfma32_f16(vf[4 * k + 2 * y + 1], pb[k], acc[2 * y + 1]);
        }
      }
      if (more) read_k(buf, tile + 1);
    } else {
      if (__any(bm > most)) {
        const float up = bm > most ? ceilf(bm) - 7.0f : 0.0f;
        const float a = most == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-up);
        if (bm > most) most = 15.0f;
        m += up;
        const float m0 = round_bf(-m), m1 = round_bf(-m - m0);
        pieces.w = h ? pack_bf(m1, -m - m0 - m1) : pack_bf(1.0f, m0);
#pragma unroll
        for (int e = 0; e < 16; e++) sc[e] -= up;
        l *= a;
#pragma unroll
        for (int d = 0; d < 4; d++) acc[d] *= a;
      }
#pragma unroll
      for (int e = 0; e < 16; e++) sc[e] = __builtin_amdgcn_exp2f(sc[e]);
      u32x4_t pb[2];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f32x4_t r = *reinterpret_cast<const f32x4_t*>(&vscale[it & 3][kl + 8 * j + 4 * h]);
#pragma unroll
        for (int i = 0; i < 4; i++) l = __builtin_fmaf(sc[4 * j + i], r[i], l);
        pb[j >> 1][2 * (j & 1)] = pack_f16(sc[4 * j], sc[4 * j + 1]);
        pb[j >> 1][2 * (j & 1) + 1] = pack_f16(sc[4 * j + 2], sc[4 * j + 3]);
      }
      if (more) read_k(buf, tile + 1);
#pragma unroll
      for (int k = 0; k < 8; k++) acc[k & 3] = mfma32_f16(vf[k], pb[k >> 2], acc[k & 3]);
    }
    if (marked) {
#pragma unroll 1
      for (int e = 0; e < 16; e++) {
        const int key = key0 + 8 * (e >> 2) + 4 * h + (e & 3);
        const uint32_t sw = load1(vsr, key * 4), bw = load1(vbr, key * 4);
        const uint32_t sk = load1(ksr, key * 4), bk = load1(kbr, key * 4);
        if (key < lim) {
          if (not_finite(sk) || not_finite(bk)) l = NAN;
          if (!kv4_finite(lo_f(sw), lo_f(bw))) poison[0] = NAN;
          if (!kv4_finite(hi_f(sw), hi_f(bw))) poison[1] = NAN;
        }
      }
    }
  };

  // One run over the split's keys, and its rows' results; the wide one's only
  // for the rows that see key `from`
  auto pass = [&](int from, auto wide_) {
    constexpr bool wide = decltype(wide_)::value;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
    m = mg[0] = mg[1] = l = poison[0] = poison[1] = 0.0f;
    most = most_g[0] = most_g[1] = ml = -INFINITY;
    __syncthreads();  // (the marks are cleared, the first bounds found)
    if (it0 < it1) stage(it0, 0);
    if (it0 + 1 < it1) fetch(it0 + 1);
    __syncthreads();
    for (int it = it0; it < it1; it++) {
      const int buf = (it - it0) & 1;
      // the two waves of a SIMD (w and w + 4) unpack at different ends of the
      // iteration: between barriers one's VALU work falls on the other's products
      read_k(buf, kwi * TPW);
      if (wave >= 4) {
        if (it + 1 < it1) stage(it + 1, buf ^ 1);
        if (it + 2 < it1) fetch(it + 2);
      } else if (ahead == 0) {
        find_e(it + 2, wide_);
        fetch_e(it + 3);
      }
#pragma unroll
      for (int t = 0; t < TPW; t++) multiply(it, buf, kwi * TPW + t, t + 1 < TPW, wide_);
      if (wave < 4) {
        if (it + 1 < it1) stage(it + 1, buf ^ 1);
        if (it + 2 < it1) fetch(it + 2);
      }
      __syncthreads();
    }

    // ---- relative to the weights' sum: l in [1, 2) 2^-28, exactly ----
    l = add_xor32(l);
    // V had a factor 2^15; acc is relative to 2^(m - 15), and so is l, but for the wide pass
    const float ref = wide ? ml : m - 15.0f;
    const int k = static_cast<int>(__float_as_uint(l) >> 23 & 255u) - 127;
    const int down = -k - static_cast<int>(kDown);
    int shift[2] = {down, down};
    if constexpr (wide) {
#pragma unroll
      for (int y = 0; y < 2; y++)
        shift[y] += static_cast<int>(fmaxf(-1000.0f, fminf(1000.0f, mg[y] - 15.0f - ml)));
    }
    m = l != l ? l : l > 0.0f ? ref + static_cast<float>(k) : -INFINITY;  // a NaN score: the row stays NaN
    l = __builtin_amdgcn_ldexpf(l, down);
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const float bad = add_xor32(poison[d >> 1]);
#pragma unroll
      for (int i = 0; i < 16; i++) acc[d][i] = __builtin_amdgcn_ldexpf(acc[d][i], shift[d >> 1]) + bad;
    }
    // ---- waves of the same rows, two by two ----
#pragma unroll
    for (int half = KW / 2; half > 0; half >>= 1) {
      const int sl = (kwi & (half - 1)) * RW + rwi;
      if (kwi >= half && kwi < 2 * half) {
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            *reinterpret_cast<float4*>(&jn.os[sl][lr][32 * d + 8 * j + 4 * h]) =
                make_float4(acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]);
        if (h == 0) {
          jn.ms[sl][lr] = m;
          jn.ls[sl][lr] = l;
        }
      }
      __syncthreads();
      if (kwi < half) {
        const float mo = jn.ms[sl][lr], lo = jn.ls[sl][lr], mm = fmaxf(m, mo);
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
        const float b = mo == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mo - mm);
        l = __builtin_fmaf(l, a, lo * b);
        m = l != l ? l : mm;
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float4 v = *reinterpret_cast<const float4*>(&jn.os[sl][lr][32 * d + 8 * j + 4 * h]);
            acc[d][4 * j] = __builtin_fmaf(acc[d][4 * j], a, v.x * b);
            acc[d][4 * j + 1] = __builtin_fmaf(acc[d][4 * j + 1], a, v.y * b);
            acc[d][4 * j + 2] = __builtin_fmaf(acc[d][4 * j + 2], a, v.z * b);
            acc[d][4 * j + 3] = __builtin_fmaf(acc[d][4 * j + 3], a, v.w * b);
          }
      }
      __syncthreads();
    }
    if (kwi > 0 || n <= 0 || (wide && lim <= from)) return;
    if (p.ns == 1) {
      if (lr >= n) return;
#pragma unroll
      for (int d = 0; d < 4; d++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          finish_row(p, kvh, row, 32 * d + 8 * j + 4 * h,
                     make_float4(acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]), m, l);
      return;
    }
    // partials in the lanes' order, so a store writes 1 KB in one piece
    const int64_t unit = (static_cast<int64_t>(kvh) * ((R + kKeys - 1) / kKeys) + tile_of(rwi)) * p.ns + split;
    f32x4_t* po = reinterpret_cast<f32x4_t*>(p.part_o) + unit * (kKeys * kKv4Dim / 4) + lane;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        po[64 * (4 * d + j)] = f32x4_t{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
    if (h == 0) *reinterpret_cast<float2*>(p.part_ml + (unit * kKeys + lr) * 2) = make_float2(m, l);
  };
  pass(0, std::false_type{});

  // ---- rows that see values beyond the plain pass, again ----
  const int from = first_wide;  // (the last barrier is past: all keys have been looked at)
  if (from >= min(kend_wg, it1 * KPI)) return;  // uniform
  if (tid < 4) mark[tid] = 0;
  if (ahead < 2) fetch_e(it0 + ahead);
  if (it0 < it1) fetch(it0);
  __syncthreads();
  if (ahead < 2) find_e(it0 + ahead, std::true_type{});
  if (ahead == 0) fetch_e(it0 + 2);
  pieces.w = 0u;
  pass(from, std::true_type{});
}

// Joins the splits of kv4_tile_kernel: a wave per 4 dims of each half of a
// 32-row tile, in the lane order of its partials.  Bound by the latency of its
// loads: with one split after another 32 tokens over 30032 rows (16 splits)
// took 5 us more.
__global__ void __launch_bounds__(256) kv4_merge_kernel(const Kv4AttnParams p) {
  const int R = p.Hq / p.c.n_kv_heads * p.M, tiles = (R + kKeys - 1) / kKeys;
  const int wave = wave_id(), lane = threadIdx.x & 63, lr = lane & 31, h = lane >> 5;
  const int64_t tile = blockIdx.x >> 2;
  const int k = (blockIdx.x & 3) * 4 + wave;  // 4 d + j of kv4_tile_kernel
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + tile * p.ns * kKeys + lr;
  const f32x4_t* po = reinterpret_cast<const f32x4_t*>(p.part_o) + tile * p.ns * (kKeys * kKv4Dim / 4) + 64 * k + lane;
  const int kvh = static_cast<int>(tile / tiles), r = static_cast<int>(tile % tiles) * kKeys + lr;
  // 16 splits at a time, all loads of them under way at once
  constexpr int N = 16;
  float m = -INFINITY, l = 0.0f;
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < p.ns; s0 += N) {
    float2 v[N];
    f32x4_t x[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = make_float2(-INFINITY, 0.0f);
      x[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (s0 + i < p.ns) {
        v[i] = ml[(s0 + i) * kKeys];
        x[i] = po[static_cast<int64_t>(s0 + i) * (kKeys * kKv4Dim / 4)];
      }
    }
    reads_go_out();
    float mn = m;
#pragma unroll
    for (int i = 0; i < N; i++) mn = fmaxf(mn, v[i].x);
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= a;
    o *= a;
    m = mn;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float f = v[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v[i].x - m);
      l = __builtin_fmaf(f, v[i].y, l);
      o += f * x[i];
    }
  }
  if (r < R) finish_row(p, kvh, r, 8 * k + 4 * h, make_float4(o[0], o[1], o[2], o[3]), m, l);
}

// weights[h][j] += sum over the query rows of exp2(S c2 - max c2 - log2 sum).
// A wave holds 32 keys unpacked, a workgroup 256; all of them walk the rows of
// the grid's row range 16 at a time, four such tiles to a stage of LDS (two
// stages: the next is loaded while this one is multiplied).  Read by each wave
// from the L2 instead, the queries were the bound: 140 MB for 32 tokens over
// 16384 rows, 16 us.  The accumulators' start, -16 Q_g, comes from the matrix
// cores too: a product of the pieces with -16.  With several row ranges the
// sums go to p.sums [range][head][L], added up by the last workgroup of a
// range of keys (a launch for it took 1 us more for 509 tokens over 1509 rows).
constexpr int kWeighWaves = 8, kWeighKeys = kWeighWaves * kKeys, kWeighTiles = 4;
__global__ void __launch_bounds__(64 * kWeighWaves) kv4_weigh_kernel(const Kv4AttnParams p) {
  constexpr int kRowsStage = kWeighTiles * kRows, kWords = kRowsStage * kQueryWords;
  constexpr int kPer = (kWords + 64 * kWeighWaves - 1) / (64 * kWeighWaves);
  __shared__ u32x4_t qs[2][kWords];
  __shared__ float2 ls[2][kRowsStage];
  __shared__ bool last;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, b = blockIdx.y * kWeighWaves + wave;
  const int M = p.M, R = p.Hq / p.c.n_kv_heads * M, L = p.offset + M;
  // this range's rows [ra, rb), a multiple of the stage but at the end
  const int stages = (R + kRowsStage - 1) / kRowsStage, per = (stages + gridDim.z - 1) / gridDim.z;
  const int ra = static_cast<int>(blockIdx.z) * per * kRowsStage, rb = min(R, ra + per * kRowsStage);
  const int64_t slot = static_cast<int64_t>(kvh) * p.c.capacity, row0 = static_cast<int64_t>(kvh) * R;
  const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
  const PairK nk;

  u32x4_t gq[kPer];
  float2 gl;
  const u32x4_t* src = reinterpret_cast<const u32x4_t*>(p.qp) + row0 * kQueryWords;
  auto fetch = [&](int r) {  // rows r .. of the stage; past rb the last row again
#pragma unroll
    for (int k = 0; k < kPer; k++) {
      const int w = min(tid + 64 * kWeighWaves * k, kWords - 1), row = w / kQueryWords;
      gq[k] = src[static_cast<int64_t>(min(r + row, rb - 1)) * kQueryWords + (w - row * kQueryWords)];
    }
    if (tid < kRowsStage) gl = p.lse[row0 + min(r + tid, rb - 1)];
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int k = 0; k < kPer; k++) {
      const int w = tid + 64 * kWeighWaves * k;
      if (w < kWords) qs[buf][w] = gq[k];
    }
    if (tid < kRowsStage) ls[buf][tid] = gl;
  };
  if (ra < rb) fetch(ra);

  const __amdgpu_buffer_rsrc_t kwr = rsrc(p.c.k, slot * kKv4Words, L * 64);
  const __amdgpu_buffer_rsrc_t ksr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_scales), slot, L * 4);
  const __amdgpu_buffer_rsrc_t kbr = rsrc(reinterpret_cast<const uint32_t*>(p.c.k_biases), slot, L * 4);
  u32x4_t ka[2][2][2];  // [tile][group][word]
  uint32_t kb[2];
  float ks[2][8], acc[8];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int key = b * kKeys + 16 * t;
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const u32x2_t w = load2(kwr, (key + li) * 64 + 8 * g + 32 * y);
      ka[t][y][0] = word_pairs(w.x, nk);
      ka[t][y][1] = word_pairs(w.y, nk);
    }
    kb[t] = load1(kbr, (key + li) * 4);
    const u32x4_t s = load4(ksr, (key + 4 * g) * 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      ks[0][4 * t + i] = lo_f(s[i]);
      ks[1][4 * t + i] = hi_f(s[i]);
      acc[4 * t + i] = 0.0f;
    }
  }

  if (ra < rb) stage(0);
  __syncthreads();
  int buf = 0;
  for (int r0 = ra; r0 < rb; r0 += kRowsStage, buf ^= 1) {
    const bool more = r0 + kRowsStage < rb;
    if (more) fetch(r0 + kRowsStage);
    int t0 = r0 % M;  // token of the tile's first row
    for (int tile = 0; tile < kWeighTiles; tile++) {
      const int rt = r0 + tile * kRows, n = min(kRows, rb - rt);
      if (n <= 0 || b * kKeys >= L) break;  // uniform
      const bool wraps = t0 + n > M;
      const int tmax = wraps ? M - 1 : t0 + n - 1, tmin = wraps ? 0 : t0;
      t0 += kRows;
      if (t0 >= M) t0 = (rt + kRows) % M;
      if (b * kKeys > p.offset + tmax) continue;  // uniform: none of these rows sees any of these keys
      const u32x4_t* q = &qs[buf][(tile * kRows + li) * kQueryWords];
      const u32x4_t w = q[16], pieces = g ? u32x4_t{0u, 0u, 0u, 0u} : w;
      const float2 st = ls[buf][tile * kRows + li];
      // rows all alike: -16 Q_0, -16 Q_1
      const f32x4_t s0 = mfma(u32x4_t{0xC180u, 0xC180u, 0xC180u, 0u}, pieces, zero);
      const f32x4_t s1 = mfma(u32x4_t{0xC1800000u, 0xC1800000u, 0xC1800000u, 0u}, pieces, zero);
      const u32x4_t q0 = q[4 * g], q1 = q[4 * g + 1], q2 = q[4 * g + 2], q3 = q[4 * g + 3];
      float e[8];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        f32x4_t d0 = mfma(ka[t][0][0], q0, s0);
        f32x4_t d1 = mfma(ka[t][1][0], q2, s1);
        d0 = mfma(ka[t][0][1], q1, d0);
        d1 = mfma(ka[t][1][1], q3, d1);
        const f32x4_t db = mfma(u32x4_t{kb[t], kb[t], kb[t], kb[t]}, pieces, zero);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float s = __builtin_fmaf(ks[0][4 * t + i], d0[i], __builtin_fmaf(ks[1][4 * t + i], d1[i], db[i]));
          e[4 * t + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c2, -st.x) - st.y);
        }
      }
      if (n < kRows || b * kKeys + kKeys > p.offset + tmin + 1) {
        const int lim = li < n ? p.offset + (rt + li) % M + 1 : 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (b * kKeys + 16 * (i >> 2) + 4 * g + (i & 3) >= lim) e[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) acc[i] += e[i];
    }
    if (more) stage(buf ^ 1);
    __syncthreads();
  }
  // over the 16 queries of a lane row; lane (li, g) of li < 8 stores key 4 g +
  // li % 4 of tile li / 4
  float mine = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float v = row16_sum(acc[i]);
    if (li == i) mine = v;
  }
  const int key = b * kKeys + 16 * (li >> 2) + 4 * g + (li & 3);
  const bool own = li < 8 && key < L;
  if (gridDim.z == 1) {
    if (own) p.weights[slot + key] += mine;
    return;
  }
  // ---- the last workgroup of these keys adds the ranges' sums, in order ----
  auto sums = [&](int z, int j) { return p.sums + (static_cast<int64_t>(z) * gridDim.x + kvh) * L + j; };
  if (own) __hip_atomic_store(sums(blockIdx.z, key), mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    unsigned* c = p.cnt + (kvh * gridDim.y + blockIdx.y) * kCounterWords;
    last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.z - 1;
    if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  const int j = blockIdx.y * kWeighKeys + tid;
  if (!last || tid >= kWeighKeys || j >= L) return;
  float v = 0.0f;
#pragma unroll 8
  for (int z = 0; z < static_cast<int>(gridDim.z); z++)
    v += __hip_atomic_load(sums(z, j), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  p.weights[slot + j] += v;
}

constexpr int64_t kMaxQueryRows = 1 << 28;  // Hq * M of a call

bool attn_shape_ok(int Hq, int Hkv, int M, int64_t L) {
  if (Hkv <= 0 || Hkv > 65535 || Hq <= 0 || Hq > 65535 || Hq % Hkv || M <= 0 || L < M || L > kKv4MaxCapacity ||
      static_cast<int64_t>(Hq) * M > kMaxQueryRows)
    return false;
  return (static_cast<int64_t>(Hq / Hkv) * M + 255) / 256 <= 65535;  // row tiles: grid z
}

// Workgroups that a call's splits aim at: one per CU.  So keys are split over
// at most half as many (kv head, row tile) pairs, and the weights' rows over as
// many (kv head, key range) pairs: a counter each.
constexpr int kSplitGrid = 256;
static_assert(kSplitGrid / 2 <= kMaxCounters);

// Where the keys of a call are split, and where its workspace's parts are.
struct Kv4Plan {
  int rc;  // query rows of the kernel: 4, 8, 16, 64, 256
  int nw;  // its waves
  int tiles, ns, bps;
  int wz;  // row ranges of the weights' grid (1 where that has more than kSplitGrid / 2 workgroups)
  size_t lse, qp, part_o, part_ml, sums, bytes;  // byte offsets; the counters come first
};

// The kernel and split count for R > 8 query rows per kv head, by estimated
// time (us) over rounds of 256 workgroups.  16 rows: 5.8 a round and 1.53 per
// step of a wave (32 keys; two waves share a SIMD).  64 and 256 rows: 1.93 per
// iteration (128 keys), 2.05 + 0.4 per full tile (64 keys).  Splits cost the
// last workgroup's merge, or a second launch that reads all partials from
// memory.
// Measured (32 q heads over 8; 16 / 64 / 256 rows, us): 32 tokens over 4032
// 14.8 / 19.1 / 22.4, over 16384 35 / 32 / 35, over 30032 60 / 45 / 49; 64 over
// 4064 21 / 23 / 29; 128 over 4128 31 / 32 / 34, over 16128 102 / 76 / 59; 200
// over 200 12.6 / 12.1 / 16; 512 over 512 28 / 16 / 23, over 2512 78 / 45 / 48;
// 1024 over 1024 66 / 43 / 38.
void choose_kernel(int Hkv, int64_t R, int M, int L, int* rc, int* ns_out) {
  const double seen = L - 0.5 * (M - 1);  // keys of an average query
  double least = 1e30;
  for (int rows : {16, 64, 256}) {
    const int keys = rows == 16 ? 256 : rows == 64 ? 128 : 64;  // of a workgroup's step
    const int64_t pairs = Hkv * ((R + rows - 1) / rows);
    if ((R + rows - 1) / rows > 65535) continue;  // (grid z)
    const int steps = (L + keys - 1) / keys;
    const int most = static_cast<int>(std::min<int64_t>({std::max<int64_t>(1, kSplitGrid / pairs), steps, kMaxSplits}));
    for (int ns = 1; ns <= most; ns++) {
      const int bps = (steps + ns - 1) / ns;
      if (ns != (steps + bps - 1) / bps) continue;  // as another count
      const double rounds = std::ceil(static_cast<double>(pairs) * ns / kSplitGrid);
      // (the 64-row kernel's time is its last row tile's, the others' an average one's)
      const double n = std::max(1.0, (rows == 64 ? L : seen) / (static_cast<double>(keys) * ns));
      const double mb = 520e-6 * kKeys * Hkv * ((R + kKeys - 1) / kKeys) * ns;  // of partials
      double t;
      if (rows == 16) t = 1.0 + rounds * (5.8 + 1.53 * n) + (ns > 1 ? 3.0 : 0.0);
      else
        t = rows == 64 ? 8.2 + rounds * n * 1.93 + (ns > 1 ? 1.5 + 0.7 * mb : 0.0)
                       : 13.1 + rounds * n * (2.05 + 0.4 * std::min<double>(R, 256.0) / 256.0) + (ns > 1 ? 0.35 * mb : 0.0);
      if (t < least) {
        least = t;
        *rc = rows;
        *ns_out = ns;
      }
    }
  }
}

Kv4Plan make_plan(int Hq, int Hkv, int M, int L, bool weigh) {
  Kv4Plan a{};
  const int64_t R = static_cast<int64_t>(Hq / Hkv) * M;
  a.nw = 8;
  int ns = 1, keys;  // keys of a workgroup's step
  if (R <= 8) {
    a.rc = R <= 4 ? 4 : 8;
    // workgroups of 4 waves as long as one step of each covers the context
    // with a workgroup per CU: they start and join sooner (32 heads over 8, us
    // with 4 / 8 waves: 4097 rows 8.6 / 10.6, 8192 9.2 / 10.5, 12001 10.4 / 10.9,
    // 20001 12.2 / 13.1, but 131072 37 / 34)
    keys = a.rc == 4 ? 64 : 32;
    a.nw = Hkv * ((L + 4 * keys - 1) / (4 * keys)) <= kSplitGrid ? 4 : 8;
    keys *= a.nw;
    ns = std::min<int64_t>({std::max<int64_t>(1, kSplitGrid / Hkv), (L + keys - 1) / keys, kMaxSplits});
  } else {
    choose_kernel(Hkv, R, M, L, &a.rc, &ns);
    keys = a.rc == 16 ? 256 : a.rc == 64 ? 128 : 64;
  }
  const int steps = (L + keys - 1) / keys;
  a.tiles = static_cast<int>((R + a.rc - 1) / a.rc);
  a.bps = (steps + ns - 1) / ns;
  a.ns = (steps + a.bps - 1) / a.bps;
  // the weights: row ranges until there are as many workgroups as CUs, of at
  // least two stages each
  const int64_t key_groups = static_cast<int64_t>(Hkv) * ((L + kWeighKeys - 1) / kWeighKeys);
  const int64_t stages = (R + kWeighTiles * kRows - 1) / (kWeighTiles * kRows);
  a.wz = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((stages + 1) / 2, kSplitGrid / key_groups)));
  const size_t rows = static_cast<size_t>(Hq) * M;
  size_t at = BMX_KV4_COUNTER_BYTES;
  a.lse = at;
  if (weigh) at += rows * sizeof(float2);
  at = (at + 15) & ~static_cast<size_t>(15);
  a.qp = at;
  if (weigh) at += rows * kQueryWords * sizeof(uint4);
  a.part_o = at;
  const size_t part_rows = a.rc > kRows ? Hkv * ((R + kKeys - 1) / kKeys) * kKeys : rows;
  if (a.ns > 1) at += part_rows * a.ns * kKv4Dim * sizeof(float);
  a.part_ml = at;
  if (a.ns > 1) at += part_rows * a.ns * 2 * sizeof(float);
  a.sums = at;
  if (weigh && a.wz > 1) at += static_cast<size_t>(a.wz) * Hkv * L * sizeof(float);
  a.bytes = at;
  return a;
}

// What any call of up to M queries that ends at up to row L needs, so a bound
// that grows with both: at most kSplitGrid workgroups of 256 rows where keys
// are split at all, tiles filled up to 32 rows, and the weights' sums for at
// most 256 workgroups of 256 keys.
size_t plan_bound(int Hq, int Hkv, int M, int L, bool weigh) {
  const size_t rows = static_cast<size_t>(Hq) * M;
  const size_t steps = (static_cast<size_t>(L) + 63) / 64;  // the smallest a split may be
  const size_t parts = std::min<size_t>((rows + static_cast<size_t>(Hkv) * kKeys) * std::min<size_t>(steps, kMaxSplits),
                                        static_cast<size_t>(kSplitGrid) * 256);
  return BMX_KV4_COUNTER_BYTES + parts * (kKv4Dim + 2) * sizeof(float) +
         (weigh ? rows * (sizeof(float2) + kQueryWords * sizeof(uint4)) + 16 + 256 * kWeighKeys * sizeof(float) : 0);
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_attention_kv4_workspace_bytes(int n_heads, int n_kv_heads, int M, int L, int weigh) {
  return attn_shape_ok(n_heads, n_kv_heads, M, L) ? plan_bound(n_heads, n_kv_heads, M, L, weigh != 0) : 0;
}

extern "C" int bmx_attention_gqa_kv4(const bmx_bf16* q, const bmx_kv4* cache, bmx_bf16* out, float* weights,
                                     int n_heads, int M, int head_dim, int offset, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (int rc = check_kv4("attention_kv4", cache, head_dim)) return rc;
  if (!q || !out || !workspace) return set_error(BMX_E_ARG, "attention_kv4: null pointer");
  const int Hkv = cache->n_kv_heads;
  if (M < 0 || n_heads <= 0 || n_heads % Hkv)
    return set_error(BMX_E_SHAPE, "attention_kv4: M=%d, %d heads over %d kv heads", M, n_heads, Hkv);
  if (int rc = check_kv4_rows("attention_kv4", cache, M, offset)) return rc;
  const int L = offset + M;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(weights, 16))
    return set_error(BMX_E_ALIGN, "attention_kv4: q, out, weights and workspace must be 16-byte aligned");
  if (M == 0) return BMX_OK;
  if (!attn_shape_ok(n_heads, Hkv, M, L))
    return set_error(BMX_E_SHAPE, "attention_kv4: %d heads, M=%d too large for one call", n_heads, M);
  const Kv4Plan a = make_plan(n_heads, Hkv, M, L, weights != nullptr);
  const size_t need = plan_bound(n_heads, Hkv, M, L, weights != nullptr);
  if (workspace_bytes < need || need < a.bytes)
    return set_error(BMX_E_ARG, "attention_kv4: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const size_t bytes = static_cast<size_t>(n_heads) * M * kKv4Dim * sizeof(uint16_t);
  if (kv4_overlap(q, bytes, out, bytes)) return set_error(BMX_E_ARG, "attention_kv4: out overlaps q");
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
  // workgroups go to the XCDs in turn by their linear number, x first
  p.local = a.rc <= kRows && a.ns > 1 && Hkv % 8 == 0 && attention_xcd_local(as_stream(stream));
  const dim3 grid(Hkv, a.ns, a.tiles), block(64 * a.nw);
  const hipStream_t st = as_stream(stream);
  if (a.rc == 4 && a.nw == 4) hipLaunchKernelGGL((kv4_few_kernel<4, 4>), grid, block, 0, st, p);
  else if (a.rc == 4) hipLaunchKernelGGL((kv4_few_kernel<4, 8>), grid, block, 0, st, p);
  else if (a.rc == 8 && a.nw == 4) hipLaunchKernelGGL((kv4_few_kernel<8, 4>), grid, block, 0, st, p);
  else if (a.rc == 8) hipLaunchKernelGGL((kv4_few_kernel<8, 8>), grid, block, 0, st, p);
  else if (a.rc == kRows) hipLaunchKernelGGL((kv4_rows_kernel<8>), grid, block, 0, st, p);
  else if (a.rc == 64) hipLaunchKernelGGL(kv4_tile_kernel<2>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(kv4_tile_kernel<8>, grid, block, 0, st, p);
  if (int rc = check_launch("attention_kv4")) return rc;
  if (a.rc > kRows && a.ns > 1) {
    const int64_t units = Hkv * ((static_cast<int64_t>(n_heads / Hkv) * M + kKeys - 1) / kKeys);
    hipLaunchKernelGGL(kv4_merge_kernel, dim3(static_cast<unsigned>(4 * units)), dim3(256), 0, st, p);
    if (int rc = check_launch("attention_kv4 merge")) return rc;
  }
  if (!weights) return BMX_OK;
  p.sums = reinterpret_cast<float*>(ws + a.sums);
  hipLaunchKernelGGL(kv4_weigh_kernel, dim3(Hkv, (L + kWeighKeys - 1) / kWeighKeys, a.wz), dim3(64 * kWeighWaves), 0, st,
                     p);
  return check_launch("attention_kv4 weights");
}
