// Causal GQA attention of a batch's packed queries over a paged KV cache
// (gfx950).
//
//   out[i, h] = softmax(scale q[h, i] k^T) v over rows 0 .. p of the token's
//   sequence, p its position
//
// Of a kv head and a sequence the query rows are r = token * rep + (q head
// within the kv head's rep), so that any number of heads fills a tile.
//
// By the rows a sequence can have (max_new * rep):
//   up to 32 (decode, verified drafts): paged_few_kernel, bound by memory.  K and
//     V go from memory to registers and from there into the products.
//   up to 64: paged_mid_kernel, by 64-key blocks through LDS.
//     Either way the key blocks of all (sequence, kv head) pairs in a row are cut
//     into equal shares, one per workgroup, so lengths need not be alike; what
//     several workgroups did of a pair is joined by the last of them or by
//     paged_few_merge_kernel.
//   more (prompts, chunks, and decode steps beside them): paged_tile_kernel,
//     bound by the products and the softmax between them, by tiles of 128 or 256
//     rows that paged_plan_kernel lists longest first and cuts where they are
//     few, paged_tile_merge_kernel joining the pieces.
// Rows common to all sequences (`shared`) are one more "sequence" of all the
// batch's query rows, taken by tiles: in the launch of the rest where a sequence
// has few rows (paged_shared_kernel), before it otherwise (paged_prefix_kernel).
// The merges fold in what comes of them.
//
// Scores are in base 2: p = 2^(s c - m), c = |scale| log2 e (a negative scale
// flips q's signs).  The running m is set 2^16 above a row's largest score, and
// anew only once that has grown by 2^8, each row by itself: sums and outputs are
// fp32 either way, and the rescaling of the outputs all but vanishes.  Weights of
// at most 2^-8, and 2^-16 where m was just set, keep the sums of 2^15 rows of values
// of 2^120 in range (of 256 next to bf16's largest); values of 2^-100 still have
// 2^-116, above the smallest normal.  With one bf16 piece of p, outputs were off by
// 0.0024 of their norm where their own rounding is 0.0017, so p has
// more bits: two bf16 pieces (16 bits), in every kernel, so that a token's
// precision does not depend on what else is in its batch, and V stays the bf16
// that it is, of any size.  (Tiles with p and V in fp16 save the second product,
// a 4096-token prompt 166 us for 204, for 5 bits of p, for values below 2^-25
// beside larger ones, and for a second run of tiles whose values lie far apart.)
#include <math.h>

#include <algorithm>

#include "paged.h"
#include "paged_pieces.h"

namespace bmx {
namespace {

constexpr int kD = kPagedDim;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kAbove = 16.0f;  // log2 by which m is set above the largest score
constexpr float kLazy = 8.0f;    // log2 by which that may grow before m is set anew
constexpr float kLeast = 1.17549435e-38f;  // of c: a scale of 0 leaves a hidden key's -inf what it is

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

struct PagedAttn {
  const uint16_t* q;  // [Hq, T, 128]
  const uint16_t* k;  // [n_pages, Hkv, page_size, 128]
  const uint16_t* v;
  uint16_t* out;      // [T, Hq*128]
  const int* starts;
  const int* lens;
  const int* pages;
  int B, max_pages, T, max_new;
  int Hq, Hkv, rep, n_pages, shift;
  int shared;
  float c2;           // |scale| log2(e)
  uint32_t flip;      // sign bits of a bf16 pair where scale < 0
  // ---- workspace ----
  int* plan;          // few rows: share, blocks before each sequence; tiles: PlanHead and its lists
  float* row_o;       // few rows: [T, Hq, 128] parts that start a pair's blocks
  float* row_ml;      // [T, Hq, 2]
  float* wg_o;        // few rows: [workgroups, rows, 128] parts that continue a pair's; tiles: [slots, Hkv, tile_rows, 128]
  float* wg_ml;
  float* pre_o;       // [np, T, Hq, 128] parts over the shared rows
  float* pre_ml;
  int np;             // key splits of the shared rows
  int pre_bps;        // 64-key blocks of such a split
  int most_items, most_cuts;  // of the plan's lists
  int tile_rows;      // 128 or 256
  int few_shift;      // of few rows: log2 of a block's keys
  unsigned* cnt;      // arrivals of a pair's parts, kCounterStride apart, zero between calls; null: a launch joins them
};

// ---- parts that workgroups of one launch hand to one another ----
// A pair's parts are written through to memory (agent-scope stores), which a
// workgroup waits for before it counts its arrival; the last to arrive reads
// them with agent-scope loads.  Nothing that an XCD's L2 holds from earlier is
// read, and no L2 is flushed.  The counter wraps to zero with the last arrival.
constexpr int kCounterStride = 16;  // words: a counter to a 64-byte piece of memory
constexpr int kMaxCounters = BMX_PAGED_COUNTER_BYTES / (4 * kCounterStride);
__device__ __forceinline__ void put2(float* to, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(to),
                     static_cast<uint64_t>(__float_as_uint(x)) | (static_cast<uint64_t>(__float_as_uint(y)) << 32),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* from) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// A maximum of -inf (no key seen) counts as 0
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
// The maximum that a partial result is stored with.  -inf tells the merge that
// nothing was seen; scores that are all NaN leave it there too, with a sum that
// is NaN, and must not be skipped.
__device__ __forceinline__ float part_max(float m, float l) { return l == l ? m : 0.0f; }

typedef __attribute__((ext_vector_type(2))) float f32x2_t;
// Two bf16 values in a word: one v_cvt_pk_bf16_f32
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
}
// The bf16 pairs (-1, 0) and (0, -1) held in registers: as constants in the
// instruction they came out as other numbers (the products as 0).
struct MinusOne {
  uint32_t low, high;
};
__device__ __forceinline__ MinusOne minus_one() {
  MinusOne c{0x0000bf80u, 0xbf800000u};
  asm volatile("" : "+v"(c.low), "+v"(c.high));
  return c;
}
// Eight probabilities as two bf16 operands, hi + lo
__device__ __forceinline__ void split8(const float (&p)[8], const MinusOne& one, bf16x8_t& hi, bf16x8_t& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    h[u] = pack2(p[2 * u], p[2 * u + 1]);
    // p - hi, exact: products with -1 and 0
    const float a = dot2_bf16(h[u], one.low, p[2 * u]), b = dot2_bf16(h[u], one.high, p[2 * u + 1]);
    l[u] = pack2(a, b);
  }
  hi = __builtin_bit_cast(bf16x8_t, make_uint4(h[0], h[1], h[2], h[3]));
  lo = __builtin_bit_cast(bf16x8_t, make_uint4(l[0], l[1], l[2], l[3]));
}

// ---- values that are not finite, in rows that only some queries see ----
// A product over keys would carry 0 x inf of a hidden row into a query.  So in
// the blocks that only some queries see whole, values that are not finite enter
// the product as zeros, and where there were any (rare), the queries that see
// them get them added at the end.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {  // bits 15, 31: halves whose exponent is all ones
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
__device__ __forceinline__ uint32_t finite_part(uint32_t w) { return w & ~((not_finite(w) >> 15) * 0xffffu); }
// o plus a pair of values where these are not finite
__device__ __forceinline__ void add_not_finite(float& o0, float& o1, uint32_t w) {
  if (not_finite(w) & 0x8000u) o0 += bf2f(w & 0xffffu);
  if (not_finite(w) & 0x80000000u) o1 += bf2f(w >> 16);
}
// Where row `key` of a sequence's page table lies (in values, of kv head h); -1: nowhere
__device__ __forceinline__ int64_t row_at(const PagedAttn& p, const int* table, int h, int key) {
  const int pg = table[key >> p.shift];
  if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.n_pages)) return -1;
  return (((static_cast<int64_t>(pg) * p.Hkv + h) << p.shift) + (key & ((1 << p.shift) - 1))) * kD;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ===========================================================================
// few query rows
// ===========================================================================
constexpr int kFewKeys = 128;   // of a block: 32 per wave
constexpr int kFewOs = kD + 4;  // LDS stride of an output row

// Exclusive prefix over 256 threads, and the total; tmp: 4 ints
__device__ __forceinline__ int scan256(int v, int* tmp, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const int s = tmp[w];
    if (w < wave) before += s;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// Key blocks of a sequence (past the shared rows): 0 where it has no new token
__device__ __forceinline__ int few_blocks(const PagedAttn& p, const PagedSeq& s) {
  if (s.tokens == 0) return 0;
  const int end = min(s.pos + min(s.tokens, p.max_new), p.max_pages << p.shift);
  return max(end - p.shared + (1 << p.few_shift) - 1, 0) >> p.few_shift;
}

// A workgroup's share of all pairs' blocks, [t, t1): a pair (sequence, kv head;
// heads inner) and a block of it at a time.
struct Share {
  int t, t1, share, b, h, j, nb;
  PagedSeq sq;
};
// The share of workgroup wg of wgs; false where it is empty.  *lone: whether any
// sequence has new tokens and no block.  tmp: 8 ints, found: 5.
__device__ __forceinline__ bool first_share(const PagedAttn& p, int wg, int wgs, int* tmp, int* found, Share& s, bool* lone) {
  const int tid = threadIdx.x;
  const int per = (p.B + 255) >> 8, b0 = tid * per;
  int mine = 0;
  bool none = false;
  PagedSeq only{0, 0, 0};
  for (int i = 0; i < per && b0 + i < p.B; i++) {
    only = paged_seq(p.starts[b0 + i], p.starts[b0 + i + 1], p.lens[b0 + i], p.T);
    const int n = few_blocks(p, only);
    mine += n;
    none = none || (only.tokens > 0 && n == 0);
  }
  const bool some = __any(none);
  if ((tid & 63) == 0) tmp[4 + (tid >> 6)] = some;
  int all;
  const int before = scan256(mine, tmp, &all);
  *lone = (tmp[4] | tmp[5] | tmp[6] | tmp[7]) != 0;
  const int share = max(1, (p.Hkv * all + wgs - 1) / wgs);
  s.share = share;
  s.t = wg * share;
  s.t1 = min(s.t + share, p.Hkv * all);
  if (wg == 0 || (s.t < s.t1 && p.Hkv * before <= s.t && s.t < p.Hkv * (before + mine))) {
    int at = before;
    for (int i = 0; i < per && b0 + i < p.B; i++) {
      const PagedSeq q = per == 1 ? only : paged_seq(p.starts[b0 + i], p.starts[b0 + i + 1], p.lens[b0 + i], p.T);
      const int n = few_blocks(p, q);
      if (wg == 0) p.plan[1 + b0 + i] = at;
      if (p.Hkv * at <= s.t && s.t < p.Hkv * (at + n)) {
        found[0] = b0 + i;
        found[1] = at;
        found[2] = q.row0;
        found[3] = q.tokens;
        found[4] = q.pos;
      }
      at += n;
    }
    if (wg == 0 && tid == 0) p.plan[0] = share;
  }
  __syncthreads();
  if (s.t >= s.t1) return false;
  s.b = uniform(found[0]);
  const int rel = s.t - p.Hkv * uniform(found[1]);
  s.sq = PagedSeq{uniform(found[2]), uniform(found[3]), uniform(found[4])};
  s.nb = few_blocks(p, s.sq);
  if (s.nb == 0) return false;  // (not reached: the scan found blocks here)
  s.h = min(rel / s.nb, p.Hkv - 1);
  s.j = min(rel - s.h * s.nb, s.nb - 1);
  return true;
}
// n blocks on, to the start of the next pair; false at the end
__device__ __forceinline__ bool next_share(const PagedAttn& p, int n, Share& s) {
  s.t += n;
  s.j = 0;
  if (s.t >= s.t1) return false;
  if (++s.h < p.Hkv) return true;
  s.h = 0;
  do {
    if (++s.b == p.B) return false;  // (not reached: blocks remain, so a sequence with some does)
    s.sq = paged_seq(p.starts[s.b], p.starts[s.b + 1], p.lens[s.b], p.T);
    s.nb = few_blocks(p, s.sq);
  } while (s.nb == 0);
  return true;
}

// A row's parts, folded one after another: 32 lanes per row, 4 values each.
struct Fold {
  float m = -INFINITY, l = 0.0f;
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __device__ __forceinline__ void add(const float2& ml, const float4& v) {
    if (ml.x == -INFINITY) return;  // nothing seen
    const float mn = fmaxf(m, ml.x);
    const float wa = __builtin_amdgcn_exp2f(m - mn), wb = __builtin_amdgcn_exp2f(ml.x - mn);
    l = l * wa + ml.y * wb;
    a.x = a.x * wa + v.x * wb;
    a.y = a.y * wa + v.y * wb;
    a.z = a.z * wa + v.z * wb;
    a.w = a.w * wa + v.w * wb;
    m = mn;
  }
  // parts i0, i0 + by, ... < n, `step` rows apart, lane's values from d on, kB of
  // them in flight; HANDED: written in this launch
  template <bool HANDED, int kB>
  __device__ __forceinline__ void add_batch(const float* o, const float* ml, int64_t step, int i0, int by, int n, int d) {
    float2 mv[kB];
    float4 ov[kB];
#pragma unroll
    for (int u = 0; u < kB; u++) {
      const int64_t r = min(i0 + u * by, n - 1) * step;
      if constexpr (HANDED) {
        mv[u] = get2(ml + r * 2);
        const float2 x = get2(o + r * kD + d), y = get2(o + r * kD + d + 2);
        ov[u] = make_float4(x.x, x.y, y.x, y.y);
      } else {
        mv[u] = *reinterpret_cast<const float2*>(ml + r * 2);
        ov[u] = *reinterpret_cast<const float4*>(o + r * kD + d);
      }
    }
#pragma unroll
    for (int u = 0; u < kB; u++)
      if (i0 + u * by < n) add(mv[u], ov[u]);
  }
  template <bool HANDED = false>
  __device__ __forceinline__ void add_all(const float* o, const float* ml, int64_t step, int i0, int by, int n, int d) {
    for (; i0 + 3 * by < n; i0 += 8 * by) add_batch<HANDED, 8>(o, ml, step, i0, by, n, d);
    for (; i0 < n; i0 += 2 * by) add_batch<HANDED, 2>(o, ml, step, i0, by, n, d);
  }
  __device__ __forceinline__ void store(uint16_t* dst) const {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack2(a.x * inv, a.y * inv), pack2(a.z * inv, a.w * inv));
  }
};

// Tokens of sequences without a block, which see nothing: zeros.  The workgroups
// take sequences in turn.
__device__ __forceinline__ void few_lone(const PagedAttn& p) {
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const PagedSeq sq = paged_seq(p.starts[b], p.starts[b + 1], p.lens[b], p.T);
    if (sq.tokens == 0 || few_blocks(p, sq) > 0) continue;
    uint4* to = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(sq.row0) * p.Hq * kD);
    for (int i = threadIdx.x; i < min(sq.tokens, p.max_new) * p.Hq * kD / 8; i += 256) to[i] = make_uint4(0, 0, 0, 0);
  }
}

// Up to 16 NT query rows of a pair, in blocks of 128 keys.  Per wave and step of
// 32 keys, in two 16-key tiles:
//   S^T = K Q^T (v_mfma_f32_16x16x32_bf16): lane l holds query row l % 16 and
//     keys 4 (l / 16) + i of each tile;
//   O^T += V^T P^T: the eight keys of a lane's scores are its k slice as they
//     lie; lane l loads values 8 (l % 16) .. + 7 of just these keys and turns
//     them by byte permutes, so neither K, V nor P goes through LDS.  Product
//     j's row l % 16 is value 8 (l % 16) + j: a lane ends with the outputs
//     32 (l / 16) .. + 31 of its query.
// The next step's K is requested when this step's scores are done, its V when
// the values are turned, also where the next step is another pair's: short
// sequences wait for no first load but the workgroup's.
// Bound by memory: two workgroups to a CU keep 2 x 4 waves x 16 KB on their way.
// 64 single tokens over 500 to 8191 rows, 8 kv heads: 135 us, 711 MB at 5.3 TB/s (a
// large copy moves 4.9); one over 131000 beside 7 short ones
// 106 us, 5.1 TB/s.  One over 4096: 13 us, of which the join's launch is 4.5, and the rest is the latency
// of the table, its rows and the sum through LDS.
struct FewLds {
  float os[4][16][kFewOs];
  float ms[4][32], ls[4][32];
  int tmp[8], found[5];
};
template <int NT>
__device__ __forceinline__ void few_run(const PagedAttn& p, FewLds& lds, int wg, int wgs) {
  static_assert(NT <= 2);
  auto& os = lds.os;
  auto& ms = lds.ms;
  auto& ls = lds.ls;
  int* const found = lds.found;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, li = lane & 15, g = lane >> 4;
  const MinusOne one = minus_one();
  Share at;
  bool lone;
  const bool some = first_share(p, wg, wgs, lds.tmp, found, at, &lone);
  if (NT == 1 && lone && p.cnt) few_lone(p);
  if (!some) return;
  // What the loads of a pair's rows need
  struct Where {
    const int* table;
    int h, c0, end;  // its kv head; the wave's keys of its first block; rows < end are seen by some query
  };
  auto where = [&](const Share& s) {
    return Where{p.pages + static_cast<int64_t>(s.b) * p.max_pages, s.h, p.shared + s.j * kFewKeys + wave * 32,
                 min(s.sq.pos + min(s.sq.tokens, p.max_new), p.max_pages << p.shift)};
  };
  uint4 kb[2][4], vw[8], qf[NT][4];
  int64_t base[2];  // elements to the 16-key tiles' rows; -1: no such page
  int pg[2];        // page numbers, asked for a step before the rows they lead to
  auto ask = [&](const Where& w, int c0, int (&to)[2]) {
#pragma unroll
    for (int u = 0; u < 2; u++) to[u] = c0 + 16 * u < w.end ? w.table[(c0 + 16 * u) >> p.shift] : -1;
  };
  auto locate = [&](const Where& w, int c0, const int (&from)[2]) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int at = uniform(from[u]), key = c0 + 16 * u;
      base[u] = static_cast<unsigned>(at) < static_cast<unsigned>(p.n_pages)
                    ? (((static_cast<int64_t>(at) * p.Hkv + w.h) << p.shift) + (key & ((1 << p.shift) - 1))) * kD
                    : -1;
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint16_t* src = p.k + max(base[u], static_cast<int64_t>(0)) + li * kD + 8 * g;
#pragma unroll
      for (int ks = 0; ks < 4; ks++) kb[u][ks] = *reinterpret_cast<const uint4*>(src + 32 * ks);
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int e = 0; e < 8; e++)
      vw[e] = *reinterpret_cast<const uint4*>(p.v + max(base[e >> 2], static_cast<int64_t>(0)) +
                                              (4 * g + (e & 3)) * kD + 8 * li);
  };
  auto row_of = [&](const Share& s, int nt, int& tok, int& hd) {  // the lane's query row (past the last: that)
    const int r = min(16 * nt + li, min(s.sq.tokens, p.max_new) * p.rep - 1);
    tok = r / p.rep;
    hd = s.h * p.rep + r - tok * p.rep;
  };
  auto load_q = [&](const Share& s) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      int tok, hd;
      row_of(s, nt, tok, hd);
      const uint16_t* src = p.q + (static_cast<int64_t>(hd) * p.T + s.sq.row0 + tok) * kD + 8 * g;
#pragma unroll
      for (int ks = 0; ks < 4; ks++) qf[nt][ks] = *reinterpret_cast<const uint4*>(src + 32 * ks);
    }
  };
  Where now = where(at);
  ask(now, now.c0, pg);
  load_q(at);
  locate(now, now.c0, pg);
  ask(now, now.c0 + kFewKeys, pg);
  load_k();
  load_v();
  bool more_shares;
  do {
    // ---- the segment: blocks j .. j + n - 1 of a pair ----
    const PagedSeq sq = at.sq;
    const int h = at.h, j = at.j, nb = at.nb, n = min(at.t1 - at.t, nb - j);
    // the next one: its first rows are asked for in this one's last step
    Share next = at;
    more_shares = next_share(p, n, next);
    Where then = now;
    int first_pg[2] = {-1, -1};
    if (more_shares) {
      then = where(next);
      ask(then, then.c0, first_pg);
    }
    const int R = min(sq.tokens, p.max_new) * p.rep;
    const int cap = p.max_pages << p.shift, end = now.end;
    const int first = min(sq.pos + 1, cap);  // rows < first are seen by every query
    const int* table = now.table;
    int lim[NT];   // rows < lim are seen by the lane's query
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      int tok, hd;
      row_of(at, nt, tok, hd);
      lim[nt] = min(sq.pos + tok + 1, cap);
#pragma unroll
      for (int ks = 0; ks < 4; ks++) {
        qf[nt][ks].x ^= p.flip;
        qf[nt][ks].y ^= p.flip;
        qf[nt][ks].z ^= p.flip;
        qf[nt][ks].w ^= p.flip;
      }
    }
    f32x4_t o[NT][8];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      m[nt] = -INFINITY;
      l[nt] = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; d++) o[nt][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool odd = false;  // some value that is not finite was left out
    int c0 = now.c0;
    for (int s = 0; s < n; s++, c0 += kFewKeys) {
      const bool ok0 = base[0] >= 0, ok1 = base[1] >= 0;
      const bool whole = ok0 && ok1 && c0 + 32 <= first;  // every query sees every key
      // ---- scores ----
      f32x4_t sc[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          sc[nt][u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < 4; ks++)
            sc[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kb[u][ks]),
                                                                __builtin_bit_cast(bf16x8_t, qf[nt][ks]), sc[nt][u], 0,
                                                                0, 0);
        }
      if (s + 1 < n) {
        locate(now, c0 + kFewKeys, pg);
        load_k();
        ask(now, c0 + 2 * kFewKeys, pg);
      } else if (more_shares) {
        locate(then, then.c0, first_pg);
        load_k();
        load_q(next);
        ask(then, then.c0 + kFewKeys, pg);
      }
      bf16x8_t hi[NT], lo[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        if (!whole) {
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (!((u ? ok1 : ok0) && c0 + 16 * u + 4 * g + i < lim[nt])) sc[nt][u][i] = -INFINITY;
        }
        float mx = sc[nt][0][0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, sc[nt][e >> 2][e & 3]);
        mx = max_xor32(max_xor16(mx)) * p.c2;
        if (__any(mx > m[nt] + (kLazy - kAbove))) {
          const float m1 = mx > m[nt] + (kLazy - kAbove) ? mx + kAbove : m[nt];
          const float alpha = __builtin_amdgcn_exp2f(m[nt] - finite_max(m1));
          m[nt] = m1;
          l[nt] *= alpha;
#pragma unroll
          for (int d = 0; d < 8; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[nt][d][i] *= alpha;
        }
        const float mu = finite_max(m[nt]);
        float e8[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          e8[e] = __builtin_amdgcn_exp2f(fmaf(sc[nt][e >> 2][e & 3], p.c2, -mu));
          l[nt] += e8[e];
        }
        split8(e8, one, hi[nt], lo[nt]);
      }
      // ---- rows that no query sees count as zeros ----
      if (!(ok0 && ok1 && c0 + 32 <= end)) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!((e < 4 ? ok0 : ok1) && c0 + 16 * (e >> 2) + 4 * g + (e & 3) < end)) vw[e] = make_uint4(0, 0, 0, 0);
      }
      if (first < end && c0 + 32 > first) {  // (uniform) rows that only some queries see
        uint32_t nf = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          nf |= not_finite(vw[e].x) | not_finite(vw[e].y) | not_finite(vw[e].z) | not_finite(vw[e].w);
          vw[e] = make_uint4(finite_part(vw[e].x), finite_part(vw[e].y), finite_part(vw[e].z), finite_part(vw[e].w));
        }
        odd = odd || __any(nf != 0);
      }
#pragma unroll
      for (int d2 = 0; d2 < 4; d2++) {
        auto word = [&](int e) { return d2 == 0 ? vw[e].x : d2 == 1 ? vw[e].y : d2 == 2 ? vw[e].z : vw[e].w; };
        uint32_t a[2][4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          a[0][e] = __builtin_amdgcn_perm(word(2 * e + 1), word(2 * e), 0x05040100u);
          a[1][e] = __builtin_amdgcn_perm(word(2 * e + 1), word(2 * e), 0x07060302u);
        }
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const int d = 2 * d2 + z;
          const uint4 av = make_uint4(a[z][0], a[z][1], a[z][2], a[z][3]);
          const bf16x8_t vb = __builtin_bit_cast(bf16x8_t, av);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, hi[nt], o[nt][d], 0, 0, 0);
            o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, lo[nt], o[nt][d], 0, 0, 0);
          }
        }
      }
      if (s + 1 < n || more_shares) load_v();
    }
    if (odd) {  // uniform
      const int k0 = p.shared + j * kFewKeys;
      for (int key = max(k0, p.shared + ((first - p.shared) & ~31)); key < min(k0 + n * kFewKeys, end); key++) {
        const int64_t at = row_at(p, table, h, key);
        if (at < 0) continue;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int d = 0; d < 8; d += 2) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(p.v + at + 32 * g + 8 * i + d);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              float x = o[nt][d][i], y = o[nt][d + 1][i];
              if (key < lim[nt]) add_not_finite(x, y, w);
              o[nt][d][i] = x;
              o[nt][d + 1][i] = y;
            }
          }
      }
    }
    // ---- the parts of four waves joined, 16 rows at a time ----
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float sum = add_xor32(add_xor16(l[nt]));
      if (g == 0) {
        ms[wave][16 * nt + li] = part_max(m[nt], sum);
        ls[wave][16 * nt + li] = sum;
      }
    }
    const bool direct = n == nb && !p.shared;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      if (16 * nt >= R) break;  // uniform
      if (nt > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float* dst = &os[wave][li][32 * g + 8 * i];
        *reinterpret_cast<float4*>(dst) = make_float4(o[nt][0][i], o[nt][1][i], o[nt][2][i], o[nt][3][i]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(o[nt][4][i], o[nt][5][i], o[nt][6][i], o[nt][7][i]);
      }
      __syncthreads();
      constexpr int kE = 8;  // values of a thread
      const int row = tid >> 4, d0 = kE * (tid & 15), r = 16 * nt + row;
      if (r < R) {
        float mm = -INFINITY, ll = 0.0f, a[kE] = {};
#pragma unroll
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, ms[w][r]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
          if (ms[w][r] == -INFINITY) continue;  // (its outputs are zeros)
          const float x = __builtin_amdgcn_exp2f(ms[w][r] - mm);
          ll += x * ls[w][r];
#pragma unroll
          for (int d = 0; d < kE; d++) a[d] += x * os[w][row][d0 + d];
        }
        const int tok = r / p.rep, hd = h * p.rep + r - tok * p.rep;
        const int64_t dst = static_cast<int64_t>(sq.row0 + tok) * p.Hq + hd;
        if (direct) {
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
          for (int d = 0; d < kE; d += 4)
            *reinterpret_cast<uint2*>(p.out + dst * kD + d0 + d) =
                make_uint2(pack2(a[d] * inv, a[d + 1] * inv), pack2(a[d + 2] * inv, a[d + 3] * inv));
        } else {
          const int64_t slot = j == 0 ? dst : static_cast<int64_t>(wg) * (16 * NT) + r;
          float* po = (j == 0 ? p.row_o : p.wg_o) + slot * kD + d0;
          float* pml = (j == 0 ? p.row_ml : p.wg_ml) + slot * 2;
          if (NT == 1 && p.cnt) {
#pragma unroll
            for (int d = 0; d < kE; d += 2) put2(po + d, a[d], a[d + 1]);
            if (d0 == 0) put2(pml, part_max(mm, ll), ll);
          } else {
#pragma unroll
            for (int d = 0; d < kE; d += 4) *reinterpret_cast<float4*>(po + d) = make_float4(a[d], a[d + 1], a[d + 2], a[d + 3]);
            if (d0 == 0) *reinterpret_cast<float2*>(pml) = make_float2(part_max(mm, ll), ll);
          }
        }
      }
    }
    if (NT == 1 && !direct && p.cnt) {
      // ---- the last of the pair's workgroups to arrive folds its parts ----
      const int u0 = at.t - j, w0 = u0 / at.share, parts = (u0 + nb - 1) / at.share - w0 + 1;
      vm_wait<0>();  // this thread's part is in memory
      __syncthreads();
      if (tid == 0) {
        unsigned* const c = p.cnt + (static_cast<int64_t>(at.b) * p.Hkv + h) * kCounterStride;
        found[0] = __builtin_amdgcn_atomic_inc32(c, parts - 1, __ATOMIC_RELAXED, "agent") == static_cast<unsigned>(parts - 1);
      }
      __syncthreads();
      if (uniform(found[0])) {
        // 32 lanes to a row, or several times 32 where there are fewer rows than eight
        const int by = R > 4 ? 1 : R > 2 ? 2 : R > 1 ? 4 : 8, sub = tid >> 5, ln = tid & 31, d = 4 * ln, i0 = sub % by;
        for (int r = sub / by; r < (R + 7) / 8 * 8; r += 8 / by) {
          Fold f;
          const int rr = min(r, R - 1), tok = rr / p.rep;
          const int64_t dst = static_cast<int64_t>(sq.row0 + tok) * p.Hq + h * p.rep + rr - tok * p.rep;
          if (i0 == 0) f.add_batch<true, 1>(p.row_o + dst * kD, p.row_ml + dst * 2, 0, 0, 1, 1, d);
          const int64_t first = static_cast<int64_t>(w0 + 1) * (16 * NT) + rr;
          f.add_all<true>(p.wg_o + first * kD, p.wg_ml + first * 2, 16 * NT, i0, by, parts - 1, d);
          if (by > 1) {  // (uniform: one turn)
            float4* as = reinterpret_cast<float4*>(&os[0][0][0]);
            float2* mls = reinterpret_cast<float2*>(&os[2][0][0]);
            as[sub * 32 + ln] = f.a;
            if (ln == 0) mls[sub] = make_float2(part_max(f.m, f.l), f.l);
            __syncthreads();
            f = Fold();
            for (int u = 0; u < by; u++) f.add(mls[sub - i0 + u], as[(sub - i0 + u) * 32 + ln]);
          }
          if (i0 == 0 && r < R) f.store(p.out + dst * kD + d);
          if (by > 1) break;
        }
      }
    }
    __syncthreads();  // (os, ms and ls are the next segment's)
    at = next;
    now = then;
  } while (more_shares);
}

template <int NT>
__global__ void __launch_bounds__(256, 2) paged_few_kernel(const PagedAttn p) {
  __shared__ __align__(16) FewLds lds;
  few_run<NT>(p, lds, blockIdx.x, gridDim.x);
}

// The rows of (sequence z, kv head y) that paged_few_kernel did not finish:
// parts over the shared rows, the part that starts the pair's blocks, and one
// of each further workgroup they go through.  8 rows to a workgroup, or (WIDE)
// one, whose parts its eight 32-lane groups share out: the 32 rows of one
// sequence of 4097, 32 parts each, take 5.2 us instead of 7.4.
template <int NT, bool WIDE>
__global__ void __launch_bounds__(256) paged_few_merge_kernel(const PagedAttn p) {
  __shared__ __align__(16) float4 as[8][32];
  __shared__ float2 mls[8];
  const int b = blockIdx.z, h = blockIdx.y, sub = threadIdx.x >> 5, ln = threadIdx.x & 31, d = 4 * ln;
  const int r = WIDE ? blockIdx.x : blockIdx.x * 8 + sub;
  const PagedSeq sq = paged_seq(p.starts[b], p.starts[b + 1], p.lens[b], p.T);
  if (r >= min(sq.tokens, p.max_new) * p.rep) return;
  const int nb = few_blocks(p, sq), share = p.plan[0], u0 = p.Hkv * p.plan[1 + b] + h * nb;
  const int w0 = u0 / share, w1 = (u0 + nb - 1) / share;
  if (!p.shared && nb > 0 && w0 == w1) return;  // done
  const int tok = r / p.rep;
  const int64_t at = static_cast<int64_t>(sq.row0 + tok) * p.Hq + h * p.rep + r - tok * p.rep;
  const int i0 = WIDE ? sub : 0, by = WIDE ? 8 : 1;
  Fold f;
  if (p.shared) f.add_all(p.pre_o + at * kD, p.pre_ml + at * 2, static_cast<int64_t>(p.T) * p.Hq, i0, by, p.np, d);
  if (nb > 0) {
    if (i0 == 0)
      f.add(*reinterpret_cast<const float2*>(p.row_ml + at * 2), *reinterpret_cast<const float4*>(p.row_o + at * kD + d));
    const int64_t first = static_cast<int64_t>(w0 + 1) * (16 * NT) + r;
    if (w1 > w0) f.add_all(p.wg_o + first * kD, p.wg_ml + first * 2, 16 * NT, i0, by, w1 - w0, d);
  }
  if constexpr (WIDE) {
    as[sub][ln] = f.a;
    if (ln == 0) mls[sub] = make_float2(part_max(f.m, f.l), f.l);
    __syncthreads();
    if (sub != 0) return;
    f = Fold();
#pragma unroll
    for (int u = 0; u < 8; u++) f.add(mls[u], as[u][ln]);
  }
  f.store(p.out + at * kD + d);
}

// ===========================================================================
// many query rows
// ===========================================================================
constexpr int kTileKeys = 64;  // of a block
constexpr int kTileBytes = kTileKeys * kD * 2;  // of a K or V tile
// K and V, two of each; which waves' rows of the two blocks exist; a flag of each wave
constexpr size_t kTileLds = 4 * kTileBytes + 3 * 8 * sizeof(int);

// A piece of work: rows r0 .. of sequence b, 64-key blocks [j0, j1), and the
// slot that takes its result (-1: it is the whole of it).
struct Item {
  int b, r0, j0, j1, slot, pad[3];
};
// A tile whose keys were cut into n pieces, in slots slot ..: rows r0 .. R - 1
// (at most a tile's) of the sequence whose packed rows begin at row0
struct Cut {
  int row0, R, r0, slot, n, pad[3];
};
struct PlanHead {
  int items, cuts, pad[2];
};
__device__ __forceinline__ Item* plan_items(const PagedAttn& p) { return reinterpret_cast<Item*>(p.plan + 4); }
__device__ __forceinline__ Cut* plan_cuts(const PagedAttn& p) {
  return reinterpret_cast<Cut*>(plan_items(p) + p.most_items);
}

template <class T>
__device__ __forceinline__ __attribute__((address_space(3))) T* lds_ptr(uint32_t off) {
  return reinterpret_cast<__attribute__((address_space(3))) T*>(off);
}
// lane l's 16 bytes at base + off go to LDS byte `dst` + 16 l; base and dst are
// wave-uniform (lds_load16 with the base in scalar registers)
__device__ __forceinline__ void lds_load16_at(const void* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory");
}

__device__ __align__(256) uint32_t g_zeros[64];  // a row that is read in the place of one that no query sees

// Where a tile's rows go: to `out`, or as partial results, at the rows' places
// [T, Hq] or at the tile's own.
struct Result {
  float* o;
  float* ml;
  bool by_row;
};

// The order of a loop's instructions: groups of n products, LDS reads, or vector
// arithmetic (exponentials included) as listed.
#define SCHED(kind, n) __builtin_amdgcn_sched_group_barrier(kind, n, 0)
constexpr int kSchedMfma = 0x8, kSchedRead = 0x100, kSchedValu = 0x402;

// The 32 NW / WK rows from r0 on of (sequence, kv head) -- of all the batch's rows,
// over the shared ones, where PRE -- against 64-key blocks, 32 rows to a wave (WK = 2:
// to two, half of each block's keys each).
//   S^T = K Q^T (v_mfma_f32_32x32x16_bf16): lane l holds query row l % 32 and
//     keys 8 (r / 4) + 4 (l / 32) + r % 4 of its 16 registers r per 32 keys;
//   O^T += V^T P^T: the eight keys of a step are eight neighbouring score
//     registers; V^T comes out of LDS by transposed reads (ds_read_b64_tr_b16:
//     16 lanes read 4 keys x 16 values and each gets one value of the 4 keys).
// K and V tiles go from memory straight to LDS, a block ahead; a row's 16-byte
// chunk c lies at c ^ (4 (row % 4) + row / 4 % 4), which keeps both kinds of
// read off each other's banks.  64 KB of LDS and up to 256 registers: two
// workgroups share a CU, one's exponentials beside the other's products.
// One prompt of 4096 tokens, 32 heads: 200 to 217 us (cards differ; the kernel 208),
// 137 GFLOP at 0.66 PFLOP/s, where a large matrix product reaches 1.12; the two
// pieces of the weights make it 206 GFLOP of products, 0.99.  The matrix cores are
// busy 51 % of the cycles and the vector units 46 %: the two overlap only in part.
template <bool PRE, int NW, int WK>
__device__ __forceinline__ void tile_run(const PagedAttn& p, char* lds, const PagedSeq& sq, int b, int h, int r0, int j0,
                                         int j1, const Result& to) {
  constexpr int WR = NW / WK, NK = 2 / WK;  // row groups of waves; 32-key tiles of a wave
  constexpr int kOwn = kTileKeys / NW;      // rows of K and V that a wave stages
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, j = lane & 31, hf = lane >> 5;
  const int wr = wave % WR, wk = wave / WR;
  int* exist = reinterpret_cast<int*>(lds + 4 * kTileBytes);  // [2][NW]
  int* left_out = exist + 2 * NW;  // [NW]: of a wave's rows, some value that is not finite was left out
  const MinusOne one = minus_one();
  const int cap = p.max_pages << p.shift;
  const int tokens = PRE ? p.T : min(sq.tokens, p.max_new);
  const int R = tokens * p.rep;
  const int key0 = PRE ? 0 : p.shared;
  auto limit = [&](int r) {  // rows seen by query row r
    return PRE ? p.shared : min(sq.pos + r / p.rep + 1, cap);
  };
  const int end = limit(min(r0 + 32 * WR, R) - 1), first = limit(r0);  // by some, by every row of the tile
  const int rw = r0 + 32 * wr;
  const bool live = rw < R;                                        // (uniform) the wave has rows
  const int end_w = live ? limit(min(rw + 32, R) - 1) : 0, first_w = live ? limit(rw) : 0;  // by some, by every row of the wave
  const int rr = min(rw + j, R - 1), tok = rr / p.rep, hd = h * p.rep + rr - tok * p.rep;
  const int lim = limit(rr);
  const int* table = p.pages + static_cast<int64_t>(b) * p.max_pages;
  uint4 qf[8];
  {
    const uint16_t* src = p.q + (static_cast<int64_t>(hd) * p.T + sq.row0 + tok) * kD + 8 * hf;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      qf[ks] = *reinterpret_cast<const uint4*>(src + 16 * ks);
      qf[ks].x ^= p.flip;
      qf[ks].y ^= p.flip;
      qf[ks].z ^= p.flip;
      qf[ks].w ^= p.flip;
    }
  }
  f32x16_t o[4];
#pragma unroll
  for (int dt = 0; dt < 4; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[dt][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  // ---- staging: the wave's rows of each tile, 4 rows to an instruction ----
  const int lrow = lane >> 4;  // row of the four
  // chunk (lane % 16) of LDS holds the row's chunk ^ swizzle
  const uint32_t voff0 = lrow * 256 + (((lane & 15) ^ (4 * lrow) ^ (kOwn / 4 * wave & 3)) << 4);
  // (the page is asked for a block before its rows)
  int asked = -1;
  auto ask = [&](int jb) {
    const int k0 = key0 + jb * kTileKeys + kOwn * wave;
    asked = k0 < end ? table[k0 >> p.shift] : -1;
  };
  auto stage = [&](int jb, int buf) {
    const int k0 = key0 + jb * kTileKeys + kOwn * wave;
    const int pg = uniform(asked);
    ask(jb + 1);
    const bool ok = static_cast<unsigned>(pg) < static_cast<unsigned>(p.n_pages);
    if (lane == 0) exist[NW * buf + wave] = ok;
    const int64_t at = ok ? (((static_cast<int64_t>(pg) * p.Hkv + h) << p.shift) + (k0 & ((1 << p.shift) - 1))) * kD : 0;
    const uint32_t dst = uniform(lds_offset(lds) + buf * 2 * kTileBytes + wave * kOwn * 256);
    uint32_t v0 = voff0;
    asm volatile("" : "+v"(v0));
    const uint32_t voff[4] = {v0, v0 ^ (1024 | 16), v0 ^ (2048 | 32), v0 ^ (3 * 1024 | 48)};  // + 4 i rows
    if (ok && k0 + kOwn <= end) {  // uniform
#pragma unroll
      for (int i = 0; i < kOwn / 4; i++) {
        lds_load16_at(p.k + at, voff[i], dst + 1024 * i);
        lds_load16_at(p.v + at, voff[i], dst + kTileBytes + 1024 * i);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kOwn / 4; i++) {
      const bool in = ok && k0 + 4 * i + lrow < end;
      const char* zero = reinterpret_cast<const char*>(g_zeros) + 16 * (lane & 15);
      lds_load16(in ? reinterpret_cast<const char*>(p.k + at) + voff[i] : zero, dst + 1024 * i);
      lds_load16(in ? reinterpret_cast<const char*>(p.v + at) + voff[i] : zero, dst + kTileBytes + 1024 * i);
    }
  };
  // ... and what is done to the wave's rows of V once they are there: in blocks
  // that only some queries see whole, values that are not finite become 0
  auto settle = [&](int jb, int buf) {
    const int k0 = key0 + jb * kTileKeys;
    if (PRE || k0 + kTileKeys <= first || first >= end) return;  // uniform
    char* at = lds + buf * 2 * kTileBytes + kTileBytes + wave * kOwn * 256 + lane * 16;
    uint4 w[kOwn / 4];
    uint32_t nf = 0;
#pragma unroll
    for (int i = 0; i < kOwn / 4; i++) {
      w[i] = *reinterpret_cast<const uint4*>(at + i * 1024);
      nf |= not_finite(w[i].x) | not_finite(w[i].y) | not_finite(w[i].z) | not_finite(w[i].w);
      w[i] = make_uint4(finite_part(w[i].x), finite_part(w[i].y), finite_part(w[i].z), finite_part(w[i].w));
    }
    if (!__any(nf != 0)) return;
    if (lane == 0) left_out[wave] = 1;
#pragma unroll
    for (int i = 0; i < kOwn / 4; i++) *reinterpret_cast<uint4*>(at + i * 1024) = w[i];
  };
  // ---- LDS addresses: of a row's chunk, the others' follow by exclusive or
  // (made anew in every block: 16 registers otherwise) ----
  const int swk = 4 * (j & 3) + ((j >> 2) & 3);
  const uint32_t kat0 = lds_offset(lds) + wk * NK * 32 * 256 + j * 256 + ((hf ^ swk) << 4);
  const int i16 = lane & 15, grp = (lane >> 4) & 1;
  uint32_t vat0[2];  // [half of the 8 keys], of key step 0 and dim tile 0
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int row = 8 * u + 4 * hf + (i16 >> 2);
    const int ch = (2 * grp + ((i16 & 3) >> 1)) ^ (4 * (row & 3) + ((row >> 2) & 3));
    vat0[u] = lds_offset(lds) + kTileBytes + wk * NK * 32 * 256 + row * 256 + ch * 16 + 8 * (i16 & 1);
  }
  auto block = [&](int bo, int k0, const int (&e4)[4], bool all) {
    uint32_t kat = kat0 + bo, vat[2] = {vat0[0] + bo, vat0[1] + bo};
    asm volatile("" : "+v"(kat), "+v"(vat[0]), "+v"(vat[1]));
    // ---- scores ----
    f32x16_t sc[NK];
#pragma unroll
    for (int kt = 0; kt < NK; kt++)
#pragma unroll
      for (int r = 0; r < 16; r++) sc[kt][r] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
      for (int kt = 0; kt < NK; kt++) {
        const u32x4_t a = *lds_ptr<u32x4_t>((kat ^ (ks << 5)) + kt * 32 * 256);
        sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                         __builtin_bit_cast(bf16x8_t, qf[ks]), sc[kt], 0, 0, 0);
      }
    // (reads of K two steps ahead of the products that take them)
    SCHED(kSchedRead, 2 * NK);
#pragma unroll
    for (int i = 0; i < 6; i++) {
      SCHED(kSchedMfma, NK);
      SCHED(kSchedRead, NK);
    }
    SCHED(kSchedMfma, 2 * NK);
    if (!all || k0 + 32 * NK > first_w) {  // uniform
      #pragma unroll
      for (int kt = 0; kt < NK; kt++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int key = 32 * kt + 8 * (r >> 2) + 4 * hf + (r & 3);
          const bool see = k0 + key < lim && (WK == 1 || wk == 0 ? e4[2 * kt + (r >> 3)] : e4[2 + (r >> 3)]);
          sc[kt][r] = see ? sc[kt][r] : -INFINITY;
        }
    }
    // ---- softmax ----
    float mx = sc[0][0];
#pragma unroll
    for (int r = 1; r < 16 * NK; r++) mx = fmaxf(mx, sc[r >> 4][r & 15]);
    mx = max_xor32(mx) * p.c2;
    if (__any(mx > m + (kLazy - kAbove))) {
      const float m1 = mx > m + (kLazy - kAbove) ? mx + kAbove : m;
      const float alpha = __builtin_amdgcn_exp2f(m - finite_max(m1));
      m = m1;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[dt][r] *= alpha;
    }
    // ---- O^T += V^T P^T, 16 keys a step; a step's exponentials beside the
    // products of the one before ----
    auto values = [&](int dt, int s) {
      const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<s16x4_t>((vat[0] ^ (dt << 6)) + s * 16 * 256));
      const s16x4_t c = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<s16x4_t>((vat[1] ^ (dt << 6)) + s * 16 * 256));
      const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, c);
      return make_uint4(x.x, x.y, y.x, y.y);
    };
    const float mu = finite_max(m);
    float sum = 0.0f;
    auto weigh = [&](int s, float (&e8)[8]) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        e8[e] = __builtin_amdgcn_exp2f(fmaf(sc[s >> 1][8 * (s & 1) + e], p.c2, -mu));
        sum += e8[e];
      }
    };
    uint4 va[4];
#pragma unroll
    for (int dt = 0; dt < 4; dt++) va[dt] = values(dt, 0);
    bf16x8_t hi, lo;
    auto weigh2 = [&](int s) {
      float e8[8];
      weigh(s, e8);
      split8(e8, one, hi, lo);
    };
    weigh2(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 2 * NK; s++) {
      const bf16x8_t h1 = hi, h2 = lo;
      uint4 vc[4];
#pragma unroll
      for (int dt = 0; dt < 4; dt++) vc[dt] = va[dt];
      if (s < 2 * NK - 1) {
#pragma unroll
        for (int dt = 0; dt < 4; dt++) va[dt] = values(dt, s + 1);
        weigh2(s + 1);
      }
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vc[dt]), h1, o[dt], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vc[dt]), h2, o[dt], 0, 0, 0);
      if (s < 2 * NK - 1) {
        SCHED(kSchedRead, 8);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          SCHED(kSchedMfma, 1);
          SCHED(kSchedValu, 6);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l += sum;
  };
  __syncthreads();  // (an earlier piece's reads of LDS are over)
  if (lane == 0) left_out[wave] = 0;  // (each wave its own, which it alone sets)
  if (j0 < j1) {
    ask(j0);
    stage(j0, 0);
    vm_wait<0>();
    settle(j0, 0);
  }
  for (int jb = j0; jb < j1; jb++) {
    const int buf = (jb - j0) & 1, bo = buf * 2 * kTileBytes;
    __syncthreads();
    int e4[4], least = 1;
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
      const int4 e = *reinterpret_cast<const int4*>(exist + NW * buf + i);
      least = min(least, min(min(e.x, e.y), min(e.z, e.w)));
      if constexpr (NW == 4) {
        e4[0] = e.x, e4[1] = e.y, e4[2] = e.z, e4[3] = e.w;
      } else {
        e4[i / 2] = e.x, e4[i / 2 + 1] = e.z;  // (two waves to 16 rows)
      }
    }
    const bool all = uniform(least) != 0;
    if (jb + 1 < j1) stage(jb + 1, buf ^ 1);
    const int k0 = key0 + jb * kTileKeys + wk * NK * 32;
    // (uniform: keys hidden from all of the wave's rows are only settled)
    if (k0 < end_w) block(bo, k0, e4, all);
    if (jb + 1 < j1) {
      vm_wait<0>();
      settle(jb + 1, buf ^ 1);
    }
  }
  l = add_xor32(l);
  if constexpr (!PRE) {
    int odd = 0;  // (the last block was settled before its barrier)
#pragma unroll
    for (int w = 0; w < NW; w++) odd |= left_out[w];
    if (j0 < j1 && uniform(odd)) {
      const int from = key0 + max(j0 * kTileKeys, (first - key0) & ~(kTileKeys - 1));
      for (int key = from; key < min(key0 + j1 * kTileKeys, end); key++) {
        const int64_t at = row_at(p, table, h, key);
        if (at < 0 || key >= lim) continue;
#pragma unroll
        for (int dt = 0; dt < 4; dt++)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            float x = o[dt][r], y = o[dt][r + 1];
            add_not_finite(x, y, *reinterpret_cast<const uint32_t*>(p.v + at + 32 * dt + 8 * (r >> 2) + 4 * hf + (r & 3)));
            o[dt][r] = x;
            o[dt][r + 1] = y;
          }
      }
    }
  }
  if constexpr (WK > 1) {
    // ---- the key halves of a row group joined: the second wave's state through LDS ----
    static_assert(WK == 2);
    __syncthreads();  // (reads of K and V are over)
    float4* st = reinterpret_cast<float4*>(lds + wr * (64 * 64 * 4 + 1024));
    float2* sml = reinterpret_cast<float2*>(st + 16 * 64);
    if (wk == 1) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        st[i * 64 + lane] = make_float4(o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2],
                                        o[i >> 2][4 * (i & 3) + 3]);
      sml[lane] = make_float2(part_max(m, l), l);
    }
    __syncthreads();
    if (wk == 1) return;
    const float2 ml = sml[lane];
    if (!(l == l)) m = 0.0f;
    const float mn = fmaxf(m, ml.x);
    const float wa = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float wb = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
    l = l * wa + ml.y * wb;
    m = mn;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float4 x = st[i * 64 + lane];
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int r = 0; r < 4; r++) o[i >> 2][4 * (i & 3) + r] = o[i >> 2][4 * (i & 3) + r] * wa + v[r] * wb;
    }
  }
  auto finish = [&]() {
    const int64_t row = static_cast<int64_t>(sq.row0 + tok) * p.Hq + hd;
    if (!to.o) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint16_t* dst = p.out + row * kD + 4 * hf;
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
          const f32x16_t& a = o[dt];
          *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * r4) =
              make_uint2(pack2(a[4 * r4] * inv, a[4 * r4 + 1] * inv), pack2(a[4 * r4 + 2] * inv, a[4 * r4 + 3] * inv));
        }
      return;
    }
    const int64_t part = to.by_row ? row : 32 * wr + j;
    if (hf == 0) *reinterpret_cast<float2*>(to.ml + part * 2) = make_float2(part_max(m, l), l);
    float* dst = to.o + part * kD + 4 * hf;
#pragma unroll
    for (int dt = 0; dt < 4; dt++)
#pragma unroll
      for (int r4 = 0; r4 < 4; r4++)
        *reinterpret_cast<float4*>(dst + 32 * dt + 8 * r4) =
            make_float4(o[dt][4 * r4], o[dt][4 * r4 + 1], o[dt][4 * r4 + 2], o[dt][4 * r4 + 3]);
  };
  if (rw + j < R) finish();
}

// Key split z of 128- (NW = 8: 256-) row tile i of all the batch's rows, over the
// shared rows
template <int NW>
__device__ __forceinline__ void prefix_run(const PagedAttn& p, char* lds, int h, int i, int z) {
  const int nb = (p.shared + kTileKeys - 1) / kTileKeys, j0 = z * p.pre_bps;
  const int64_t slot = static_cast<int64_t>(z) * p.T * p.Hq;
  tile_run<true, NW, 1>(p, lds, PagedSeq{0, p.T, 0}, 0, h, i * (32 * NW), j0, min(j0 + p.pre_bps, nb),
                        Result{p.pre_o + slot * kD, p.pre_ml + slot * 2, true});
}

// Grid (kv heads, row tiles, key splits).
template <int NW>
__global__ void __launch_bounds__(64 * NW, 2) paged_prefix_kernel(const PagedAttn p) {
  extern __shared__ __align__(256) char lds[];  // (a row's 256 bytes: the addresses are made by exclusive or)
  prefix_run<NW>(p, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The plan's items, longest first: kv head blockIdx % Hkv, items a, 2A-1-a,
// 2A+a, ... of the A workgroups of a head, so that who had a longer one has a
// shorter one next.
template <int NW>
__global__ void __launch_bounds__(64 * NW, 2) paged_tile_kernel(const PagedAttn p) {
  extern __shared__ __align__(256) char lds[];  // (a row's 256 bytes: the addresses are made by exclusive or)
  const int h = blockIdx.x % p.Hkv, a = blockIdx.x / p.Hkv, A = gridDim.x / p.Hkv;
  const int items = p.plan[0];
  for (int r = 0; r * A < items; r++) {
    const int at = r * A + ((r & 1) ? A - 1 - a : a);
    if (at >= items) continue;
    const Item it = plan_items(p)[at];
    const int64_t slot = (static_cast<int64_t>(uniform(it.slot)) * p.Hkv + h) * (32 * NW);
    const int b = uniform(it.b);
    const PagedSeq sq = paged_seq(p.starts[b], p.starts[b + 1], p.lens[b], p.T);
    tile_run<false, NW, 1>(p, lds, sq, b, h, uniform(it.r0), uniform(it.j0), uniform(it.j1),
                       slot < 0 ? Result{nullptr, nullptr, false} : Result{p.wg_o + slot * kD, p.wg_ml + slot * 2, false});
  }
}

// Up to 64 query rows of a pair, in blocks of 64 keys by shares as few_run: two
// row groups of waves, each by two waves that take half of a block's keys.  16
// sequences of 5 tokens, 40 rows each, over 300 to 3000 rows: 29 us (the kernel 23.1), 79 MB at 3.4 TB/s: bound by
// the softmax between loads that LDS holds one block ahead.
__device__ __forceinline__ void mid_run(const PagedAttn& p, char* lds, int wg, int wgs) {
  int* const tmp = reinterpret_cast<int*>(lds + kTileLds);
  Share at;
  bool lone;
  if (!first_share(p, wg, wgs, tmp, tmp + 8, at, &lone)) return;
  bool more;
  do {
    const int n = min(at.t1 - at.t, at.nb - at.j);
    const int64_t slot = static_cast<int64_t>(wg) * 64;
    Result to{nullptr, nullptr, false};
    if (n < at.nb || p.shared)
      to = at.j == 0 ? Result{p.row_o, p.row_ml, true} : Result{p.wg_o + slot * kD, p.wg_ml + slot * 2, false};
    tile_run<false, 4, 2>(p, lds, at.sq, at.b, at.h, 0, at.j, at.j + n, to);
    more = next_share(p, n, at);
  } while (more);
}
constexpr size_t kMidLds = kTileLds + 16 * sizeof(int);

__global__ void __launch_bounds__(256, 2) paged_mid_kernel(const PagedAttn p) {
  extern __shared__ __align__(256) char lds[];
  mid_run(p, lds, blockIdx.x, gridDim.x);
}

// The shared rows (the first `pre` workgroups: kv heads x row tiles x key splits)
// and the sequences' own by shares (NT = 4: mid_run) in one launch: neither waits
// for the other's last workgroups (8 tokens over 2048 shared rows 21 us in two launches,
// 15 in one; 64 over 4096 35 and 31).
template <int NT>
__global__ void __launch_bounds__(256, 2) paged_shared_kernel(const PagedAttn p, int pre) {
  extern __shared__ __align__(256) char lds[];
  const int wg = static_cast<int>(blockIdx.x) - pre, wgs = static_cast<int>(gridDim.x) - pre;
  if (wg < 0) {
    const int i = blockIdx.x / p.Hkv;
    prefix_run<4>(p, lds, blockIdx.x % p.Hkv, i / p.np, i % p.np);
  } else if constexpr (NT == 4) {
    mid_run(p, lds, wg, wgs);
  } else {
    few_run<NT>(p, *reinterpret_cast<FewLds*>(lds), wg, wgs);
  }
}

// One workgroup lists the tiles of all sequences, cut where there are too few
// to fill the `per_head` workgroups of a kv head: longest piece first, by a
// counting sort of the pieces' lengths.  Pieces of one length come in any
// order, which moves work about and no result.
constexpr int kPlanThreads = 1024, kPlanBins = 1024;

// Exclusive prefix of v over the workgroup, and the total; tmp: 17 ints
__device__ __forceinline__ int plan_scan(int v, int* tmp, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int y = tmp[lane & 15];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const int z = __shfl_up(y, o, 16);
    if ((lane & 15) >= o) y += z;
  }
  *total = __shfl(y, 15, 64);
  return x - v + (wave ? __shfl(y, wave - 1, 64) : 0);
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedAttn p, int per_head) {
  __shared__ int tiles_before[kPagedMaxSeqs], rows_of[kPagedMaxSeqs], pos_of[kPagedMaxSeqs];
  __shared__ int bins[kPlanBins];
  __shared__ int tmp[2][16], top[16], sums[16], counts[3];  // items, cuts, slots
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < 3) counts[tid] = 0;
  bins[tid] = 0;
  // ---- sequences, and the tiles before each ----
  const int per = (p.B + kPlanThreads - 1) / kPlanThreads, b0 = tid * per;
  int mine = 0;
  for (int b = b0; b < min(b0 + per, p.B); b++) {
    const PagedSeq s = paged_seq(p.starts[b], p.starts[b + 1], p.lens[b], p.T);
    const int R = min(s.tokens, p.max_new) * p.rep;
    rows_of[b] = R;
    pos_of[b] = s.pos;
    mine += (R + p.tile_rows - 1) / p.tile_rows;
  }
  int n;
  int at = plan_scan(mine, tmp[0], &n);
  for (int b = b0; b < min(b0 + per, p.B); b++) {
    tiles_before[b] = at;
    at += (rows_of[b] + p.tile_rows - 1) / p.tile_rows;
  }
  __syncthreads();
  n = min(n, p.most_items - 2 * per_head);  // (starts out of order could count more)
  // ---- a tile's sequence, first row and blocks; a thread's first is kept ----
  auto find = [&](int i, int& b, int& r0) {
    int lo = 0, hi = p.B;  // the last sequence with tiles_before <= i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tiles_before[mid] <= i) lo = mid;
      else hi = mid;
    }
    b = lo;
    r0 = (i - tiles_before[lo]) * p.tile_rows;
    const int end = min(pos_of[lo] + (min(r0 + p.tile_rows, rows_of[lo]) - 1) / p.rep + 1, p.max_pages << p.shift);
    return max(end - p.shared + kTileKeys - 1, 0) / kTileKeys;
  };
  int kb = 0, kr0 = 0;
  const int knb = tid < n ? find(tid, kb, kr0) : 0;
  auto tile = [&](int i, int& b, int& r0) {
    if (i != tid) return find(i, b, r0);
    b = kb;
    r0 = kr0;
    return knb;
  };
  int sum = 0, most = 1;
  for (int i = tid; i < n; i += kPlanThreads) {
    int b, r0;
    const int nb = tile(i, b, r0);
    sum += nb;
    most = max(most, nb);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, 64);
    most = max(most, __shfl_xor(most, o, 64));
  }
  if (lane == 0) {
    sums[wave] = sum;
    top[wave] = most;
  }
  __syncthreads();
  sum = sums[lane & 15];
  most = top[lane & 15];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, 16);
    most = max(most, __shfl_xor(most, o, 16));
  }
  // ---- pieces of at most `size` blocks: each piece more is results to be written
  // and joined (us with 1 / 1.25 / 1.5 / 2 times the average, or uncut: 1000 tokens
  // over 3000 rows 130 / 115 / 115 / 135 / 125; a chunk of 509 beside 31 single tokens
  // 77 / 76 / 75 / 80 / 107; 64 over 30000 76 / 78 / 81 / 73 / 758; six prompts of 1 to
  // 2049 90 / 89 / 83 / 83 / 86; 509 over 3000 81 / 66 / 69 / 75 / 102) ----
  const int size = piece_size(sum, per_head, most);
  const float to_bin = static_cast<float>(kPlanBins - 1) / static_cast<float>(size);
  auto bin_of = [&](int len) { return kPlanBins - 1 - min(static_cast<int>(len * to_bin), kPlanBins - 1); };
  for (int i = tid; i < n; i += kPlanThreads) {
    int b, r0, len;
    const int parts = piece_count(tile(i, b, r0), size, &len);
    atomicAdd(&bins[bin_of(len)], parts);
  }
  __syncthreads();
  {
    int total;
    const int first = plan_scan(bins[tid], tmp[1], &total);
    bins[tid] = first;  // (each thread its own)
    if (tid == 0) counts[0] = total;
  }
  __syncthreads();
  Item* items = plan_items(p);
  Cut* cuts = plan_cuts(p);
  for (int i = tid; i < n; i += kPlanThreads) {
    int b, r0, len;
    const int nb = tile(i, b, r0), parts = piece_count(nb, size, &len);
    int slot = -1;
    if (parts > 1 || p.shared) {
      slot = atomicAdd(&counts[2], parts);
      const int c = atomicAdd(&counts[1], 1);
      const int row0 = min(max(p.starts[b], 0), p.T);
      if (c < p.most_cuts) cuts[c] = Cut{row0, rows_of[b], r0, slot, parts, {0, 0, 0}};
    }
    const int to = atomicAdd(&bins[bin_of(len)], parts);
    for (int k = 0; k < parts; k++)
      if (to + k < p.most_items)
        items[to + k] = Item{b, r0, k * len, min((k + 1) * len, nb), slot < 0 ? -1 : slot + k, {0, 0, 0}};
  }
  __syncthreads();
  if (tid == 0) {
    p.plan[0] = min(counts[0], p.most_items);
    p.plan[1] = min(counts[1], p.most_cuts);
  }
}

// The cut tiles' rows, 8 to a workgroup: parts over the shared rows, then the
// pieces'.  (6 to 8 us, most of it the launch and the latency of the plan, a part's
// maximum and its values.)
constexpr int kTileMergeGrid = 2048;
__global__ void __launch_bounds__(256) paged_tile_merge_kernel(const PagedAttn p) {
  const int groups = p.tile_rows / 8, n = p.plan[1] * p.Hkv * groups, d = 4 * (threadIdx.x & 31);
  for (int w = blockIdx.x; w < n; w += gridDim.x) {
    const int g = w % groups, h = w / groups % p.Hkv;
    const Cut c = plan_cuts(p)[w / groups / p.Hkv];
    const int k = 8 * g + (threadIdx.x >> 5), r = c.r0 + k;
    if (r >= c.R) continue;
    const int tok = r / p.rep;
    const int64_t at = static_cast<int64_t>(c.row0 + tok) * p.Hq + h * p.rep + r - tok * p.rep;
    Fold f;
    if (p.shared) f.add_all(p.pre_o + at * kD, p.pre_ml + at * 2, static_cast<int64_t>(p.T) * p.Hq, 0, 1, p.np, d);
    const int64_t first = (static_cast<int64_t>(c.slot) * p.Hkv + h) * p.tile_rows + k;
    f.add_all(p.wg_o + first * kD, p.wg_ml + first * 2, static_cast<int64_t>(p.Hkv) * p.tile_rows, 0, 1, c.n, d);
    f.store(p.out + at * kD + d);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Rows of a (sequence, kv head) pair up to which shares serve: no launches for a
// plan, and lengths balanced to a block.  (Us, shares / tiles, 48 rows a pair, 8 kv
// heads: 16 sequences of 20 to 300 rows 14.6 / 19.8, of 2000 to 3000 48 / 57, 4 of
// 7000 to 8000 37 / 47, 16 behind 2048 shared rows 30 / 50; 64 of 500 to 4000 with up
// to 60 rows 100 / 111.)
constexpr int kFewRows = 64;
// Of these up to 32 go straight from memory to registers, more through LDS: 64 rows
// that way need more than 256 registers (36 us for 16 sequences of 5 tokens of 64
// heads over 8, where the other takes 29).  Up to 16 rows that way alone hands its
// parts over without a launch; from 17 to 32 the two are within 15 % (us, that way / this, 8 kv heads, 64-row
// pages: 16 sequences of 300 to 3000 rows, 20 query rows a pair 27.4 / 23.9, 32 of them
// 28.7 / 25.0; 64 of 500 to 4000, 32 108 / 107; one over 4096, 20 16.9 / 16.2, over 131000,
// 32 110 / 107; 16 behind 2048 shared rows, 20 24.6 / 24.2).
constexpr int kFewDirect = 32;
constexpr int kFewGrid = 512;      // workgroups of shares: two to a CU
constexpr int kTileGrid = 512;     // 128-row tiles at once: two workgroups to a CU
constexpr int kMaxPre = 64;        // key splits of the shared rows

// Rows of a tile.  256 stage a block of keys once for twice the rows, but leave a
// workgroup alone on its CU, half as many tiles to balance, and more of them idle
// in short sequences (us with 128 / 256 rows, 32 q heads over 8: one prompt of 4096
// tokens 221 / 216, 2048 over 2048 174 / 186, 512 26 / 31, six of 1 to 2049 83 / 91; a
// chunk of 509 beside 31 single tokens 75 / 91).
int tile_rows(int rep, int T, int B) { return static_cast<int64_t>(T) * rep >= static_cast<int64_t>(B) * 12288 ? 256 : 128; }

struct PagedPlan {
  int few, nt;        // few rows: 16-row tiles of a pair, 1, 2 or (by mid_run) 4
  int rows, per_head; // of a tile; tile workgroups of a kv head
  int64_t all;        // tiles of all the batch's rows
  int np;             // most key splits of the shared rows
  int most_items, most_cuts;
  size_t plan, row_ml, row_o, wg_ml, wg_o, pre_ml, pre_o;  // byte offsets
  size_t bytes;       // enough for every batch that is no larger
};

// Where a call's workspace has its parts.  The same offsets would do for any
// smaller batch only if it took the same kernel and tiles, so `bytes` counts the
// largest of all their needs, each of which grows with the batch.
PagedPlan make_plan(int Hq, int Hkv, int T, int B, int max_new, bool shared) {
  PagedPlan a{};
  const int rep = Hq / Hkv;
  const size_t rows = static_cast<size_t>(T) * Hq;
  const int64_t R = static_cast<int64_t>(max_new) * rep;
  size_t at = 0, most = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 255) & ~static_cast<size_t>(255);
    return was;
  };
  auto parts = [&](size_t plan, size_t firsts, size_t others) {
    at = BMX_PAGED_COUNTER_BYTES;
    a.plan = take(plan);
    a.row_ml = take(firsts * 2 * sizeof(float));
    a.row_o = take(firsts * kD * sizeof(float));
    a.wg_ml = take(others * 2 * sizeof(float));
    a.wg_o = take(others * kD * sizeof(float));
    most = std::max(most, at);
  };
  auto few = [&]() {
    const int64_t r = std::min<int64_t>(R, kFewRows);
    a.nt = r <= 16 ? 1 : r <= kFewDirect ? 2 : 4;
    parts((1 + static_cast<size_t>(B)) * sizeof(int), rows, static_cast<size_t>(kFewGrid) * 16 * a.nt);
  };
  auto rows_of_tile = [&](int tile_rows) {
    a.rows = tile_rows;
    a.per_head = std::max(1, kTileGrid * 128 / tile_rows / Hkv);
    a.all = (static_cast<int64_t>(T) * rep + tile_rows - 1) / tile_rows;
  };
  auto tile = [&](int tile_rows) {
    rows_of_tile(tile_rows);
    // whole tiles, and as many pieces more as there are workgroups
    const int64_t tiles = a.all + std::min(B, T);
    a.most_items = static_cast<int>(tiles) + 2 * a.per_head;
    a.most_cuts = static_cast<int>(shared ? tiles : std::min<int64_t>(tiles, 2 * a.per_head));
    parts(sizeof(PlanHead) + a.most_items * sizeof(Item) + a.most_cuts * sizeof(Cut), 0,
          static_cast<size_t>(shared ? a.most_items : 2 * a.per_head) * Hkv * tile_rows);
  };
  a.few = R <= kFewRows;
  if (a.few) {
    rows_of_tile(128);  // (the shared rows': of paged_shared_kernel)
    few();
  } else {
    if (rep <= kFewRows) few();
    const int mine = tile_rows(rep, T, B);
    tile(128 + 256 - mine);
    tile(mine);
  }
  if (shared) {
    a.np = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxPre, a.per_head / a.all)));
    // (np splits of T rep rows each: at most per_head tiles, or one split of them all)
    const size_t slots = Hkv * std::min<size_t>(kMaxPre * static_cast<size_t>(T) * rep,
                                                std::max<size_t>(static_cast<size_t>(a.per_head) * a.rows,
                                                                 static_cast<size_t>(T) * rep));
    at = most;
    a.pre_ml = take(slots * 2 * sizeof(float));
    a.pre_o = take(slots * kD * sizeof(float));
    most = at;
  }
  a.bytes = most;
  return a;
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_attention_paged_workspace_bytes(int n_heads, int n_kv_heads, int tokens, int n_seqs,
                                                      int max_new, int shared) {
  if (n_kv_heads <= 0 || n_kv_heads > 1024 || n_heads <= 0 || n_heads > 65535 || n_heads % n_kv_heads ||
      tokens <= 0 || n_seqs <= 0 || n_seqs > kPagedMaxSeqs || max_new < 1 || max_new > tokens ||
      static_cast<int64_t>(tokens) * n_heads > (1 << 28))
    return 0;
  return make_plan(n_heads, n_kv_heads, tokens, n_seqs, max_new, shared != 0).bytes;
}

extern "C" int bmx_attention_paged(const bmx_bf16* q, const bmx_paged_kv* cache, const bmx_batch* batch, bmx_bf16* out,
                                   int n_heads, int head_dim, int shared, float scale, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (int rc = check_paged("attention_paged", cache, batch, n_heads, head_dim)) return rc;
  if (!q || !out || !workspace) return set_error(BMX_E_ARG, "attention_paged: null pointer");
  const int T = batch->tokens, B = batch->n_seqs, Hkv = cache->n_kv_heads;
  if (shared < 0 || shared % cache->page_size || shared > batch->max_pages * cache->page_size)
    return set_error(BMX_E_ARG, "attention_paged: shared=%d must be whole pages of %d, at most %d", shared,
                     cache->page_size, batch->max_pages);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16))
    return set_error(BMX_E_ALIGN, "attention_paged: q, out and workspace must be 16-byte aligned");
  if (T == 0 || B == 0) return BMX_OK;
  const size_t bytes = static_cast<size_t>(T) * n_heads * kD * sizeof(uint16_t);
  if (B == 1) shared = 0;  // (one sequence shares with nobody)
  // (blocks of all pairs are counted in an int)
  const int64_t blocks = (static_cast<int64_t>(batch->max_pages) * cache->page_size + 63) / 64;
  if (B * Hkv * blocks > (1 << 30))
    return set_error(BMX_E_SHAPE, "attention_paged: %d sequences of up to %d pages, %d kv heads: too many", B,
                     batch->max_pages, Hkv);
  const PagedPlan a = make_plan(n_heads, Hkv, T, B, batch->max_new, shared > 0);
  // (and so are those of all tiles)
  if (!a.few && (a.all + std::min(B, T)) * blocks > (1 << 30))
    return set_error(BMX_E_SHAPE, "attention_paged: %d tokens over up to %d pages: too many", T, batch->max_pages);
  if (workspace_bytes < a.bytes)
    return set_error(BMX_E_ARG, "attention_paged: workspace of %zu bytes, %zu needed", workspace_bytes, a.bytes);
  // (of the workspace, what the call uses)
  const Span from{q, bytes}, to{out, bytes}, space{workspace, a.bytes};
  if (overlaps(to, {from}) || over_cache(to, *cache) || over_batch(to, *batch))
    return set_error(BMX_E_ARG, "attention_paged: out overlaps q, the cache or the batch's arrays");
  if (overlaps(space, {from, to}) || over_cache(space, *cache) || over_batch(space, *batch))
    return set_error(BMX_E_ARG, "attention_paged: the workspace overlaps q, out, the cache or the batch's arrays");
  char* ws = static_cast<char*>(workspace);
  auto part = [&](size_t off) { return reinterpret_cast<float*>(ws + off); };
  const int nb = (shared + kTileKeys - 1) / kTileKeys;
  // at least 4 blocks to a split of the shared rows, whose parts have to be joined
  // (us, so / as many splits as fill the CUs, 20 tokens each: 2 sequences behind 2048
  // shared rows 37 / 44, 4 behind 1024 37 / 42, 16 behind 512 45.8 / 47.6, 2 behind 512
  // 33.9 / 31.4; 2 single tokens behind 512 14.5 / 11.8)
  // -- nor more than the shared rows' part of the places, where the sequences' own
  // are few: a pair's, whose lengths are not known here, for three blocks of a tile
  // (us, so / without: 64 single tokens over 4096 shared rows 28.1 / 31.0, 160 over 2048
  // 36.3 / 40.9, 30 of one q head a kv head over 16384 25.2 / 28.2, 200 over 4096
  // 55.8 / 60.1; 32 over 8192, 64 over 1024, 160 over 32768 alike; with two blocks
  // 31.0, 35.1, 27.9, 56.4, with five 29.5, 43.1, 25.5, 57.4 and 160 over 32768 170 for 164)
  int splits = std::min(a.np, (nb + 3) / 4);
  const int64_t pairs = static_cast<int64_t>(B) * Hkv, pre_tiles = Hkv * a.all;
  if (a.few && splits > 1) {
    const int64_t places = kFewGrid * pre_tiles * nb / (pre_tiles * nb + 3 * pairs);
    splits = static_cast<int>(std::min<int64_t>(splits, std::max<int64_t>(1, (places + pre_tiles / 2) / pre_tiles)));
  }
  const int bps = splits ? (nb + splits - 1) / splits : 0;
  const int np = bps ? (nb + bps - 1) / bps : 0;
  PagedAttn p{q, cache->k, cache->v, out, batch->starts, batch->lens, batch->pages, B, batch->max_pages, T,
                    batch->max_new, n_heads, Hkv, n_heads / Hkv, cache->n_pages, log2_of(cache->page_size), shared,
                    fabsf(scale) * kLog2e, scale < 0.0f ? 0x80008000u : 0u, reinterpret_cast<int*>(ws + a.plan),
                    part(a.row_o), part(a.row_ml), part(a.wg_o), part(a.wg_ml), part(a.pre_o), part(a.pre_ml), np, bps,
                    a.most_items, a.most_cuts, a.rows, a.nt == 4 ? 6 : 7, nullptr};
  p.c2 = p.c2 < kLeast ? kLeast : p.c2;
  const hipStream_t st = as_stream(stream);
  if (a.few) {
    // Where a pair's workgroups have few parts between them, they hand these to
    // the last of them; a launch that spreads the rows over the card joins many.
    // (Us, handed / launch: 160 sequences of 20 to 300 rows, 4 query rows a pair
    // 20.9 / 24.7, 4 of 200 to 900 9.5 / 11.2, 64 of 500 to 8191 134 / 136; 1 of 4097,
    // 33 parts a row 14.4 / 13.0; 4 with 28 query rows a pair 20.5 / 14.3; with
    // parts over shared rows as well, 64 sequences 50 / 34.)
    const int most_blocks = (batch->max_pages * cache->page_size + kFewKeys - 1) / kFewKeys;
    const int64_t pieces = std::min<int64_t>(kFewGrid / pairs, most_blocks) + 1;
    if (a.nt == 1 && !shared && pairs <= kMaxCounters && static_cast<int64_t>(batch->max_new) * p.rep * pieces <= 96)
      p.cnt = reinterpret_cast<unsigned*>(ws);
    // (few rows have many parts each; us with 8 rows / 1 row to a workgroup: 64
    // sequences, 32 rows each, over 4096 shared keys 35.1 / 41.2, 1 of 4097 15.7 / 13.4)
    const bool wide = static_cast<int64_t>(T) * n_heads <= 1024;
    const int rows = batch->max_new * p.rep;
    const dim3 merge(wide ? rows : (rows + 7) / 8, Hkv, B);
    auto launch = [&](auto few, auto with_shared, auto joint, auto joint_wide) {
      const size_t lds = shared || a.nt == 4 ? kMidLds : 0;
      if (int rc = shared ? allow_lds(with_shared, lds) : allow_lds(few, lds)) return rc;
      const int pre = shared ? Hkv * static_cast<int>(a.all) * np : 0;
      // Shares for the places that the shared rows' tiles leave of a round, so that
      // none waits for a place -- if that is a quarter of them and they get four
      // pairs each at most.  (Us, so / always kFewGrid: 64 tokens over 4096 shared rows
      // 28.1 / 31.5, 32 over 8192 26.7 / 28.8, 160 over 2048 36.3 / 41.0; 160 over 512 or
      // 32768, 64 over 2048 with 500 to 3000 of their own alike.)
      const int left = kFewGrid - pre % kFewGrid;
      const int few_grid = 4 * left >= kFewGrid && pairs <= 4 * left ? left : kFewGrid;
      if (shared) hipLaunchKernelGGL(with_shared, dim3(pre + few_grid), dim3(256), lds, st, p, pre);
      else hipLaunchKernelGGL(few, dim3(kFewGrid), dim3(256), lds, st, p);
      if (int rc = check_launch("attention_paged")) return rc;
      if (p.cnt) return 0;
      if (wide) hipLaunchKernelGGL(joint_wide, merge, dim3(256), 0, st, p);
      else hipLaunchKernelGGL(joint, merge, dim3(256), 0, st, p);
      return check_launch("attention_paged merge");
    };
    if (a.nt == 1) return launch(paged_few_kernel<1>, paged_shared_kernel<1>, paged_few_merge_kernel<1, false>,
                                  paged_few_merge_kernel<1, true>);
    if (a.nt == 2) return launch(paged_few_kernel<2>, paged_shared_kernel<2>, paged_few_merge_kernel<2, false>,
                                  paged_few_merge_kernel<2, true>);
    return launch(paged_mid_kernel, paged_shared_kernel<4>, paged_few_merge_kernel<4, false>, paged_few_merge_kernel<4, true>);
  }
  if (shared) {
    if (a.all > 65535) return set_error(BMX_E_SHAPE, "attention_paged: tokens=%d too many for shared rows", T);
    const auto kernel = a.rows == 256 ? paged_prefix_kernel<8> : paged_prefix_kernel<4>;
    if (int rc = allow_lds(kernel, kTileLds)) return rc;
    hipLaunchKernelGGL(kernel, dim3(Hkv, static_cast<unsigned>(a.all), np), dim3(2 * a.rows), kTileLds, st, p);
    if (int rc = check_launch("attention_paged shared rows")) return rc;
  }
  const auto kernel = a.rows == 256 ? paged_tile_kernel<8> : paged_tile_kernel<4>;
  if (int rc = allow_lds(kernel, kTileLds)) return rc;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p, a.per_head);
  hipLaunchKernelGGL(kernel, dim3(a.per_head * Hkv), dim3(2 * a.rows), kTileLds, st, p);
  hipLaunchKernelGGL(paged_tile_merge_kernel, dim3(kTileMergeGrid), dim3(256), 0, st, p);
  return check_launch("attention_paged");
}
