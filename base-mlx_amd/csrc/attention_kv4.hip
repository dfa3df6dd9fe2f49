// Attention over the 4-bit KV cache, and the weight each cached position
// drew (gfx950).
//
//   S[t, j] = scale * sum_d q[t, d] (s n + b)[j, d],  j <= offset + t
//   P = softmax(S),  out = bf16(P (s n + b)),  weights[h, j] += sum P[., j]
// With Q_g the sum of q over group g, a score is
//   scale * sum_g (s_g sum_d q_d n_d + b_g Q_g).
#include <math.h>

#include "kv4.h"

namespace bmx {
namespace {

struct Kv4AttnParams {
  const uint16_t* q;  // [Hq, M, 128]
  bmx_kv4 c;
  uint16_t* out;   // [M, Hq*128]
  float* lse;      // [Hq, M] log of the softmax's sum, or null
  float* weights;  // [Hkv, cap], or null
  int Hq, M, offset;
  float scale;
};

// Dot product of q (LDS, fp32) with row `slot`'s keys.
__device__ __forceinline__ float kv4_score(const float* q, const float* qsum, const bmx_kv4& c, int64_t slot,
                                           float scale) {
  const uint32_t* w = c.k + slot * kKv4Words;
  float s = 0.0f;
#pragma unroll
  for (int g = 0; g < 2; g++) {
    float d = 0.0f;
    for (int i = 0; i < 8; i++) {
      const uint32_t wd = w[8 * g + i];
#pragma unroll
      for (int e = 0; e < 8; e++)
        d = __builtin_fmaf(q[64 * g + 8 * i + e], static_cast<float>((wd >> (4 * e)) & 15u), d);
    }
    s = __builtin_fmaf(bf2f(c.k_scales[2 * slot + g]), d, s);
    s = __builtin_fmaf(bf2f(c.k_biases[2 * slot + g]), qsum[g], s);
  }
  return s * scale;
}

template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* tmp) {
  for (int o = 1; o < 64; o <<= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  return MAX ? fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3])) : (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
}

// One workgroup per (token, q head), 256 keys at a time.
__global__ void __launch_bounds__(256) kv4_attn_kernel(const Kv4AttnParams p) {
  __shared__ float q[kKv4Dim], qsum[2], tmp[4], ps[256], os[256];
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int64_t base = static_cast<int64_t>(h / (p.Hq / p.c.n_kv_heads)) * p.c.capacity;
  if (tid < kKv4Dim) q[tid] = bf2f(p.q[(static_cast<int64_t>(h) * p.M + t) * kKv4Dim + tid]);
  __syncthreads();
  if (tid < 2) {
    float s = 0.0f;
    for (int i = 0; i < 64; i++) s += q[64 * tid + i];
    qsum[tid] = s;
  }
  __syncthreads();
  const int L = p.offset + t + 1;
  float mx = -INFINITY, l = 0.0f, o = 0.0f;
  const int d = tid & 127, half = tid >> 7;
  for (int j0 = 0; j0 < L; j0 += 256) {
    const int j = j0 + tid;
    const float s = j < L ? kv4_score(q, qsum, p.c, base + j, p.scale) : -INFINITY;
    const float nm = fmaxf(mx, block_reduce<true>(s, tmp));
    const float e = nm == -INFINITY ? 0.0f : expf(s - nm), a = nm == -INFINITY ? 1.0f : expf(mx - nm);
    ps[tid] = s != s ? s : e;
    l = l * a + block_reduce<false>(ps[tid], tmp);
    o *= a;
    mx = nm;
    __syncthreads();
    for (int i = half; i < 256 && j0 + i < L; i += 2) {
      const int64_t slot = base + j0 + i;
      const float n = static_cast<float>((p.c.v[slot * kKv4Words + d / 8] >> (4 * (d & 7))) & 15u);
      const float v = __builtin_fmaf(bf2f(p.c.v_scales[2 * slot + d / 64]), n, bf2f(p.c.v_biases[2 * slot + d / 64]));
      o = __builtin_fmaf(ps[i], v, o);
    }
    __syncthreads();
  }
  os[tid] = o;
  __syncthreads();
  if (tid < kKv4Dim)
    p.out[(static_cast<int64_t>(t) * p.Hq + h) * kKv4Dim + tid] = f2bf((os[tid] + os[tid + 128]) / l);
  if (p.lse && tid == 0) p.lse[static_cast<int64_t>(h) * p.M + t] = mx + logf(l);
}

// One thread per cached row; every query row of its kv head in turn.
__global__ void __launch_bounds__(256) kv4_weigh_kernel(const Kv4AttnParams p) {
  __shared__ float q[kKv4Dim], qsum[2];
  const int rep = p.Hq / p.c.n_kv_heads, h = blockIdx.y;
  const int j = blockIdx.x * 256 + threadIdx.x;
  const int64_t slot = static_cast<int64_t>(h) * p.c.capacity + j;
  float acc = 0.0f;
  for (int r = 0; r < rep * p.M; r++) {
    const int t = r % p.M;
    const int64_t row = static_cast<int64_t>(h) * rep * p.M + r;
    __syncthreads();
    if (threadIdx.x < kKv4Dim) q[threadIdx.x] = bf2f(p.q[row * kKv4Dim + threadIdx.x]);
    __syncthreads();
    if (threadIdx.x < 2) {
      float s = 0.0f;
      for (int i = 0; i < 64; i++) s += q[64 * threadIdx.x + i];
      qsum[threadIdx.x] = s;
    }
    __syncthreads();
    if (j <= p.offset + t) acc += expf(kv4_score(q, qsum, p.c, slot, p.scale) - p.lse[row]);
  }
  if (j < p.offset + p.M) p.weights[slot] += acc;
}

constexpr int64_t kMaxRows = 1 << 28;  // Hq * M of a call

bool attn_shape_ok(int Hq, int Hkv, int M, int64_t L) {
  return Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0 && M > 0 && L >= M &&
         L <= kKv4MaxCapacity && static_cast<int64_t>(Hq) * M <= kMaxRows;
}

size_t attn_workspace_bytes(int Hq, int Hkv, int M, int L, bool weigh) {
  return BMX_KV4_COUNTER_BYTES + (weigh ? static_cast<size_t>(Hq) * M * sizeof(float) : 0);
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_attention_kv4_workspace_bytes(int n_heads, int n_kv_heads, int M, int L, int weigh) {
  return attn_shape_ok(n_heads, n_kv_heads, M, L) ? attn_workspace_bytes(n_heads, n_kv_heads, M, L, weigh != 0) : 0;
}

extern "C" int bmx_attention_gqa_kv4(const bmx_bf16* q, const bmx_kv4* cache, bmx_bf16* out, float* weights,
                                     int n_heads, int M, int head_dim, int offset, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (int rc = check_kv4("attention_kv4", cache, head_dim)) return rc;
  if (!q || !out || !workspace) return set_error(BMX_E_ARG, "attention_kv4: null pointer");
  if (M < 0 || n_heads <= 0 || n_heads % cache->n_kv_heads)
    return set_error(BMX_E_SHAPE, "attention_kv4: M=%d, %d heads over %d kv heads", M, n_heads, cache->n_kv_heads);
  if (int rc = check_kv4_rows("attention_kv4", cache, M, offset)) return rc;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(weights, 16))
    return set_error(BMX_E_ALIGN, "attention_kv4: q, out, weights and workspace must be 16-byte aligned");
  if (M == 0) return BMX_OK;
  if (!attn_shape_ok(n_heads, cache->n_kv_heads, M, static_cast<int64_t>(offset) + M))
    return set_error(BMX_E_SHAPE, "attention_kv4: %d heads, M=%d too large for one call", n_heads, M);
  const size_t need = attn_workspace_bytes(n_heads, cache->n_kv_heads, M, offset + M, weights != nullptr);
  if (workspace_bytes < need)
    return set_error(BMX_E_ARG, "attention_kv4: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  float* lse = weights ? reinterpret_cast<float*>(static_cast<char*>(workspace) + BMX_KV4_COUNTER_BYTES) : nullptr;
  const Kv4AttnParams p{q, *cache, out, lse, weights, n_heads, M, offset, scale};
  hipLaunchKernelGGL(kv4_attn_kernel, dim3(M, n_heads), dim3(256), 0, as_stream(stream), p);
  if (int rc = check_launch("attention_kv4")) return rc;
  if (!weights) return BMX_OK;
  hipLaunchKernelGGL(kv4_weigh_kernel, dim3((offset + M + 255) / 256, cache->n_kv_heads), dim3(256), 0,
                     as_stream(stream), p);
  return check_launch("attention_kv4 weights");
}
