// The 4-bit KV cache: argument checks and device helpers shared by the
// kernels that write, read, attend over and cut it.
//
// A cached row is 128 values in two groups of 64; value d is
//   s[d / 64] * n[d] + b[d / 64],  n = (word[d / 8] >> 4 (d % 8)) & 15,
// with bf16 s and b (the MLX affine format of the framework's weights).
#pragma once

#include "bmx_device.h"

namespace bmx {

constexpr int kKv4Dim = 128;                 // head_dim
constexpr int kKv4Words = 16;                // words per row
constexpr int kKv4MaxCapacity = 65535 * 256;  // rows: a head's words stay below 2^31 bytes, 256 keys a grid row

// Checks of the struct itself; `what` names the entry point.
int check_kv4(const char* what, const bmx_kv4* c, int head_dim);
// ... and of rows [offset, offset + M) in it
int check_kv4_rows(const char* what, const bmx_kv4* c, int M, int offset);

// Whether a bytes from x and b bytes from y have any in common
inline bool kv4_overlap(const void* x, size_t a, const void* y, size_t b) {
  const uintptr_t i = reinterpret_cast<uintptr_t>(x), j = reinterpret_cast<uintptr_t>(y);
  return i < j + b && j < i + a;
}

// bmx_kv4_read, checked arguments
int launch_kv4_read(const bmx_kv4& c, uint16_t* k, uint16_t* v, int M, int start, hipStream_t stream);

// Scale of a group from its smallest and largest value; NaN if `nan` (the
// group holds a NaN) or the range is not finite.
__device__ __forceinline__ uint16_t kv4_scale(float lo, float hi, bool nan) {
  const float range = hi - lo;
  return nan || !(range <= 3.402823466e38f) ? 0x7fc0u : f2bf(range / 15.0f);
}
// Nibble of x under the stored scale s (as a float; r = 1 / s) and the group's
// minimum: rne((x - lo) / s), at most 15.  The quotient is formed as (x - lo)
// r, off by less than 2^-21 of at most 16 from the rounded quotient; only
// within 2^-17 of a half step can that round to another number, and there (and
// where r is infinite) the division itself decides.
__device__ __forceinline__ uint32_t kv4_nibble(float x, float lo, float s, float r) {
  const float d = x - lo;
  float t = d * r, n = rintf(t);
  if (!(fabsf(fabsf(t - n) - 0.5f) >= 7.62939453125e-6f)) n = rintf(d / s);
  // s = 0 gives NaN or inf, s = NaN gives NaN: both pack as 0 and read back as lo and NaN
  return s > 0.0f ? static_cast<uint32_t>(fminf(n, 15.0f)) : 0u;
}
// The smallest and largest of a value over 64 lanes
__device__ __forceinline__ float kv4_max64(float v) { return max_xor32(max_xor16(row16_max(v))); }
__device__ __forceinline__ float kv4_min64(float v) { return -kv4_max64(-v); }

}  // namespace bmx
