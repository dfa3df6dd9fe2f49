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

// bmx_kv4_read, checked arguments
int launch_kv4_read(const bmx_kv4& c, uint16_t* k, uint16_t* v, int M, int start, hipStream_t stream);

// Scale of a group from its smallest and largest value; NaN if `nan` (the
// group holds a NaN) or the range is not finite.
__device__ __forceinline__ uint16_t kv4_scale(float lo, float hi, bool nan) {
  const float range = hi - lo;
  return nan || !(range <= 3.402823466e38f) ? 0x7fc0u : f2bf(range / 15.0f);
}
// Nibble of x under the stored scale (as a float) and the group's minimum.
__device__ __forceinline__ uint32_t kv4_nibble(float x, float lo, float s) {
  const float n = rintf((x - lo) / s);
  // s = 0 gives NaN or inf, s = NaN gives NaN: both pack as 0 and read back as lo and NaN
  return s > 0.0f ? static_cast<uint32_t>(fminf(n, 15.0f)) : 0u;
}

}  // namespace bmx
