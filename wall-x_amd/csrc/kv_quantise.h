// A row of a key / value cache in e4m3 (kv_cache.hip, paged_cache.hip): scale = max |x| / 448 (at least 2^-126), code = e4m3(x / scale), to
// nearest even.
#pragma once

#include "common.h"

namespace wx {

// x / scale, correctly rounded: r is 1 / scale to nearest, the remainder of x r is exact in one fused multiply-add
__device__ __forceinline__ float quotient(float x, float scale, float r) {
  const float q = x * r;
  return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, scale, x), r, q), x);  // (-0 stays -0)
}

template <int DT, int L>
__device__ __forceinline__ void quantise(const float* x, float& scale, uint32_t (&codes)[2]) {
  // largest magnitude by its bits: a NaN compares above everything and stays
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < L; d <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
  scale = __uint_as_float(top) / 448.f;
  scale = scale < 0x1p-126f ? 0x1p-126f : scale;
  float y[8];
  if (scale < __builtin_huge_valf()) {
    const float r = 1.f / scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = quotient(x[e], scale, r);
  } else {  // not finite: the row reads back as NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] / scale;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * u], y[4 * u + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * u + 2], y[4 * u + 3], w, true);
    codes[u] = static_cast<uint32_t>(w);
  }
}

}  // namespace wx
