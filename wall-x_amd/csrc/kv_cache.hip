// Quantises keys and values into an e4m3 cache as they are written (gfx950).
//
// Of each token and key / value head: scale = max |x| / 448 (at least 2^-126), code = e4m3(x / scale), to nearest even.
// One pass, HBM-bound: 2 D bytes in, D + 4 out, for keys and values alike.  A group of 8 or 16 lanes owns one such row of both (16
// bytes of each a lane), finds the row's largest magnitude through lane exchanges and stores the 8 codes a lane as 8 bytes.
#include "attention.h"
#include "common.h"

namespace wx {
namespace {

struct CacheArgs {
  const uint16_t *k, *v;       // [batch, n_kv, seq, D] through strides
  int64_t ks[3], vs[3];
  uint8_t *k_cache, *v_cache;  // [batch, n_kv, capacity, D]
  float *k_scale, *v_scale;    // [batch, n_kv, capacity]
  const int32_t *start, *lengths;
  int rows;                    // of one of the batch: seq * n_kv
  int n_kv;
  Divider by_kv, by_blocks;    // by_blocks: workgroups to one of the batch
  int64_t capacity;
};

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

// A workgroup's rows are of one of the batch, whose start and length are then uniform.  64 x 880 tokens of 2 heads of 128 (66 MB): 14.0 us
// in the kernel, 4.7 TB/s (17.9 with the rows numbered through in 64 bits and non-temporal loads; two rows to a group of lanes change
// nothing).
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(CacheArgs a) {
  constexpr int L = D == 64 ? 8 : 16, kGroups = 256 / L;  // lanes a row (10 of 16 work for D = 80)
  const int b = a.by_blocks.div(blockIdx.x), c = threadIdx.x % L;
  const int at = (static_cast<int>(blockIdx.x) - b * static_cast<int>(a.by_blocks.d)) * kGroups + static_cast<int>(threadIdx.x) / L;
  const int s = a.by_kv.div(at), hk = at - s * a.n_kv;
  const int64_t pos = static_cast<int64_t>(a.start[b]) + s;
  if (at >= a.rows || pos < 0 || pos >= a.capacity || (a.lengths != nullptr && s >= a.lengths[b])) return;  // (a whole group of lanes)
  const bool mine = c * 8 < D;
  float xk[8] = {}, xv[8] = {};
  if (mine) {
    const u32x4 k = *reinterpret_cast<const u32x4*>(a.k + b * a.ks[0] + hk * a.ks[1] + s * a.ks[2] + 8 * c);
    const u32x4 v = *reinterpret_cast<const u32x4*>(a.v + b * a.vs[0] + hk * a.vs[1] + s * a.vs[2] + 8 * c);
    unpack16<DT>(k, xk);
    unpack16<DT>(v, xv);
  }
  float k_scale, v_scale;
  uint32_t kc[2], vc[2];
  quantise<DT, L>(xk, k_scale, kc);
  quantise<DT, L>(xv, v_scale, vc);
  const int64_t row = (static_cast<int64_t>(b) * a.n_kv + hk) * a.capacity + pos;
  if (mine) {
    *reinterpret_cast<uint2*>(a.k_cache + row * D + 8 * c) = uint2{kc[0], kc[1]};
    *reinterpret_cast<uint2*>(a.v_cache + row * D + 8 * c) = uint2{vc[0], vc[1]};
  }
  if (c == 0) {
    a.k_scale[row] = k_scale;
    a.v_scale[row] = v_scale;
  }
}

}  // namespace
}  // namespace wx

using namespace wx;

extern "C" int wx_kv_cache_write(const void* k, const void* v, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                 const int32_t* start, const int32_t* lengths, int64_t batch, int n_kv_heads, int64_t seq,
                                 int64_t capacity, int head_dim, const int64_t k_strides[3], const int64_t v_strides[3], int dtype,
                                 wx_stream_t stream) {
  const char* who = "wx_kv_cache_write";
  if (batch < 0 || n_kv_heads < 0 || seq < 0 || capacity < 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (head_dim != 64 && head_dim != 80 && head_dim != 128) return fail(WX_ERR_UNSUPPORTED, "%s: head_dim %d must be 64, 80 or 128", who, head_dim);
  if (dtype != WX_BF16 && dtype != WX_F16) return fail(WX_ERR_UNSUPPORTED, "%s: dtype %d must be bf16 or fp16", who, dtype);
  if (!k_strides || !v_strides) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null strides", who);
  if (batch == 0 || n_kv_heads == 0 || seq == 0 || capacity == 0) return WX_OK;
  if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !start) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  for (const void* p : {k, v, static_cast<const void*>(k_cache), static_cast<const void*>(v_cache)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return fail(WX_ERR_UNSUPPORTED, "%s: strides must keep rows 16-byte aligned", who);
  if (seq > 0x7fffffffll / n_kv_heads || batch > 0x7fffffffll) return fail(WX_ERR_UNSUPPORTED, "%s: too many tokens", who);
  CacheArgs a{};
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  for (int i = 0; i < 3; ++i) a.ks[i] = k_strides[i], a.vs[i] = v_strides[i];
  a.k_cache = static_cast<uint8_t*>(k_cache), a.v_cache = static_cast<uint8_t*>(v_cache), a.k_scale = k_scale, a.v_scale = v_scale;
  a.start = start, a.lengths = lengths;
  a.rows = static_cast<int>(seq * n_kv_heads), a.n_kv = n_kv_heads, a.capacity = capacity;
  const int64_t each = 256 / (head_dim == 64 ? 8 : 16), of_one = (a.rows + each - 1) / each, blocks = batch * of_one;
  a.by_kv = Divider(n_kv_heads), a.by_blocks = Divider(static_cast<uint32_t>(of_one));
  if (too_many_blocks(blocks, 256)) return fail(WX_ERR_UNSUPPORTED, "%s: too many tokens", who);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  hipStream_t s = as_stream(stream);
#define WX_CACHE(DT)                                                                                            \
  if (head_dim == 64) hipLaunchKernelGGL((kv_cache_write_kernel<DT, 64>), grid, block, 0, s, a);                \
  else if (head_dim == 80) hipLaunchKernelGGL((kv_cache_write_kernel<DT, 80>), grid, block, 0, s, a);           \
  else hipLaunchKernelGGL((kv_cache_write_kernel<DT, 128>), grid, block, 0, s, a)
  if (dtype == WX_BF16) {
    WX_CACHE(WX_BF16);
  } else {
    WX_CACHE(WX_F16);
  }
#undef WX_CACHE
  return check_launch(who);
}
