// Attention of requests' newest tokens over a paged key / value cache (gfx950).
#include "attention.h"
#include "common.h"

namespace wx {
namespace {

struct PagedArgs {
  const uint16_t* q;               // [batch, n_q, seq, D] through strides; token t is position t % seq of row t / seq
  int64_t qs[3];
  const void *k, *v;               // [pages, n_kv, page_size, D]
  const float *k_scale, *v_scale;  // e4m3: [pages, n_kv, page_size]
  uint16_t* out;                   // [tokens, n_q, D]
  const int32_t *table, *lengths, *starts;  // [requests, width], [requests], [requests + 1] or null: seq tokens each
  int causal, tokens, requests, n_q, n_kv, group, seq, width, page_size, n_pages;
  Divider by_seq, by_page, by_q;
  float c;                         // scale * log2(e)
};

// The first version: a wavefront per token and query head, a key per lane.
template <int DT, int D, bool F8>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedArgs a) {
  const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = a.by_q.div(id), hq = id - t * a.n_q;
  if (t >= a.tokens) return;
  const int hk = hq / a.group;
  int req = -1, i = 0, n = 0;
  for (int r = 0; r < a.requests; ++r) {
    const int from = a.starts ? min(max(a.starts[r], 0), a.tokens) : r * a.seq, to = a.starts ? min(a.starts[r + 1], a.tokens) : from + a.seq;
    if (t >= from && t < to) req = r, i = t - from, n = to - from;
  }
  float o[2] = {0.f, 0.f}, m = -kInf, l = 0.f;
  if (req >= 0) {
    const int b = a.by_seq.div(t);
    const uint16_t* q = a.q + b * a.qs[0] + hq * a.qs[1] + static_cast<int64_t>(t - b * a.seq) * a.qs[2];
    const int length = min(max(a.lengths[req], 0), a.width * a.page_size), hi = a.causal ? min(length, length - n + i + 1) : length;
    for (int k0 = 0; k0 < hi; k0 += 64) {
      const int key = min(k0 + lane, hi - 1), place = a.by_page.div(key), page = a.table[static_cast<int64_t>(req) * a.width + place];
      const bool there = k0 + lane < hi && page >= 0 && page < a.n_pages;
      const int64_t row = (static_cast<int64_t>(there ? page : 0) * a.n_kv + hk) * a.page_size + key - place * a.page_size;
      float s = 0.f;
      for (int c = 0; c < D; c += 2) {
        float x0, x1;
        if constexpr (F8) {
          const int w = static_cast<const uint16_t*>(a.k)[(row * D + c) / 2];
          x0 = __builtin_amdgcn_cvt_f32_fp8(w, 0), x1 = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        } else {
          const uint32_t w = static_cast<const uint32_t*>(a.k)[(row * D + c) / 2];
          x0 = Elem<DT>::load(w & 0xffffu), x1 = Elem<DT>::load(w >> 16);
        }
        s += x0 * Elem<DT>::load(q[c]);
        s += x1 * Elem<DT>::load(q[c + 1]);
      }
      if constexpr (F8) s *= a.k_scale[row];
      s = there ? s : -kInf;
      const float top = wave_max(s), mn = fmaxf(m, top), alpha = mn == -kInf ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
      m = mn;
      const float p = there ? __builtin_amdgcn_exp2f((s - (m == -kInf ? 0.f : m)) * a.c) : 0.f;
      l = l * alpha + wave_sum(p);
      o[0] *= alpha, o[1] *= alpha;
      const uint64_t seen = __ballot(there);
      for (int j = 0; j < 64; ++j) {
        if (!(seen >> j & 1)) continue;
        const float pj = __shfl(p, j);
        const int64_t r = (static_cast<int64_t>(__shfl(static_cast<int>(row >> 32), j)) << 32) | static_cast<uint32_t>(__shfl(static_cast<int>(row), j));
        for (int u = 0; u < 2; ++u)
          if (lane + 64 * u < D) {
            const int64_t e = r * D + lane + 64 * u;
            o[u] += pj * (F8 ? __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(a.v)[e], 0) * a.v_scale[r] : Elem<DT>::load(static_cast<const uint16_t*>(a.v)[e]));
          }
      }
    }
  }
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < D) a.out[(static_cast<int64_t>(t) * a.n_q + hq) * D + lane + 64 * u] = static_cast<uint16_t>(Elem<DT>::store(m == -kInf && l == 0.f ? 0.f : o[u] / l));
}

template <int DT, bool F8>
int launch(const PagedArgs& a, int head_dim, hipStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * a.n_q + 3) / 4;
  if (too_many_blocks(blocks, 256)) return fail(WX_ERR_UNSUPPORTED, "wx_paged_attention: too many tokens");
  const dim3 grid(static_cast<unsigned>(blocks));
  if (head_dim == 64) hipLaunchKernelGGL((paged_attn_kernel<DT, 64, F8>), grid, dim3(256), 0, s, a);
  else if (head_dim == 80) hipLaunchKernelGGL((paged_attn_kernel<DT, 80, F8>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((paged_attn_kernel<DT, 128, F8>), grid, dim3(256), 0, s, a);
  return check_launch("wx_paged_attention");
}

}  // namespace
}  // namespace wx

using namespace wx;

extern "C" size_t wx_paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int n_q_heads, int n_kv_heads, int head_dim) {
  (void)tokens, (void)requests, (void)n_q_heads, (void)n_kv_heads, (void)head_dim;
  return 0;
}

extern "C" int wx_paged_attention(const void* q, const void* k_pages, const void* v_pages, const float* k_scale, const float* v_scale, void* out,
                                  const int32_t* page_table, const int32_t* lengths, const int32_t* starts, int causal, int64_t batch, int n_q_heads,
                                  int n_kv_heads, int64_t seq, int64_t requests, int64_t pages_per_request, int64_t num_pages, int page_size,
                                  int head_dim, const int64_t q_strides[3], float scale, int dtype, void* workspace, size_t workspace_bytes,
                                  wx_stream_t stream) {
  const char* who = "wx_paged_attention";
  if (batch < 0 || n_q_heads < 0 || n_kv_heads < 0 || seq < 0 || requests < 0 || pages_per_request < 0 || num_pages < 0)
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (page_size <= 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: page_size must be positive", who);
  if (head_dim != 64 && head_dim != 80 && head_dim != 128) return fail(WX_ERR_UNSUPPORTED, "%s: head_dim %d must be 64, 80 or 128", who, head_dim);
  if (dtype != WX_BF16 && dtype != WX_F16) return fail(WX_ERR_UNSUPPORTED, "%s: dtype %d must be bf16 or fp16", who, dtype);
  if (n_kv_heads == 0 ? n_q_heads != 0 : n_q_heads % n_kv_heads != 0)
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: %d query heads are no multiple of %d key / value heads", who, n_q_heads, n_kv_heads);
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", who);
  if (!q_strides) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null strides", who);
  if ((k_scale == nullptr) != (v_scale == nullptr)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: scales of keys and values, or neither", who);
  if (!starts && requests != batch) return fail(WX_ERR_INVALID_ARGUMENT, "%s: without starts a request is a row of q", who);
  if (batch == 0 || n_q_heads == 0 || seq == 0) return WX_OK;
  const int group = n_q_heads / n_kv_heads;
  if (group > 1024) return fail(WX_ERR_UNSUPPORTED, "%s: more than 1024 query heads to a key / value head", who);
  if (seq > 0x3fffffffll / n_q_heads || batch > 0x3fffffffll / (seq * n_q_heads)) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 rows", who);
  if (requests > 0x3fffffffll || pages_per_request > 0x3fffffffll / page_size) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 keys to a request", who);
  if (num_pages > 0x7fffffffll / page_size) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", who);
  if (!q || !out || (requests > 0 && (!lengths || (pages_per_request > 0 && num_pages > 0 && (!page_table || !k_pages || !v_pages)))))
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  for (const void* p : {q, k_pages, v_pages, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0 || q_strides[i] < 0) return fail(WX_ERR_UNSUPPORTED, "%s: q's strides must be positive and keep rows 16-byte aligned", who);
  (void)workspace, (void)workspace_bytes;
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.k = k_pages, a.v = v_pages, a.k_scale = k_scale, a.v_scale = v_scale, a.out = static_cast<uint16_t*>(out);
  a.table = page_table, a.lengths = lengths, a.starts = starts, a.causal = causal != 0;
  a.tokens = static_cast<int>(batch * seq), a.requests = static_cast<int>(requests), a.n_q = n_q_heads, a.n_kv = n_kv_heads, a.group = group;
  a.seq = static_cast<int>(seq), a.width = num_pages ? static_cast<int>(pages_per_request) : 0, a.page_size = page_size, a.n_pages = static_cast<int>(num_pages);
  a.by_seq = Divider(static_cast<uint32_t>(seq)), a.by_page = Divider(page_size), a.by_q = Divider(n_q_heads);
  a.c = scale * kLog2e;
  hipStream_t s = as_stream(stream);
  if (dtype == WX_BF16) return k_scale ? launch<WX_BF16, true>(a, head_dim, s) : launch<WX_BF16, false>(a, head_dim, s);
  return k_scale ? launch<WX_F16, true>(a, head_dim, s) : launch<WX_F16, false>(a, head_dim, s);
}
