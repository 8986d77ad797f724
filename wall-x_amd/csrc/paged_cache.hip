// The bookkeeping of a paged key / value cache and the write into it (gfx950).
//
// Pages.  Request r of lengths[r] tokens owns the first ceil(lengths[r] / page_size) entries of its row of the page table; pages that nobody
// owns are a stack.  A resize frees pages of requests that shrink and grants pages to those that grow: freed page i (counted by request,
// then by place) goes to place count + freed - 1 - i of the stack, grant j takes place count + freed - 1 - j.  So grants take freed
// pages first, a growth that is taken back leaves the stack as it was, and both are closed forms of two prefix sums over the requests.
#include <algorithm>

#include "attention.h"
#include "common.h"
#include "kv_quantise.h"

namespace wx {
namespace {

constexpr int kMaxRequests = 4096;  // of one call: five numbers each in LDS

struct ResizeArgs {
  const int32_t *lengths, *wanted;  // [requests]
  int32_t *table;                   // [requests, width]
  int32_t *stack;                   // [stack_size]
  const int32_t *count;
  int32_t *new_lengths, *new_count, *starts, *slots;
  int64_t* positions;
  int requests, width, stack_size, page_size, max_tokens;
  Divider by_page;
};

// In-place exclusive prefix sums of s[0 .. n), total in s[n], by 256 threads.
__device__ __forceinline__ void block_prefix(int* s, int n) {
  __shared__ int wave_sums[4];
  const int tid = threadIdx.x, lane = tid & 63, each = (n + 255) / 256, first = min(tid * each, n), last = min(first + each, n);
  int mine = 0;
  for (int i = first; i < last; ++i) mine += s[i];
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == 63) wave_sums[tid >> 6] = sum;
  __syncthreads();
  int at = sum - mine;
  for (int w = 0; w < tid >> 6; ++w) at += wave_sums[w];
  for (int i = first; i < last; ++i) {
    const int x = s[i];
    s[i] = at;
    at += x;
  }
  if (tid == 255) s[n] = at;
  __syncthreads();
}

// The largest r with prefix[r] <= x: of equal ones, whose requests have nothing, the last, which owns x.
__device__ __forceinline__ int owner(const int* prefix, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(256) void paged_resize_kernel(ResizeArgs a) {
  __shared__ int lds[5 * kMaxRequests + 3];
  const int R = a.requests, tid = threadIdx.x;
  int *held = lds, *want = held + R, *given = want + R, *taken = given + R + 1, *tokens = taken + R + 1;
  const int most = a.width * a.page_size;
  auto pages = [&](int n) { return a.by_page.div(n + a.page_size - 1); };
  for (int r = tid; r < R; r += 256) {
    const int h = min(max(a.lengths[r], 0), most), w = min(max(a.wanted[r], 0), most), have = pages(h), need = pages(w);
    held[r] = h, want[r] = w;
    given[r] = max(have - need, 0), taken[r] = max(need - have, 0);
  }
  const int count = min(max(*a.count, 0), a.stack_size);
  __syncthreads();
  block_prefix(given, R);
  block_prefix(taken, R);
  // (a stack without room for what comes back, which its caller did not size for its pages, loses the last of it)
  const int freed = min(given[R], a.stack_size - count), top = count + freed, granted = min(taken[R], top);
  for (int r = tid; r < R; r += 256) {
    const int have = pages(held[r]), got = min(max(top - taken[r], 0), taken[r + 1] - taken[r]);
    const int n = taken[r + 1] - taken[r] > got ? min(want[r], (have + got) * a.page_size) : want[r];
    want[r] = n;
    tokens[r] = max(n - held[r], 0);
  }
  __syncthreads();
  block_prefix(tokens, R);
  const int id = blockIdx.x * 256 + tid, all = gridDim.x * 256;
  // the page of grant j: a freed one, or the stack's
  auto granted_page = [&](int j) {
    if (j >= freed) return a.stack[top - 1 - j];
    const int r = owner(given, R, j);
    return a.table[static_cast<int64_t>(r) * a.width + pages(want[r]) + j - given[r]];
  };
  for (int j = id; j < granted; j += all) {
    const int r = owner(taken, R, j);
    a.table[static_cast<int64_t>(r) * a.width + pages(held[r]) + j - taken[r]] = granted_page(j);
  }
  for (int i = granted + id; i < freed; i += all) a.stack[top - 1 - i] = granted_page(i);
  for (int r = id; r <= R; r += all) {
    a.starts[r] = min(tokens[r], a.max_tokens);
    if (r < R) a.new_lengths[r] = want[r];
  }
  if (id == 0) *a.new_count = top - granted;
  for (int t = id; t < a.max_tokens; t += all) {
    int slot = -1, position = 0;
    if (t < tokens[R]) {
      const int r = owner(tokens, R, t);
      position = held[r] + t - tokens[r];
      const int place = a.by_page.div(position), have = pages(held[r]);
      const int page = place < have ? a.table[static_cast<int64_t>(r) * a.width + place] : granted_page(taken[r] + place - have);
      const int64_t to = static_cast<int64_t>(page) * a.page_size + position - place * a.page_size;
      slot = page < 0 || to > 0x7fffffff ? -1 : static_cast<int>(to);
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
}

struct WriteArgs {
  const uint16_t *k, *v;      // [batch, n_kv, seq, D] through strides
  int64_t ks[3], vs[3];
  void *k_pages, *v_pages;    // [pages, n_kv, page_size, D]
  float *k_scale, *v_scale;   // [pages, n_kv, page_size]
  const int32_t* slots;       // [batch, seq]
  int rows, n_kv, seq, page_size;
  int n_slots;                // pages * page_size
  Divider by_kv, by_seq, by_page;
};

// A group of 8 or 16 lanes owns a token's row of a head, of keys and values both.
template <int DT, int D, bool F8>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
  constexpr int L = D == 64 ? 8 : 16;
  const int at = static_cast<int>(blockIdx.x) * (256 / L) + static_cast<int>(threadIdx.x) / L, c = threadIdx.x % L;
  if (at >= a.rows) return;
  const int t = a.by_kv.div(at), hk = at - t * a.n_kv, slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;  // (a whole group of lanes)
  const int b = a.by_seq.div(t), s = t - b * a.seq, page = a.by_page.div(slot);
  const int64_t row = (static_cast<int64_t>(page) * a.n_kv + hk) * a.page_size + slot - page * a.page_size;
  const bool mine = c * 8 < D;
  u32x4 k = {}, v = {};
  if (mine) {
    k = *reinterpret_cast<const u32x4*>(a.k + b * a.ks[0] + hk * a.ks[1] + s * a.ks[2] + 8 * c);
    v = *reinterpret_cast<const u32x4*>(a.v + b * a.vs[0] + hk * a.vs[1] + s * a.vs[2] + 8 * c);
  }
  if constexpr (F8) {
    float xk[8] = {}, xv[8] = {}, k_scale, v_scale;
    uint32_t kc[2], vc[2];
    unpack16<DT>(k, xk);
    unpack16<DT>(v, xv);
    quantise<DT, L>(xk, k_scale, kc);
    quantise<DT, L>(xv, v_scale, vc);
    if (mine) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.k_pages) + row * D + 8 * c) = uint2{kc[0], kc[1]};
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v_pages) + row * D + 8 * c) = uint2{vc[0], vc[1]};
    }
    if (c == 0) {
      a.k_scale[row] = k_scale;
      a.v_scale[row] = v_scale;
    }
  } else if (mine) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.k_pages) + row * D + 8 * c) = k;
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.v_pages) + row * D + 8 * c) = v;
  }
}

template <int DT, bool F8>
void launch_write(const WriteArgs& a, int head_dim, dim3 grid, hipStream_t s) {
  if (head_dim == 64) hipLaunchKernelGGL((paged_write_kernel<DT, 64, F8>), grid, dim3(256), 0, s, a);
  else if (head_dim == 80) hipLaunchKernelGGL((paged_write_kernel<DT, 80, F8>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((paged_write_kernel<DT, 128, F8>), grid, dim3(256), 0, s, a);
}

}  // namespace
}  // namespace wx

using namespace wx;

extern "C" int wx_paged_kv_resize(const int32_t* lengths, const int32_t* wanted, int32_t* page_table, int32_t* free_pages, const int32_t* free_count,
                                  int32_t* new_lengths, int32_t* new_free_count, int32_t* starts, int32_t* slots, int64_t* positions,
                                  int64_t requests, int64_t pages_per_request, int64_t free_capacity, int page_size, int64_t max_tokens,
                                  wx_stream_t stream) {
  const char* who = "wx_paged_kv_resize";
  if (requests < 0 || pages_per_request < 0 || free_capacity < 0 || max_tokens < 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (page_size <= 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: page_size must be positive", who);
  if (requests > kMaxRequests) return fail(WX_ERR_UNSUPPORTED, "%s: more than %d requests", who, kMaxRequests);
  if (page_size > (1 << 20) || pages_per_request > 0x3fffffffll / page_size) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 tokens to a request", who);
  if (free_capacity > 0x7fffffffll / page_size) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", who);
  if (max_tokens > 0x3fffffffll || requests * pages_per_request > 0x7fffffffll / page_size)
    return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", who);
  if (!new_free_count || !free_count || !starts) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if ((requests > 0 && (!lengths || !wanted || !new_lengths || (pages_per_request > 0 && !page_table))) || (free_capacity > 0 && !free_pages) ||
      (max_tokens > 0 && (!slots || !positions)))
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  ResizeArgs a{};
  a.lengths = lengths, a.wanted = wanted, a.table = page_table, a.stack = free_pages, a.count = free_count;
  a.new_lengths = new_lengths, a.new_count = new_free_count, a.starts = starts, a.slots = slots, a.positions = positions;
  a.requests = static_cast<int>(requests), a.width = static_cast<int>(pages_per_request), a.stack_size = static_cast<int>(free_capacity);
  a.page_size = page_size, a.max_tokens = static_cast<int>(max_tokens), a.by_page = Divider(page_size);
  // a workgroup for every 1024 tokens: each finds the prefix sums for itself
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((max_tokens + 1023) / 1024, 4 * device_cu_count()));
  hipLaunchKernelGGL(paged_resize_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream), a);
  return check_launch(who);
}

extern "C" int wx_paged_kv_write(const void* k, const void* v, void* k_pages, void* v_pages, float* k_scale, float* v_scale, const int32_t* slots,
                                 int64_t batch, int n_kv_heads, int64_t seq, int64_t num_pages, int page_size, int head_dim,
                                 const int64_t k_strides[3], const int64_t v_strides[3], int dtype, wx_stream_t stream) {
  const char* who = "wx_paged_kv_write";
  if (batch < 0 || n_kv_heads < 0 || seq < 0 || num_pages < 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (page_size <= 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: page_size must be positive", who);
  if (head_dim != 64 && head_dim != 80 && head_dim != 128) return fail(WX_ERR_UNSUPPORTED, "%s: head_dim %d must be 64, 80 or 128", who, head_dim);
  if (dtype != WX_BF16 && dtype != WX_F16) return fail(WX_ERR_UNSUPPORTED, "%s: dtype %d must be bf16 or fp16", who, dtype);
  if (!k_strides || !v_strides) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null strides", who);
  if ((k_scale == nullptr) != (v_scale == nullptr)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: scales of keys and values, or neither", who);
  if (num_pages > 0x7fffffffll / page_size) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", who);
  if (batch == 0 || n_kv_heads == 0 || seq == 0 || num_pages == 0) return WX_OK;
  if (!k || !v || !k_pages || !v_pages || !slots) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  for (const void* p : {k, v, static_cast<const void*>(k_pages), static_cast<const void*>(v_pages)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return fail(WX_ERR_UNSUPPORTED, "%s: strides must keep rows 16-byte aligned", who);
  if (seq > 0x7fffffffll / n_kv_heads || batch > 0x7fffffffll / (seq * n_kv_heads)) return fail(WX_ERR_UNSUPPORTED, "%s: too many tokens", who);
  WriteArgs a{};
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  for (int i = 0; i < 3; ++i) a.ks[i] = k_strides[i], a.vs[i] = v_strides[i];
  a.k_pages = k_pages, a.v_pages = v_pages, a.k_scale = k_scale, a.v_scale = v_scale, a.slots = slots;
  a.rows = static_cast<int>(batch * seq * n_kv_heads), a.n_kv = n_kv_heads, a.seq = static_cast<int>(seq), a.page_size = page_size;
  a.n_slots = static_cast<int>(num_pages * page_size);
  a.by_kv = Divider(n_kv_heads), a.by_seq = Divider(static_cast<uint32_t>(seq)), a.by_page = Divider(page_size);
  const int64_t each = 256 / (head_dim == 64 ? 8 : 16), blocks = (static_cast<int64_t>(a.rows) + each - 1) / each;
  if (too_many_blocks(blocks, 256)) return fail(WX_ERR_UNSUPPORTED, "%s: too many tokens", who);
  const dim3 grid(static_cast<unsigned>(blocks));
  hipStream_t s = as_stream(stream);
  if (dtype == WX_BF16) k_scale ? launch_write<WX_BF16, true>(a, head_dim, grid, s) : launch_write<WX_BF16, false>(a, head_dim, grid, s);
  else k_scale ? launch_write<WX_F16, true>(a, head_dim, grid, s) : launch_write<WX_F16, false>(a, head_dim, grid, s);
  return check_launch(who);
}
