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

constexpr int kMaxRequests = 4096;  // of one call: five numbers of each in LDS

struct ResizeArgs {
  const int32_t *lengths, *wanted;  // [requests]
  int32_t *table;                   // [requests, width]
  int32_t *stack;                   // [stack_size]
  const int32_t *count;
  int32_t *new_lengths, *new_count, *starts, *slots;
  int64_t* positions;
  int requests, width, stack_size, page_size, max_tokens;
  int book_blocks;                  // workgroups that keep the tables and the stack; the others write the slot map
  Divider by_page;
};

// In-place exclusive prefix sums of N arrays of n numbers, totals behind them, by 256 threads.
template <int N>
__device__ __forceinline__ void block_prefix(int* const (&s)[N], int n) {
  __shared__ int wave_sums[4][N];
  const int tid = threadIdx.x, wave = tid >> 6, each = (n + 255) / 256, first = min(tid * each, n), last = min(first + each, n);
  int mine[N] = {}, at[N];
  for (int i = first; i < last; ++i)
#pragma unroll
    for (int u = 0; u < N; ++u) mine[u] += s[u][i];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int sum = wave_prefix(mine[u]);
    if ((tid & 63) == 63) wave_sums[wave][u] = sum;
    at[u] = sum - mine[u];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < N; ++u) {
    at[u] += (wave > 0 ? wave_sums[0][u] : 0) + (wave > 1 ? wave_sums[1][u] : 0) + (wave > 2 ? wave_sums[2][u] : 0);
    for (int i = first; i < last; ++i) {
      const int x = s[u][i];
      s[u][i] = at[u];
      at[u] += x;
    }
    if (tid == 255) s[u][n] = at[u];
  }
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

// Every workgroup finds the prefix sums for itself (2 numbers a request from memory); some then keep the tables, the others write the slot map, four
// tokens to a thread: of neighbouring tokens the request, and mostly the page, is one.  What takes the time is the chain of loads, scans and searches:
// 64 requests of a token each 4.5 us a launch; 1000 requests that take 206 thousand tokens 9.9 (13.2 with a token to a thread and all of it one
// after the other in every workgroup).
template <int MAX>
__global__ __launch_bounds__(256) void paged_resize_kernel(ResizeArgs a) {
  __shared__ int held[MAX], want[MAX], given[MAX + 1], taken[MAX + 1], tokens[MAX + 1];
  const int R = a.requests, tid = threadIdx.x;
  const int most = a.width * a.page_size;
  auto pages = [&](int n) { return a.by_page.div(n + a.page_size - 1); };
  const int count = min(max(*a.count, 0), a.stack_size);
  for (int r = tid; r < R; r += 256) {
    const int h = min(max(a.lengths[r], 0), most), w = min(max(a.wanted[r], 0), most), have = pages(h), need = pages(w);
    held[r] = h, want[r] = w;
    given[r] = max(have - need, 0), taken[r] = max(need - have, 0);
  }
  __syncthreads();
  block_prefix<2>({given, taken}, R);
  // (a stack without room for what comes back, which its caller did not size for its pages, loses the last of it)
  const int freed = min(given[R], a.stack_size - count), top = count + freed, granted = min(taken[R], top);
  for (int r = tid; r < R; r += 256) {
    const int n = taken[r + 1] - taken[r], got = min(max(top - taken[r], 0), n);
    const int w = n > got ? min(want[r], (pages(held[r]) + got) * a.page_size) : want[r];
    want[r] = w;
    tokens[r] = max(w - held[r], 0);
  }
  __syncthreads();
  block_prefix<1>({tokens}, R);
  const bool books = static_cast<int>(blockIdx.x) < a.book_blocks;
  const int id = (static_cast<int>(blockIdx.x) - (books ? 0 : a.book_blocks)) * 256 + tid, all = (books ? a.book_blocks : static_cast<int>(gridDim.x) - a.book_blocks) * 256;
  // the page of grant j: a freed one, or the stack's
  auto granted_page = [&](int j) {
    if (j >= freed) return a.stack[top - 1 - j];
    const int r = owner(given, R, j);
    return a.table[static_cast<int64_t>(r) * a.width + pages(want[r]) + j - given[r]];
  };
  for (int r = id; books && r <= R; r += all) {
    a.starts[r] = min(tokens[r], a.max_tokens);
    if (r < R) a.new_lengths[r] = want[r];
  }
  if (books && id == 0) *a.new_count = top - granted;
  for (int j = id; books && j < granted; j += all) {
    const int r = owner(taken, R, j);
    a.table[static_cast<int64_t>(r) * a.width + pages(held[r]) + j - taken[r]] = granted_page(j);
  }
  for (int i = granted + id; books && i < freed; i += all) a.stack[top - 1 - i] = granted_page(i);
  for (int t0 = 4 * id; !books && t0 < a.max_tokens; t0 += 4 * all) {
    int r = t0 < tokens[R] ? owner(tokens, R, t0) : R, known = -1, page = -1;  // `page` is place `known` of request r
    int slots[4];
    int64_t positions[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + u;
      slots[u] = -1, positions[u] = 0;
      if (t >= tokens[R]) continue;
      while (t >= tokens[r + 1]) ++r, known = -1;  // (some later request has t: the last prefix sum is beyond it)
      const int position = held[r] + t - tokens[r], place = a.by_page.div(position);
      if (place != known) {
        const int have = pages(held[r]);
        page = place < have ? a.table[static_cast<int64_t>(r) * a.width + place] : granted_page(taken[r] + place - have);
        known = place;
      }
      const int64_t slot = static_cast<int64_t>(page) * a.page_size + position - place * a.page_size;
      slots[u] = page < 0 || slot > 0x7fffffff ? -1 : static_cast<int>(slot);
      positions[u] = position;
    }
    if (t0 + 4 <= a.max_tokens) {
      *reinterpret_cast<int4*>(a.slots + t0) = int4{slots[0], slots[1], slots[2], slots[3]};
      *reinterpret_cast<longlong2*>(a.positions + t0) = longlong2{positions[0], positions[1]};
      *reinterpret_cast<longlong2*>(a.positions + t0 + 2) = longlong2{positions[2], positions[3]};
    } else {
      for (int u = 0; t0 + u < a.max_tokens; ++u) {
        a.slots[t0 + u] = u == 0 ? slots[0] : (u == 1 ? slots[1] : slots[2]);
        a.positions[t0 + u] = u == 0 ? positions[0] : (u == 1 ? positions[1] : positions[2]);
      }
    }
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
  if ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: slots and positions must be 16-byte aligned", who);
  ResizeArgs a{};
  a.lengths = lengths, a.wanted = wanted, a.table = page_table, a.stack = free_pages, a.count = free_count;
  a.new_lengths = new_lengths, a.new_count = new_free_count, a.starts = starts, a.slots = slots, a.positions = positions;
  a.requests = static_cast<int>(requests), a.width = static_cast<int>(pages_per_request), a.stack_size = static_cast<int>(free_capacity);
  a.page_size = page_size, a.max_tokens = static_cast<int>(max_tokens), a.by_page = Divider(page_size);
  a.book_blocks = static_cast<int>(std::min<int64_t>(max_tokens / page_size / 256 + (requests + 255) / 256 + 1, 64));
  const dim3 grid(static_cast<unsigned>(a.book_blocks + std::min<int64_t>((max_tokens + 1023) / 1024, 4 * device_cu_count())));
  if (requests <= 1024) hipLaunchKernelGGL(paged_resize_kernel<1024>, grid, dim3(256), 0, as_stream(stream), a);  // (20 KB of LDS, not 80)
  else hipLaunchKernelGGL(paged_resize_kernel<kMaxRequests>, grid, dim3(256), 0, as_stream(stream), a);
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
