// Attention of requests' newest tokens over a paged key / value cache: each request has its own number of queries and keys, none of which the
// host knows (gfx950).
//
// The host knows neither number, so the launch is of a fixed number of workgroups, each of which finds its share of all the work by itself, from
// the lengths (paged_plan.h): one request over 32768 keys and 64 over 900 fill the chip alike, without the host and without a plan in memory.  What
// shares leave of items that they cut is joined by a second launch, in order.  (Joined by the workgroup whose part is the last to arrive, with stores and
// loads past the XCDs' L2: 64 x 32 queries 81 us for 52, 8 long requests 42 for 37.)
//
// What bounds it.  Single tokens over long caches: memory; 112 MB of 8 requests over 20 to 32 thousand keys stream in some 24 us, 4.7 TB/s, and
// 6 before and 7 behind that go into the plan, the first pages and keys, and the join: 35 to 40 us in all.  32 requests of up to 5 tokens over up to 16000
// bf16 keys: 262 MB in 67 us.  Short caches: the chain of loads alone; of 20.5 us for 64 single tokens over 900 keys 2.6 go into the plan,
// 1.8 to the first keys' request, 2.8 into the one tile a wavefront has, 2.1 into the wavefronts' join, 4 into the parts'.  Chunks: 2048 queries over 16384
// e4m3 keys 303 us, 0.85 PFLOP/s (the contiguous cache's kernel: 392), bf16 keys 290 (contiguous 313); a tile of 64 keys takes a SIMD's two wavefronts 4800
// cycles, in which their products need 2048 and their other instructions 3300.  16 prompts of 912 bf16 tokens: 88 to 97 us, a workgroup to an item; 8 of them 48.
#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "common.h"
#include "paged_plan.h"

namespace wx {
namespace {

using namespace paged;

#define WX_GLOBAL(p) ((const __attribute__((address_space(1))) void*)(p))

struct PagedArgs {
  const uint16_t* q;               // [batch, n_q, seq, D] through strides; token t is position t % seq of row t / seq
  int64_t qs[3];
  const void *k, *v;               // [pages, n_kv, page_size, D]
  const float *k_scale, *v_scale;  // e4m3: [pages, n_kv, page_size]
  uint16_t* out;                   // [tokens, n_q, D]
  const int32_t *table, *lengths, *starts;  // [requests, width], [requests], [requests + 1] or null: seq tokens each
  int causal, tokens, requests, n_q, n_kv, group, seq, width, page_size, n_pages;
  int most_keys;                   // width * page_size
  Divider by_seq, by_page, by_group;
  float c;                         // scale * log2(e)
  int shares, blocks, shift;       // see paged_plan.h
  int part_rows;                   // most rows of an item
  float* sums;                     // parts: [2 shares, part_rows, D]
  float2* stats;                   // [2 shares, part_rows] (maximum, sum of powers)
  Part* part;                      // [shares]
  __device__ __forceinline__ float reciprocal(float x) const { return __builtin_amdgcn_rcpf(x); }
  __device__ __forceinline__ int uniform(int x) const { return __builtin_amdgcn_readfirstlane(x); }
};

template <class T>
__device__ __forceinline__ T uniform(T x) {
  static_assert(sizeof(T) % 4 == 0, "");
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
}

template <class T>
__device__ __forceinline__ T of_lane(T x, int lane) {
  static_assert(sizeof(T) % 4 == 0, "");
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) w[i] = __builtin_amdgcn_readlane(w[i], lane);
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
}
// Up to 64 requests are a wavefront's, and every wavefront finds the share for itself, without a barrier (32 requests of drafts 69 -> 67 us, 16 prompts
// 104 -> 102); more are spread over the workgroup's threads.  Tokens [0, none_from) and [none_to, all) are no request's.
template <bool F8>
__device__ __forceinline__ Share share(const PagedArgs& a, int& none_from, int& none_to) {
  __shared__ int s_sums[4][kSums], s_longest[4], s_moved[2];
  __shared__ Place s_place;
  __shared__ Request s_q;
  __shared__ int s_r, s_none[2];
  const bool alone = a.requests <= 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, each = alone ? 1 : (a.requests + 255) / 256;
  const int first = min((alone ? lane : tid) * each, a.requests), last = min(first + each, a.requests);
  int mine[kSums] = {}, sum[kSums], longest = 0;
  if (tid == 0) s_moved[0] = 0, s_moved[1] = 0;
  Request q = {};
  for (int r = first; r < last; ++r) {
    q = request(a, r);
    add_request(a, q, mine, longest);
    if (!alone && r == 0) s_none[0] = q.first;
    if (!alone && r == a.requests - 1) s_none[1] = q.first + q.n;
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i) sum[i] = wave_prefix(mine[i]);
  longest = max(wave_extreme<true>(longest), __builtin_amdgcn_readlane(wave_extreme<true>(__shfl_xor(longest, 32)), 0));
  int all[kSums], before[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) all[i] = __builtin_amdgcn_readlane(sum[i], 63), before[i] = sum[i] - mine[i];
  if (!alone) {
    if (lane == 0) s_longest[wave] = longest;
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < kSums; ++i) s_sums[wave][i] = sum[i];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    if (alone) continue;
    const int w0 = s_sums[0][i], w1 = s_sums[1][i], w2 = s_sums[2][i];
    before[i] += (wave > 0 ? w0 : 0) + (wave > 1 ? w1 : 0) + (wave > 2 ? w2 : 0);
    all[i] = uniform(w0 + w1 + w2 + s_sums[3][i]);
  }
  longest = alone ? uniform(longest) : uniform(max(max(s_longest[0], s_longest[1]), max(s_longest[2], s_longest[3])));
  if (all[kHigh] > kMostHigh) none_from = a.tokens, none_to = a.tokens;
  Share s = share_of<F8>(a, blockIdx.x, gridDim.x, all, longest);
  if (all[kHigh] > kMostHigh) return s;
  const int from = of_share(s, before), to = from + of_share(s, mine);
  Place place = {};
  int moved[2] = {0, 0};
  if (s.size > 0 && ((from <= s.at && s.at < to) || (from <= s.end && s.end < to))) {
    int r_from = from;
    for (int r = first; r < last; ++r) {
      if (each > 1) q = request(a, r);
      const int m = extent(a, s, q);
      if (r_from <= s.at && s.at < r_from + m) {
        moved[0] = begin_of(a, s, q, s.at - r_from, place);
        if (!alone) s_moved[0] = moved[0], s_place = place, s_q = q, s_r = r;
      }
      Place end_place;
      if (r_from <= s.end && s.end < r_from + m) {
        moved[1] = locate(a, q, s.kind, s.end - r_from, s.each, end_place);
        if (!alone) s_moved[1] = moved[1];
      }
      r_from += m;
    }
  }
  if (alone) {  // (the lane that has the request, for the share's begin and for its end; lane 63 has none, or nothing to move)
    const uint64_t begins = __ballot(from <= s.at && s.at < to), ends = __ballot(from <= s.end && s.end < to);
    const int l = begins ? __builtin_ctzll(begins) : 0;
    place = of_lane(place, l), s.q = of_lane(q, l), s.r = l;
    moved[0] = __builtin_amdgcn_readlane(moved[0], l), moved[1] = ends ? __builtin_amdgcn_readlane(moved[1], __builtin_ctzll(ends)) : 0;
    none_from = a.requests ? __builtin_amdgcn_readlane(q.first, 0) : a.tokens;
    none_to = a.requests ? __builtin_amdgcn_readlane(q.first + q.n, a.requests - 1) : a.tokens;
  } else {
    __syncthreads();
    none_from = uniform(s_none[0]), none_to = uniform(s_none[1]);
    place = uniform(s_place), s.q = uniform(s_q), s.r = uniform(s_r);
    moved[0] = uniform(s_moved[0]), moved[1] = uniform(s_moved[1]);
  }
  s.head = place.head, s.tile = place.tile;
  if (!s.parts) s.size = uniform(s.size + (s.size > 0 ? moved[1] - moved[0] : 0)), s.x = place.x;
  return s;
}

// The next request of a kind, 64 looked at at a time; -1 if there is none.
__device__ __forceinline__ int next_request(const PagedArgs& a, int r, int kind) {
  for (; r < a.requests; r += 64) {
    const int i = r + static_cast<int>(threadIdx.x & 63);
    const uint64_t is = __ballot(i < a.requests && measure(a, request(a, min(i, a.requests - 1)), kind) != 0);
    if (is != 0) return r + __builtin_ctzll(is);
  }
  return -1;
}

// The type of the second product.  e4m3 codes are exact in both types, but fp16's range is too short for a probability times its key's
// scale: there the codes are widened to bf16 and the probabilities enter as the sum of two bf16 numbers, which is more of them than fp16 keeps.
template <int DT, bool F8>
constexpr int kValues = F8 ? WX_BF16 : DT;
template <int DT, bool F8>
constexpr bool kTwice = F8 && DT == WX_F16;

template <int DT, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t x) {
  if constexpr (DT == WX_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, HI));
}
template <int DT>
__device__ __forceinline__ u32x4 widen8(uint32_t x, uint32_t y) {
  return u32x4{widen2<DT, false>(x), widen2<DT, true>(x), widen2<DT, false>(y), widen2<DT, true>(y)};
}
// pack_step's operand in bf16, and what that rounding leaves as another (of what is not finite NaN: such rows are made again).
__device__ __forceinline__ void pack_twice(const f32x16& p, int t, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float x = p[8 * t + 2 * u], y = p[8 * t + 2 * u + 1];
    hi[u] = pack2<WX_BF16>(x, y);
    lo[u] = pack2<WX_BF16>(x - __uint_as_float(hi[u] << 16), y - __uint_as_float(hi[u] & 0xffff0000u));
  }
}
// what rounding x to bf16 leaves (nothing of what is not finite)
__device__ __forceinline__ float left_of(float x) {
  const float r = x - round_bf16(x);
  return r - r == 0.f ? r : 0.f;
}
__device__ __forceinline__ f32x16 left_of(const f32x16& x) {
  f32x16 y;
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = left_of(x[r]);
  return y;
}

// This lane's key of a tile: its row in the pages, or that it has none.
struct KeyRow {
  uint32_t row;
  bool ok;
};
__device__ __forceinline__ int page_of(const PagedArgs& a, const Segment& g, int key) {  // (key: below g.hi)
  return a.table[static_cast<int64_t>(g.r) * a.width + a.by_page.div(key)];
}
__device__ __forceinline__ KeyRow row_of(const PagedArgs& a, const Segment& g, int key, int page) {
  const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages);
  const uint32_t in = static_cast<uint32_t>(key - a.by_page.div(key) * a.page_size);
  return {ok ? (static_cast<uint32_t>(page) * a.n_kv + g.head) * a.page_size + in : 0u, ok};
}

// A lane's row: its query, where that lies, and the keys that it sees of the segment's.
struct Row {
  int at, hq, seen;
  int token;
  bool live;
};
__device__ __forceinline__ Row row_at(const PagedArgs& a, const Segment& g, int i) {
  Row w;
  w.live = i < g.rows;
  w.at = w.live ? i : 0;
  const int row = g.row0 + w.at, qi = a.by_group.div(row);
  w.hq = g.head * a.group + row - qi * a.group;
  w.token = g.q.first + qi;
  w.seen = w.live ? min(keys_seen(a, g.q, row), g.hi) : g.hi;  // (rows that there are not see everything: they take no mask)
  return w;
}
__device__ __forceinline__ const uint16_t* query(const PagedArgs& a, const Row& w) {
  const int b = a.by_seq.div(w.token);
  return a.q + b * a.qs[0] + w.hq * a.qs[1] + static_cast<int64_t>(w.token - b * a.seq) * a.qs[2];
}
__device__ __forceinline__ int64_t result(const PagedArgs& a, const Row& w, int d) { return (static_cast<int64_t>(w.token) * a.n_q + w.hq) * d; }

// Rows whose sums are not numbers (see Odd, attention.h) again, of 32 of the segment's rows from `first` on those that `again` has a bit for,
// from memory, with the maximum and the sum that they ended with.  A row that sees nothing is among them where a tile of its keys, which others see or
// which are the pool's first in the place of pages that there are none of, holds such values: its sums are zeros here, as its sum of powers is.
template <int DT, int D, bool F8>
__device__ __forceinline__ void rows_again(const PagedArgs& a, const Segment& g, int first, uint32_t again, float m, float l) {
  using T = AttnTile<D>;
  constexpr int PT = kValues<DT, F8>;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (see few_rows)
  const int h = lane >> 5;
  const Row w = row_at(a, g, first + (lane & 31));
  const bool redo = again >> (lane & 31) & 1;
  const float mc = m == -kInf ? 0.f : m * a.c;
  const uint16_t* q = query(a, w);
  auto where = [&](int key) {
    key = min(key, g.hi - 1);
    return row_of(a, g, key, page_of(a, g, key));
  };
  for (int o = 0; o < T::kOut; ++o) {
    f32x16 sum = {};
    const int c = 32 * o + (lane & 31);
    for (int k0 = g.lo; k0 < g.hi; k0 += 32) {
      f32x16 s = {};
      const KeyRow mine = where(k0 + (lane & 31));
      for (int t = 0; t < T::kSteps; ++t) {
        u32x4 x;
        if constexpr (F8) {
          const u32x2 y = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(a.k) + static_cast<uint64_t>(mine.row) * D + 16 * t + 8 * h);
          x = widen8<DT>(y[0], y[1]);
        } else {
          x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.k) + static_cast<uint64_t>(mine.row) * D + 16 * t + 8 * h);
        }
        s = mfma<DT>(x, *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h), s);
      }
      uint32_t seen = 0, zero = 0, at[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 8 * (r / 4) + 4 * h + r % 4;
        const KeyRow key = where(k0 + i);
        const bool sees = redo && k0 + i < w.seen && key.ok;
        at[r] = key.row;
        if constexpr (F8) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r] * a.k_scale[key.row], a.c, -mc)) * a.v_scale[key.row];
        else s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -mc));
        s[r] = sees ? s[r] : 0.f;
        seen |= sees ? 1u << r : 0u;
        zero |= sees && s[r] == 0.f ? 1u << r : 0u;
      }
      f32x16 rest;
      if constexpr (kTwice<DT, F8>) rest = left_of(s);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Odd odd;
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // (rows of the step's keys: register 8 t + j of this half)
          const uint64_t e = static_cast<uint64_t>(at[8 * t + j]) * D + c;
          y[j] = 0;
          if (D % 32 == 0 || c < D) {
            if constexpr (F8) y[j] = widen2<PT, false>(static_cast<const uint8_t*>(a.v)[e]) & 0xffffu;
            else y[j] = static_cast<const uint16_t*>(a.v)[e];
          }
        }
        const u32x4 x = finite8<PT>(y, odd);
        sum = mfma<PT>(x, pack_step<PT>(s, t), sum);
        if constexpr (kTwice<DT, F8>) sum = mfma<PT>(x, pack_step<PT>(rest, t), sum);
        add_odd<PT>(sum, odd, seen, zero, t);
      }
    }
    if (g.whole) store_cols<DT, D>(sum, o, l == 0.f ? 0.f : 1.f / l, redo ? a.out + result(a, w, D) : nullptr, lane);
    else if (redo) store_sums<D>(sum, o, a.sums + (static_cast<int64_t>(g.slot) * a.part_rows + w.at) * D, lane);
  }
}

// ---- the mask on 32 keys' scores: bit i of `seen` tells of key i
__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ void hide(f32x16& s, uint32_t seen, int h) {
  const uint32_t mine = seen >> (4 * h);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(mine), 8 * (r / 4) + r % 4, 1));
    s[r] = __uint_as_float((__float_as_uint(s[r]) & keep) | (0xff800000u & ~keep));
  }
}

// Running maximum, sum of powers and sums of 32 rows.
template <int D>
struct Sums {
  f32x16 acc[AttnTile<D>::kOut];
  float m, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int o = 0; o < AttnTile<D>::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[o][r] = 0.f;
    m = -kInf, l = 0.f;
  }
  // The maximum is only there to keep the powers in range: it moves when a score exceeds it by more than 2^8.
  template <int NT>
  __device__ __forceinline__ void raise(const f32x16 (&s)[NT], float c) {
    float tops[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 2) tops[r / 2 % 4] = fmaxf(fmaxf(tops[r / 2 % 4], s[n][r]), s[n][r + 1]);
    const float top = both_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    if (__any((top - m) * c > 8.f)) {
      const float mn = fmaxf(m, top), alpha = mn == -kInf ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int o = 0; o < AttnTile<D>::kOut; ++o)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[o][r] *= alpha;
    }
  }
};

// Two arrays of LDS: of few rows the wavefronts' slots for keys and for values, of many tiles in turn.
constexpr int kFewSlot = 8192 + 512;
template <int D>
constexpr int kPagedLds = 2 * 64 * AttnTile<D>::kPitch + 2 * 64 * 4 > 4 * kFewSlot ? 2 * 64 * AttnTile<D>::kPitch + 2 * 64 * 4 : 4 * kFewSlot;

// ---- few rows.  Every wavefront walks tiles of its own, of 64 (e4m3) or 32 keys, for 32 rows: up to 32 rows the four of a workgroup share the
// keys, up to 64 two and two.  K and V of a tile go straight to LDS as they are in memory, each into one slot of the wavefront's own that is
// filled again as soon as it is read: no barrier, 16 KB on their way per wavefront, eight wavefronts a CU.  e4m3 is widened behind LDS,
// which transposes bytes as well.
template <int D>
struct RawTile {  // rows of D bytes
  static constexpr int kChunks = D / 16;
  __device__ static __forceinline__ int swizzle(int row) {
    if constexpr (D == 128) return (row & 3) | (((row >> 3) ^ (row >> 2)) & 1) << 2;
    else if constexpr (D == 64) return (row >> 2) & 3;
    else return 0;
  }
  __device__ static __forceinline__ int at(int row, int chunk) { return (row * kChunks + (chunk ^ swizzle(row))) * 16; }
};

template <int DT, int D, bool F8>
__device__ __forceinline__ void few_rows(const PagedArgs& a, const Segment& g) {
  using T = AttnTile<D>;
  using R = RawTile<D>;
  constexpr int PT = kValues<DT, F8>, KB = F8 ? 64 : 32, NT = KB / 32;
  constexpr int kChunks = F8 ? R::kChunks : T::kChunks, kLoads = KB * kChunks / 64, kElem = F8 ? 1 : 2, kSlot = KB * kChunks * 16;
  unsigned char *const lds_k = lds_slot<kPagedLds<D>, 0>(), *const lds_v = lds_slot<kPagedLds<D>, 1>();
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (what is made from it is made here: kept over the segments it would be spilled)
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int blocks = g.rows <= 32 ? 1 : 2, kws = 4 / blocks, rb = wave & (blocks - 1), kw = wave / blocks;
  unsigned char *const my_k = lds_k + wave * kFewSlot, *const my_v = lds_v + wave * kFewSlot, *const my_scales = my_k + kSlot;
  static_assert(kLoads * 64 == KB * kChunks && kSlot + (F8 ? 512 : 0) <= kFewSlot && 32 * 64 * 4 <= kFewSlot, "");
  const int tiles = (g.hi - g.lo + KB - 1) / KB, mine = tiles > kw ? (tiles - kw + kws - 1) / kws : 0;
  auto key0 = [&](int i) { return g.lo + (i * kws + kw) * KB; };
  const int in_tile = lane & (KB - 1);  // a lane finds the row of one of a tile's keys
  auto ask = [&](int i) { return page_of(a, g, min(key0(i) + in_tile, g.hi - 1)); };
  int p0 = 0, p1 = 0;
  if (mine > 0) p0 = ask(0), p1 = ask(1);
  in_order();
  const Row row = row_at(a, g, rb * 32 + (lane & 31));
  u32x4 qf[T::kSteps];
  {
    const uint16_t* q = query(a, row);
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      // e4m3: two steps take 16 channels of a lane in a row
      const int c = F8 && t / 2 * 2 + 1 < T::kSteps ? 32 * (t / 2) + 16 * h + 8 * (t % 2) : 16 * t + 8 * h;
      qf[t] = *reinterpret_cast<const u32x4*>(q + c);
    }
  }
  const int all_see = wave_extreme<false>(row.seen);  // every row sees the keys before
  wait_loads();  // (queries and pages: what waits for them later would wait for the keys as well)
  uint32_t src[kLoads], scale_row = 0;
  uint64_t ok_next = 0;
  auto find = [&](int i, int page) {
    const int key = key0(i) + in_tile;
    KeyRow k = row_of(a, g, min(key, g.hi - 1), page);
    k.ok = k.ok && key < g.hi;
    return k;
  };
  auto take = [&](const KeyRow& k) {  // rows of a tile: of this lane's pieces, and of its scales
    ok_next = __ballot(k.ok);
    scale_row = k.row;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) src[u] = __shfl(k.row, (u * 64 + lane) / kChunks);
  };
  auto load_part = [&](int u, const void* from, unsigned char* slot) {
    const int n = u * 64 + lane, r = n / kChunks, c = (n % kChunks) ^ (F8 ? R::swizzle(r) : T::swizzle(r));
    const char* p = static_cast<const char*>(from) + static_cast<uint64_t>(src[u]) * (D * kElem) + c * 16;
    if (F8 || T::kChunks * 8 == D || c < D / 8) __builtin_amdgcn_global_load_lds(WX_GLOBAL(p), WX_LDS(slot + u * 1024), 16, 0, 0);
  };
  auto load = [&](const void* from, unsigned char* slot) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) load_part(u, from, slot);
  };
  auto load_values = [&] {  // and the scales, in front of them: they are there when the next keys are
    if constexpr (F8) {
      __builtin_amdgcn_global_load_lds(WX_GLOBAL(a.k_scale + scale_row), WX_LDS(my_scales), 4, 0, 0);
      __builtin_amdgcn_global_load_lds(WX_GLOBAL(a.v_scale + scale_row), WX_LDS(my_scales + 256), 4, 0, 0);
    }
    load(a.v, my_v);
  };
  auto wait = [&](bool younger) {  // the loads of one slot that are younger than what is waited for may stay in flight
    asm volatile("" ::: "memory");
    if (younger) __builtin_amdgcn_s_waitcnt(attn_wait(kLoads, 15));
    else __builtin_amdgcn_s_waitcnt(attn_wait(0, 15));
    asm volatile("" ::: "memory");
  };
  Sums<D> sums;
  sums.clear();
  uint64_t ok = 0;
  int page = 0;
  if (mine > 0) {
    take(find(0, p0));
    const KeyRow next = find(1, p1);
    load(a.k, my_k);
    page = ask(2);
    load_values();
    ok = ok_next;
    take(next);
  }
  const int rows_at = rows_base<D>(lane), cols_at = cols_base<D>(lane);
  // e4m3: bytes 8 (lane & 1) of chunk 2 o + (lane / 16 & 1), of the row that the transposing read wants of this lane
  const int raw_row = 8 * ((lane >> 3) & 1) + 4 * h + ((lane >> 1) & 3);
  for (int i = 0; i < mine; ++i) {
    const int k0 = key0(i);
    const bool more = i + 1 < mine;
    wait(true);  // keys and scales are there, values may be on their way
    f32x16 s[NT] = {};
    if constexpr (F8) {  // operands are asked for a few products ahead
      constexpr int kReads = NT * (T::kSteps / 2), kAhead = 4;
      auto read = [&](int j) { return *reinterpret_cast<const u32x4*>(my_k + R::at(32 * (j % NT) + (lane & 31), 2 * (j / NT) + h)); };
      u32x4 f[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead && j < kReads; ++j) f[j] = read(j);
      u32x2 odd[NT];
      if constexpr (T::kSteps % 2 != 0)
#pragma unroll
        for (int n = 0; n < NT; ++n) odd[n] = *reinterpret_cast<const u32x2*>(my_k + R::at(32 * n + (lane & 31), T::kSteps - 1) + 8 * h);
      in_order();
#pragma unroll
      for (int j = 0; j < kReads; ++j) {
        const u32x4 x = f[j % kAhead];
        s[j % NT] = mfma<DT>(widen8<DT>(x[0], x[1]), qf[2 * (j / NT)], s[j % NT]);
        s[j % NT] = mfma<DT>(widen8<DT>(x[2], x[3]), qf[2 * (j / NT) + 1], s[j % NT]);
        if (j + kAhead < kReads) f[j % kAhead] = read(j + kAhead);
        in_order();
      }
      if constexpr (T::kSteps % 2 != 0)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = mfma<DT>(widen8<DT>(odd[n][0], odd[n][1]), qf[T::kSteps - 1], s[n]);
    } else {
      constexpr int kAhead = 4;
      u32x4 f[kAhead];
#pragma unroll
      for (int t = 0; t < kAhead; ++t) f[t] = read_rows<D>(my_k, 0, t, rows_at);
      in_order();
#pragma unroll
      for (int t = 0; t < T::kSteps; ++t) {
        s[0] = mfma<DT>(f[t % kAhead], qf[t], s[0]);
        if (t + kAhead < T::kSteps) f[t % kAhead] = read_rows<D>(my_k, 0, t + kAhead, rows_at);
        in_order();
      }
    }
    wait_lds();  // (the slot is read before it is filled again)
    in_order();
    if (!F8 && more) load(a.k, my_k);
    in_order();
    const float* scales = reinterpret_cast<const float*>(my_scales);
    if constexpr (F8)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(scales + 32 * n + 8 * w + 4 * h);
          s[n][4 * w] *= x.x, s[n][4 * w + 1] *= x.y, s[n][4 * w + 2] *= x.z, s[n][4 * w + 3] *= x.w;
        }
    if (ok != (KB == 64 ? ~0ull : 0xffffffffull) || k0 + KB > all_see)
#pragma unroll
      for (int n = 0; n < NT; ++n) hide(s[n], static_cast<uint32_t>(ok >> (32 * n)) & first_bits(row.seen - k0 - 32 * n), h);
    sums.raise(s, a.c);
    const float mc = sums.m == -kInf ? 0.f : sums.m * a.c;
    float l[2] = {0.f, 0.f};
    u32x4 p[2 * NT], p2[kTwice<DT, F8> ? 2 * NT : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.c, -mc));
        l[r & 1] += s[n][r];
        // (e4m3: the next keys' loads between the powers.  64 x 32 queries over 800 to 912 keys 41.0 -> 39.9 us, 64 single tokens 21.0 -> 20.6; of bf16
        // keys 32 requests' drafts 67.8 -> 69.2.)
        if (F8 && r % 2) {
          in_order();
#pragma unroll
          for (int u = 0; u < kLoads; ++u)
            if (u * (8 * NT) / kLoads == 8 * n + r / 2 && more) load_part(u, a.k, my_k);
          in_order();
        }
      }
      if constexpr (F8)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(scales + KB + 32 * n + 8 * w + 4 * h);
          s[n][4 * w] *= x.x, s[n][4 * w + 1] *= x.y, s[n][4 * w + 2] *= x.z, s[n][4 * w + 3] *= x.w;
        }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (kTwice<DT, F8>) pack_twice(s[n], t, p[2 * n + t], p2[2 * n + t]);
        else p[2 * n + t] = pack_step<PT>(s[n], t);
      }
    }
    sums.l += l[0] + l[1];
    in_order();
    wait(more);
    {
      constexpr int kReads = 2 * NT * T::kOut, kAhead = F8 ? 6 : 4;
      using Read = std::conditional_t<F8, u32x2, u32x4>;
      auto read = [&](int j) -> Read {
        const int t = j / T::kOut, o = j % T::kOut;
        if constexpr (F8) {
          typedef int i32x2 __attribute__((ext_vector_type(2)));
          typedef __attribute__((address_space(3))) i32x2* P;
          int chunk = 2 * o + ((lane >> 4) & 1);
          if (R::kChunks % 2 != 0) chunk = min(chunk, R::kChunks - 1);  // (channels past the last: read, not used)
          return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((P)(my_v + R::at(16 * t + raw_row, chunk) + 8 * (lane & 1))));
        } else {
          return read_cols<D>(my_v, 0, t, o, cols_at);
        }
      };
      Read f[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) f[j] = read(j);
      in_order();
#pragma unroll
      for (int j = 0; j < kReads; ++j) {
        const int t = j / T::kOut, o = j % T::kOut;
        u32x4 x;
        if constexpr (F8) x = widen8<PT>(f[j % kAhead][0], f[j % kAhead][1]);
        else x = f[j % kAhead];
        sums.acc[o] = mfma<PT>(x, p[t], sums.acc[o]);
        if constexpr (kTwice<DT, F8>) sums.acc[o] = mfma<PT>(x, p2[t], sums.acc[o]);
        if (j + kAhead < kReads) f[j % kAhead] = read(j + kAhead);
        in_order();
      }
    }
    wait_lds();
    in_order();
    const KeyRow next = find(i + 2, page);
    page = ask(i + 3);
    in_order();
    if (more) load_values();
    in_order();
    ok = ok_next;
    take(next);
  }
  // ---- the wavefronts' sums together: each leaves its own where its slots were, 64 channels a row in either array, and 16 lanes (8 of 64
  // channels) finish a row.
  constexpr int kLanes = D == 64 ? 8 : 16, kFinish = 256 / kLanes;
  __shared__ float2 s_stats[4][32];
  __shared__ uint32_t s_again[4];
  auto sum_at = [&](int w, int r, int chunk) {  // 4 channels of row r that wavefront w left
    return reinterpret_cast<float4*>((chunk < 16 ? lds_k : lds_v) + w * kFewSlot + r * 256 + ((chunk ^ r) & 15) * 16);
  };
  const float l_mine = both_sum(sums.l);
  const uint32_t odd = columns(not_numbers<D>(sums.acc) && row.live && mine > 0);
  if (row.live) {
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (32 * o + 8 * w < D) *sum_at(wave, lane & 31, 8 * o + 2 * w + h) = float4{sums.acc[o][4 * w], sums.acc[o][4 * w + 1], sums.acc[o][4 * w + 2], sums.acc[o][4 * w + 3]};
    if (h == 0) s_stats[wave][lane] = float2{sums.m, l_mine};
  }
  if (lane == 0) s_again[wave] = odd;
  __syncthreads();
  auto joined = [&](int block, int r, float& top, float& l, float (&f)[4]) {
    top = -kInf, l = 0.f;
    for (int u = 0; u < kws; ++u) top = fmaxf(top, s_stats[u * blocks + block][r].x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f[u] = 0.f;
      if (u >= kws) continue;
      const float2 st = s_stats[u * blocks + block][r];
      f[u] = st.x == -kInf ? 0.f : __builtin_amdgcn_exp2f((st.x - top) * a.c);
      l += st.x == -kInf ? 0.f * st.y : st.y * f[u];
    }
  };
  const int c = tid % kLanes;
#pragma unroll 1
  for (int i = tid / kLanes; i < g.rows; i += kFinish) {
    float top, l, f[4];
    joined(i >> 5, i & 31, top, l, f);
    uint32_t again = 0;
    float v[8] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u >= kws) continue;
      const int w = u * blocks + (i >> 5);
      again |= s_again[w];
      if (8 * c >= D) continue;
      const float4 x = *sum_at(w, i & 31, 2 * c), y = *sum_at(w, i & 31, 2 * c + 1);
      v[0] += x.x * f[u], v[1] += x.y * f[u], v[2] += x.z * f[u], v[3] += x.w * f[u];
      v[4] += y.x * f[u], v[5] += y.y * f[u], v[6] += y.z * f[u], v[7] += y.w * f[u];
    }
    const bool store = 8 * c < D && !((again >> (i & 31) & 1) && l == l);
    if (g.whole) {
      const float inv = 1.f / l;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = l == 0.f ? 0.f : v[e] * inv;
      if (store) *reinterpret_cast<u32x4*>(a.out + result(a, row_at(a, g, i), D) + 8 * c) = pack16<DT>(v);
    } else {
      const int64_t at = static_cast<int64_t>(g.slot) * a.part_rows + i;
      if (store) {
        float4* to = reinterpret_cast<float4*>(a.sums + at * D + 8 * c);
        to[0] = float4{v[0], v[1], v[2], v[3]};
        to[1] = float4{v[4], v[5], v[6], v[7]};
      }
      if (c == 0) a.stats[at] = float2{top, l};
    }
  }
  if ((s_again[0] | s_again[1] | s_again[2] | s_again[3]) != 0 && kw == 0) {
    uint32_t again = 0;
    for (int u = 0; u < kws; ++u) again |= s_again[u * blocks + rb];
    float top, l, f[4];
    joined(rb, lane & 31, top, l, f);
    again = __builtin_amdgcn_readfirstlane(again) & columns(row.live && l == l);
    if (again != 0) rows_again<DT, D, F8>(a, g, rb * 32, again, top, l);
  }
  __syncthreads();  // (LDS is the next segment's)
}

// ---- many rows: 32 to a wavefront, 128 to a workgroup, which walks tiles of 64 keys together, loaded one ahead: straight to LDS, e4m3 through
// registers, where it is widened once for all four wavefronts.
template <int DT, int D, bool F8>
__device__ __forceinline__ void many_rows(const PagedArgs& a, const Segment& g) {
  using T = AttnTile<D>;
  constexpr int PT = kValues<DT, F8>, KB = 64, kTileBytes = KB * T::kPitch, kElem = F8 ? 1 : 2;
  unsigned char *const lds0 = lds_slot<kPagedLds<D>, 0>(), *const lds1 = lds_slot<kPagedLds<D>, 1>();
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (see few_rows)
  const int lane = tid & 63, rw = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int tiles = (g.hi - g.lo + KB - 1) / KB;
  auto ask = [&](int i) { return page_of(a, g, min(g.lo + i * KB + lane, g.hi - 1)); };  // a lane finds the row of one of a tile's 64 keys
  int p0 = 0, p1 = 0;
  if (tiles > 0) p0 = ask(0), p1 = ask(1);
  in_order();
  const Row row = row_at(a, g, rw * 32 + (lane & 31));
  u32x4 qf[T::kSteps];
  {
    const uint16_t* q = query(a, row);
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) qf[t] = *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h);
  }
  const bool wave_live = rw * 32 < g.rows;
  const int all_see = wave_extreme<false>(row.seen), some_sees = wave_live ? wave_extreme<true>(row.live ? row.seen : 0) : 0;
  wait_loads();  // (queries and pages, see few_rows)
  constexpr int kChunk = D / 16, kPieces = (KB * kChunk + 255) / 256;  // e4m3: 16-byte pieces of a row, of a thread
  // (Eight lanes write 16 bytes each at a time, every second of a row's: four of one row and four of the row whose swizzle has the others.  2048 tokens over
  // 16384 keys 307 -> 303 us.)
  auto piece_row = [](int n) { return D == 80 ? n / kChunk : (D == 128 ? n >> 4 & 3 | n >> 6 << 3 : n >> 3 & 3 | n >> 5 << 3) | (n & 4); };
  auto piece_chunk = [](int n) { return D == 80 ? n % kChunk : (n & 3) | (D == 128 ? n >> 1 & 4 : 0); };
  constexpr int kLoads = T::kChunks / 4;                               // otherwise: 16 rows by a wavefront
  uint32_t src[F8 ? kPieces : kLoads], scale_row = 0;
  uint64_t ok_next = 0;
  auto find = [&](int i, int page) {
    const int key = g.lo + i * KB + lane;
    KeyRow k = row_of(a, g, min(key, g.hi - 1), page);
    k.ok = k.ok && key < g.hi;
    return k;
  };
  auto take = [&](const KeyRow& k) {
    ok_next = __ballot(k.ok);
    scale_row = k.row;
    if constexpr (F8) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) src[u] = __shfl(k.row, piece_row(u * 256 + tid) & 63);
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) src[u] = __shfl(k.row, rw * 16 + (u * 64 + lane) / T::kChunks);
    }
  };
  u32x4 pk[F8 ? kPieces : 1], pv[F8 ? kPieces : 1];
  float scale = 0.f;
  constexpr int kWork = F8 ? 1 : 2 * kLoads;  // parts of a tile's loads
  auto fetch = [&](int w, unsigned char* slot) {
    if constexpr (F8) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int n = u * 256 + tid, c = piece_chunk(n);
        const uint64_t at = static_cast<uint64_t>(src[u]) * D + c * 16;
        if (KB * kChunk % 256 == 0 || n < KB * kChunk) {
          pk[u] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.k) + at);
          pv[u] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.v) + at);
        }
      }
      if (rw < 2) scale = (rw ? a.v_scale : a.k_scale)[scale_row];
    } else {
      const int u = w % kLoads, n = u * 64 + lane, c = (n % T::kChunks) ^ T::swizzle(n / T::kChunks);
      const char* const from = static_cast<const char*>(w < kLoads ? a.k : a.v);
      if (T::kChunks * 8 == D || c < D / 8)
        __builtin_amdgcn_global_load_lds(WX_GLOBAL(from + static_cast<uint64_t>(src[u]) * (2 * D) + c * 16),
                                         WX_LDS(slot + (w < kLoads ? 0 : kTileBytes) + rw * 16 * T::kPitch + u * 1024), 16, 0, 0);
    }
  };
  auto put = [&](unsigned char* slot) {
    if constexpr (F8) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int n = u * 256 + tid, r = piece_row(n), c = piece_chunk(n);
        if (KB * kChunk % 256 != 0 && n >= KB * kChunk) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          *reinterpret_cast<u32x4*>(slot + T::at(r, 2 * c + half)) = widen8<DT>(pk[u][2 * half], pk[u][2 * half + 1]);
          *reinterpret_cast<u32x4*>(slot + kTileBytes + T::at(r, 2 * c + half)) = widen8<PT>(pv[u][2 * half], pv[u][2 * half + 1]);
        }
      }
      if (rw < 2) reinterpret_cast<float*>(slot + 2 * kTileBytes)[rw * KB + lane] = scale;
    }
  };
  Sums<D> sums;
  sums.clear();
  const int rows_at = rows_base<D>(lane), cols_at = cols_base<D>(lane);
  auto step = [&](const unsigned char* tk, int k0, uint64_t ok, bool more, unsigned char* other) {
    constexpr int kAhead = D == 80 ? 3 : 4, NT = 2, kScores = NT * T::kSteps, kProducts = NT * 2 * T::kOut;
    const unsigned char* tv = tk + kTileBytes;
    const float* scales = reinterpret_cast<const float*>(tk + 2 * kTileBytes);
    int rows_here = rows_at, cols_here = cols_at;
    asm volatile("" : "+v"(rows_here), "+v"(cols_here));
    auto read_k = [&](int i) { return read_rows<D>(tk, 32 * (i % NT), i / NT, rows_here); };
    auto read_v = [&](int i) { return read_cols<D>(tv, 32 * (i / (2 * T::kOut)), i / T::kOut % 2, i % T::kOut, cols_here); };
    // (Scales are asked for as operands are, ahead: each read where it is used was a wait of its own.  2048 tokens over 16384 keys 348 -> 328 us.)
    // (Of fp16 with 128 channels half of them later: together they take registers that there are not, and a reload in the loop.)
    constexpr bool kLate = kTwice<DT, F8> && D == 128;
    float4 x0[F8 ? 4 : 1], x1[F8 ? 4 : 1];
    auto read_scales = [&](float4* x, int from) {
#pragma unroll
      for (int w = 0; w < 4; ++w) x[w] = *reinterpret_cast<const float4*>(scales + from + 8 * w + 4 * h);
    };
    auto times = [&](f32x16& s, const float4* x) {
#pragma unroll
      for (int w = 0; w < 4; ++w) s[4 * w] *= x[w].x, s[4 * w + 1] *= x[w].y, s[4 * w + 2] *= x[w].z, s[4 * w + 3] *= x[w].w;
    };
    f32x16 s[NT];
    u32x4 f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_k(i);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
    in_order();
    __builtin_amdgcn_s_setprio(1);  // (products go before the other wavefront's powers: 341 -> 331 us for 2048 tokens over 16384 keys)
#pragma unroll
    for (int i = 0; i < kScores; ++i) {
      s[i % NT] = mfma<DT>(f[i % kAhead], qf[i / NT], s[i % NT]);
      if (i + kAhead < kScores) f[i % kAhead] = read_k(i + kAhead);
      if (F8 && i + kAhead == kScores) read_scales(x0, 0);
      // (16 bits: the next tile's loads one at a time between the products.  All at once they wait for each other: 16 prompts of 912 tokens 99 -> 97 us.)
#pragma unroll
      for (int w = 0; !F8 && w < kWork; ++w)
        if (w * kScores / kWork == i && more) fetch(w, other);
      in_order();
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (F8) {
      if constexpr (!kLate) read_scales(x1, 32);
      in_order();
      times(s[0], x0);
      if constexpr (kLate) read_scales(x1, 32);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_v(i);
    in_order();
    if constexpr (F8) {
      times(s[1], x1);
      read_scales(x0, KB);
      in_order();
    }
    if (ok != ~0ull || k0 + KB > all_see)
#pragma unroll
      for (int n = 0; n < NT; ++n) hide(s[n], static_cast<uint32_t>(ok >> (32 * n)) & first_bits(row.seen - k0 - 32 * n), h);
    sums.raise(s, a.c);
    const float mc = sums.m == -kInf ? 0.f : sums.m * a.c;
    if constexpr (F8 && !kLate) {
      read_scales(x1, KB + 32);
      in_order();
    }
    float l[2] = {0.f, 0.f};
    auto power = [&](int n, int r) {  // of registers r and r + 1
      s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.c, -mc));
      s[n][r + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r + 1], a.c, -mc));
      l[0] += s[n][r];
      l[1] += s[n][r + 1];
      if constexpr (F8) {
        const float4 x = (n ? x1 : x0)[r / 4];
        s[n][r] *= r % 4 ? x.z : x.x, s[n][r + 1] *= r % 4 ? x.w : x.y;
      }
    };
#pragma unroll
    for (int u = 0; u < 8; ++u) power(0, 2 * u);
    if constexpr (kLate) {
      in_order();
      read_scales(x1, KB + 32);
      in_order();
    }
    u32x4 p[2], p2[2];
    auto pack = [&](int n) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (kTwice<DT, F8>) pack_twice(s[n], t, p[t], p2[t]);
        else p[t] = pack_step<PT>(s[n], t);
      }
    };
    pack(0);
    in_order();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int n = i / (2 * T::kOut), t = i / T::kOut % 2, o = i % T::kOut, at = i % (2 * T::kOut);
      if (n > 0 && at == 0) pack(n);
      sums.acc[o] = mfma<PT>(f[i % kAhead], p[t], sums.acc[o]);
      if constexpr (kTwice<DT, F8>) sums.acc[o] = mfma<PT>(f[i % kAhead], p2[t], sums.acc[o]);
      if (i + kAhead < kProducts) f[i % kAhead] = read_v(i + kAhead);
      if (n + 1 < NT) {
        const int each = (8 + 2 * T::kOut - 1) / (2 * T::kOut);
#pragma unroll
        for (int u = at * each; u < (at + 1) * each && u < 8; ++u) power(n + 1, 2 * u);
      }
      in_order();
    }
    __builtin_amdgcn_s_setprio(0);
    sums.l += l[0] + l[1];
  };
  uint64_t ok = 0;
  int page = 0;
  if (tiles > 0) {
    take(find(0, p0));
    const KeyRow next = find(1, p1);
#pragma unroll
    for (int w = 0; w < kWork; ++w) fetch(w, lds0);
    page = ask(2);
    ok = ok_next;
    take(next);
  }
  auto turn = [&](int i, unsigned char* slot, unsigned char* other) {
    const int k0 = g.lo + i * KB;
    const uint64_t seen = ok;
    const bool more = i + 1 < tiles;
    if constexpr (F8) {
      put(slot);
      const KeyRow next = find(i + 2, page);
      if (more) fetch(0, other);
      page = ask(i + 3);
      wait_lds();
      attn_barrier();
      ok = ok_next;
      take(next);
      in_order();
      if (k0 < some_sees) step(slot, k0, seen, more, other);
    } else {
      wait_loads();
      attn_barrier();
      in_order();
      if (k0 < some_sees) {
        step(slot, k0, seen, more, other);
      } else if (more) {
#pragma unroll
        for (int w = 0; w < kWork; ++w) fetch(w, other);
      }
      in_order();
      ok = ok_next;
      take(find(i + 2, page));
      page = ask(i + 3);
    }
  };
  for (int i = 0; i < tiles; i += 2) {
    turn(i, lds0, lds1);
    if (i + 1 < tiles) turn(i + 1, lds1, lds0);
  }
  const float l = both_sum(sums.l);
  const uint32_t again = columns(not_numbers<D>(sums.acc) && row.live && some_sees > g.lo) & columns(l == l);
  const bool store = row.live && !(again >> (lane & 31) & 1);
  if (g.whole) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (store && l == 0.f) {  // (0 * NaN otherwise)
#pragma unroll
      for (int c = 0; c < D / 8; c += 2) *reinterpret_cast<u32x4*>(a.out + result(a, row, D) + 8 * (c + h)) = u32x4{0u, 0u, 0u, 0u};
    }
    store_row<DT, D>(sums.acc, inv, store && l != 0.f ? a.out + result(a, row, D) : nullptr, lane);
  } else {
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
      if (store) store_sums<D>(sums.acc[o], o, a.sums + (static_cast<int64_t>(g.slot) * a.part_rows + row.at) * D, lane);
    if (row.live && h == 0) a.stats[static_cast<int64_t>(g.slot) * a.part_rows + row.at] = float2{sums.m, l};
  }
  if (again != 0) rows_again<DT, D, F8>(a, g, rw * 32, again, sums.m, l);
  __syncthreads();  // (LDS is the next segment's)
}

template <int DT, int D, bool F8>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedArgs a) {
  int none_from, none_to;
  const Share s = share<F8>(a, none_from, none_to);
  if (none_from > 0 || none_to < a.tokens) {
    const int64_t row = static_cast<int64_t>(a.n_q) * (D / 8), front = none_from * row, none = front + (a.tokens - none_to) * row;
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < none; i += static_cast<int64_t>(gridDim.x) * 256)
      reinterpret_cast<u32x4*>(a.out)[i < front ? i : i - front + none_to * row] = u32x4{0u, 0u, 0u, 0u};
  }
  const Part part = segments(
      a, s, [&](int r, int kind) { return next_request(a, r, kind); },
      [&](bool few, const Segment& g) {
        if (few) few_rows<DT, D, F8>(a, g);
        else many_rows<DT, D, F8>(a, g);
      });
  if (threadIdx.x == 0 && static_cast<int>(blockIdx.x) < a.shares) a.part[s.id] = part;
}

// Joins the parts of the item that begins in share blockIdx.x and ends in a later one.  16 lanes have a row, 8 channels each, and ask for 8 parts at
// a time.  Of up to 8 parts a wavefront has four rows; of more a workgroup, each wavefront a quarter of the parts.
constexpr int kJoinBlocks = 8;
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  __shared__ float4 s_sums[4][64][2];
  __shared__ float2 s_stats[4][4];
  const int id = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15;
  const Part p = uniform(a.part[id]);
  if (p.parts == 0) return;
  // (a part that the row sees nothing of has the weight 0 and sums of 0; what a row does see counts at the weight 0 as well, as NaN if it is not finite)
  auto weight = [&](float2 st, float top) { return st.x == -kInf ? 0.f : __builtin_amdgcn_exp2f((st.x - top) * a.c); };
  auto share_of = [](float2 st, float w) { return st.x == -kInf ? 0.f * st.y : st.y * w; };
  struct Sum {
    float top, l, o[8];
  };
  auto add = [&](Sum& s, float w, const float4& x, const float4& y) {
    s.o[0] += x.x * w, s.o[1] += x.y * w, s.o[2] += x.z * w, s.o[3] += x.w * w;
    s.o[4] += y.x * w, s.o[5] += y.y * w, s.o[6] += y.z * w, s.o[7] += y.w * w;
  };
  auto parts_of = [&](int row, int first, int last) {
    Sum s{-kInf, 0.f, {}};
    for (int i0 = first; i0 < last; i0 += 8) {
      float2 st[8];
      float4 x[8], y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {  // (past the last: the last one's, not added)
        const int i = min(i0 + u, last - 1);
        const int64_t at = static_cast<int64_t>(i == 0 ? 2 * id + 1 : 2 * (id + i)) * a.part_rows + row;
        st[u] = a.stats[at];
        const float4* from = reinterpret_cast<const float4*>(a.sums + at * D + 8 * c);
        x[u] = from[0], y[u] = from[1];
      }
      float top = s.top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (i0 + u >= last) st[u] = float2{-kInf, 0.f};
        top = fmaxf(top, st[u].x);
      }
      const float f = weight(float2{s.top, 0.f}, top);
      s.l = share_of(float2{s.top, s.l}, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s.o[e] *= f;
      s.top = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (i0 + u >= last) continue;
        const float w = weight(st[u], top);
        s.l += share_of(st[u], w);
        add(s, w, x[u], y[u]);
      }
    }
    return s;
  };
  auto store = [&](int row, Sum& s) {
    const float inv = 1.f / s.l;
#pragma unroll
    for (int e = 0; e < 8; ++e) s.o[e] = s.l == 0.f ? 0.f : s.o[e] * inv;
    const int at = p.row0 + row, i = a.by_group.div(at), hq = p.head * a.group + at - i * a.group;
    *reinterpret_cast<u32x4*>(a.out + (static_cast<int64_t>(p.first + i) * a.n_q + hq) * D + 8 * c) = pack16<DT>(s.o);
  };
  if (p.parts <= 8) {
    const int row = (blockIdx.y * 4 + wave) * 4 + (lane >> 4);
    if (row >= p.rows || 8 * c >= D) return;
    Sum s = parts_of(row, 0, p.parts);
    store(row, s);
    return;
  }
  const int each = (p.parts + 3) / 4, first = min(wave * each, p.parts), last = min(first + each, p.parts);
  for (int row0 = blockIdx.y * 4; row0 < p.rows; row0 += 4 * kJoinBlocks) {
    const int row = row0 + (lane >> 4);
    const bool live = row < p.rows && 8 * c < D;
    if (live) {
      const Sum s = parts_of(row, first, last);
      s_sums[wave][lane][0] = float4{s.o[0], s.o[1], s.o[2], s.o[3]};
      s_sums[wave][lane][1] = float4{s.o[4], s.o[5], s.o[6], s.o[7]};
      if (c == 0) s_stats[wave][lane >> 4] = float2{s.top, s.l};
    }
    __syncthreads();
    if (live && wave == 0) {
      Sum s{-kInf, 0.f, {}};
#pragma unroll
      for (int w = 0; w < 4; ++w) s.top = fmaxf(s.top, s_stats[w][lane >> 4].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 st = s_stats[w][lane >> 4];
        const float f = weight(st, s.top);
        s.l += share_of(st, f);
        add(s, f, s_sums[w][lane][0], s_sums[w][lane][1]);
      }
      store(row, s);
    }
    __syncthreads();
  }
}

int shares() { return std::max(8, 2 * device_cu_count() / 8 * 8); }
int part_rows(int64_t tokens, int group) { return static_cast<int>(std::min<int64_t>(kManyRows, tokens * group)); }

template <int DT, int D, bool F8>
int launch(PagedArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((paged_attn_kernel<DT, D, F8>), dim3(static_cast<unsigned>(a.blocks)), dim3(256), 0, s, a);
  if (int rc = check_launch("paged_attn_kernel")) return rc;
  hipLaunchKernelGGL((paged_join_kernel<DT, D>), dim3(static_cast<unsigned>(a.shares), kJoinBlocks), dim3(256), 0, s, a);
  return check_launch("paged_join_kernel");
}
template <int DT, bool F8>
int launch(PagedArgs& a, int head_dim, hipStream_t s) {
  if (head_dim == 64) return launch<DT, 64, F8>(a, s);
  if (head_dim == 80) return launch<DT, 80, F8>(a, s);
  return launch<DT, 128, F8>(a, s);
}

}  // namespace
}  // namespace wx

using namespace wx;

extern "C" size_t wx_paged_attention_workspace_bytes(int64_t tokens, int n_q_heads, int n_kv_heads, int head_dim) {
  if (tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0) return 0;
  const int64_t n = shares(), rows = 2 * n * part_rows(tokens, n_q_heads / n_kv_heads);
  return static_cast<size_t>(rows * (head_dim + 2) * 4 + n * static_cast<int64_t>(sizeof(Part)));
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
  if (num_pages > 0x7fffffffll / page_size || num_pages * page_size > 0xffffffffll / n_kv_heads) return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots or 2^32 - 1 rows of them", who);
  if (!q || !out || (requests > 0 && (!lengths || (pages_per_request > 0 && num_pages > 0 && (!page_table || !k_pages || !v_pages)))))
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  for (const void* p : {q, k_pages, v_pages, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0 || q_strides[i] < 0) return fail(WX_ERR_UNSUPPORTED, "%s: q's strides must be positive and keep rows 16-byte aligned", who);
  if (!workspace || workspace_bytes < wx_paged_attention_workspace_bytes(batch * seq, n_q_heads, n_kv_heads, head_dim))
    return fail(WX_ERR_WORKSPACE, "%s: workspace too small (see wx_paged_attention_workspace_bytes)", who);
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.k = k_pages, a.v = v_pages, a.k_scale = k_scale, a.v_scale = v_scale, a.out = static_cast<uint16_t*>(out);
  a.table = page_table, a.lengths = lengths, a.starts = starts, a.causal = causal != 0;
  a.tokens = static_cast<int>(batch * seq), a.requests = static_cast<int>(requests), a.n_q = n_q_heads, a.n_kv = n_kv_heads, a.group = group;
  a.seq = static_cast<int>(seq), a.width = num_pages ? static_cast<int>(pages_per_request) : 0, a.page_size = page_size, a.n_pages = static_cast<int>(num_pages);
  a.by_seq = Divider(static_cast<uint32_t>(seq)), a.by_page = Divider(page_size), a.by_group = Divider(group);
  a.c = scale * kLog2e;
  a.most_keys = a.width * page_size;
  a.shares = shares();
  const Launch l = launch_of(a.tokens, group, n_kv_heads, requests, seq, a.most_keys, starts != nullptr, a.shares);
  if (l.shift == 30) return fail(WX_ERR_UNSUPPORTED, "%s: too many requests or rows", who);
  a.shift = l.shift, a.blocks = l.blocks;
  a.part_rows = part_rows(a.tokens, group);
  const int64_t rows = 2ll * a.shares * a.part_rows;
  a.sums = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(a.sums + rows * head_dim);
  a.part = reinterpret_cast<Part*>(a.stats + rows);
  hipStream_t s = as_stream(stream);
  if (dtype == WX_BF16) return k_scale ? launch<WX_BF16, true>(a, head_dim, s) : launch<WX_BF16, false>(a, head_dim, s);
  return k_scale ? launch<WX_F16, true>(a, head_dim, s) : launch<WX_F16, false>(a, head_dim, s);
}
