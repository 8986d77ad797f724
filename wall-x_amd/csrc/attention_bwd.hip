// Attention backward (gfx950): with P = exp2(c S - L) recomputed from the scores and the forward's base-2 log-sum-exp L,
//   delta = rowsum(dO O),  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two kernels, seven matrix products in place of the five that share one pass: the first walks the keys of a tile of rows (dQ),
// the second the rows of a tile of keys (dK, dV, all heads of the group in turn).  Every sum is then one wavefront's own, in a
// fixed order: no atomics, the same gradients every time.
//
// 16 rows of 912 causal tokens of 16 / 2 heads of 128 (72 GFLOP in three products, 96 in four): dQ 124 us, 0.58 PFLOP/s, matrix units busy
// 31 % (the rows' four operands are on their way for a third of it); the plan 5; dK and dV 156 us, 0.62 PFLOP/s, 40 %, reading 0.6 GB of
// which half is in L2; the join 15.  5003 packed tokens of 12 / 4 heads of 64, fp16: 30, 8, 40 and 7 us.
#include <algorithm>

#include "attention.h"
#include "attention_plan.h"

namespace wx {

int attention_check(const char* who, int64_t batch, int n_q, int n_kv, int64_t n_queries, int64_t n_keys, int head_dim, int dtype, float scale);
int attention_check_strides(const char* who, const char* name, const int64_t* st, int elem_bytes, int64_t span, int64_t heads);

namespace {

struct BwdArgs {
  const uint16_t *q, *k, *v, *g;  // g = dO
  int64_t qs[3], ks[3], vs[3], gs[3];
  const uint16_t* out;            // [batch, n_queries, n_q, D]
  const uint8_t* rest;            // like out: what its rounding left times kRestUp, or null
  const float* lse;               // [batch, n_kv, rows]
  uint16_t *dq, *dk, *dv;         // [batch, n_queries, n_q, D], [batch, n_keys, n_kv, D]
  AttnMask mask;
  int batch, n_q, n_kv, n_queries, n_keys, group;
  int rows, row_blocks;           // rows of a pair, and 32-row blocks of them
  float c, scale;
  uint32_t* info;                 // [pair, row_block] blocks of kInfoWords
  int2* bounds;                   // [pair, row_block] the keys that any row of the block sees
  int key_tiles, more, units;     // of a pair: tiles of kKeyTile keys, what cutting them makes more than that at most, and the sum of both
  int aim;                        // what it should make more, if there is that much work
  Divider by_pairs, by_kv, by_group, by_in_group, by_tiles;  // by_pairs: of an XCD where they are dealt to XCDs, else all
  Spread spread;                  // of dQ's row tiles
  int4* list;                     // [pair, unit] key tile (-1: none), row blocks from .. up to, place of its sums (-1: the whole tile)
  int2* tiles;                    // [pair, key tile] number of its units, place of the first one's sums
  float* part;                    // [pair, place, kKeyTile, 2, D]
};

// What the second kernel reads of 32 rows: L (less kUp), delta, lo and hi of each, then the keys that all rows with keys see, whether some row
// sees a single one, and (fp16) the power of two that the slopes of all of them fit fp16 with.
constexpr int kInfoWords = 4 * 32 + 4;

// fp16's range is too short for probabilities of many keys and for their slopes: P is 1 / keys, dS as much smaller again as the gradient
// that comes in, and beyond 65504 where few keys meet a large one.  P enters its product times 2^15, which it cannot leave the range with.  dS of
// a row is formed times 2^15 as well (both are one subtraction from L), until a slope passes 2^15 (kMostSlope): then by as much less as
// takes the largest to below 2^10, and the sums so far with it.  The second kernel does the same for each key, of the rows that see it (so
// that a sequence's large gradients take nothing from its neighbours in the row), where the first found a slope as large among 32 rows.  Powers
// of two are exact, and taken back from the sums.  Forward and backward of 16 x 912 tokens in fp16 397 us, 386 with P and dS as they are; dQ's
// error for gradients of 0.001 over 8192 keys 0.096 % of its length (0.094 of it the result's own rounding), 0.76 with them.
template <int DT>
constexpr int kUp = DT == WX_F16 ? 15 : 0;
constexpr float kMostSlope = 32768.f;
constexpr int kSlopeTo = 9;
// By how many powers of two less a row's (key's) slopes go on, `top` being the largest of them that this lane is about to round; the same in
// both halves of a column.
__device__ __forceinline__ int slopes_less(float top) {
  top = both_max(top);
  return top > kMostSlope && top < kInf ? static_cast<int>(__float_as_uint(top) >> 23) - 127 - kSlopeTo : 0;
}

__device__ __forceinline__ const uint16_t* row_of(const uint16_t* p, const int64_t* st, int b, int h, int i) {
  return p + b * st[0] + h * st[1] + i * st[2];
}

// Rows whose sum is not a number though their L and delta are: again (see Odd, attention.h), those of this wavefront's that `again` has a bit
// for.  (A key that is not finite has no probability where L is a number, so that its slope times it is NaN.)  Their place is found once more:
// kept over the kernel's loop for this rare case it costs that registers.
template <int DT, int D, int RW>
__device__ __forceinline__ void dq_again(const BwdArgs& a, uint32_t again, float lse, float delta) {
  using T = AttnTile<D>;
  int id = blockIdx.x, tid = threadIdx.x;
  asm volatile("" : "+s"(id), "+v"(tid));
  const int lane = tid & 63, rw = __builtin_amdgcn_readfirstlane(tid >> 6) % RW, h = lane >> 5;
  int pair, tile;
  a.spread.place(id, pair, tile);
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int row = (tile * RW + rw) * 32 + (lane & 31), in_row = row < a.rows ? row : 0, qi = a.by_group.div(in_row), hq = hk * a.group + in_row - qi * a.group;
  const bool redo = again >> (lane & 31) & 1;
  int lo = 0, hi = 0;
  if (redo) key_range(a.mask, b, qi, a.n_queries, a.n_keys, lo, hi);
  const int from = wave_extreme<false>(redo ? lo : 0x7fffffff), up_to = wave_extreme<true>(hi);
  const char* kp = reinterpret_cast<const char*>(a.k + b * a.ks[0] + hk * a.ks[1]);
  const char* vp = reinterpret_cast<const char*>(a.v + b * a.vs[0] + hk * a.vs[1]);
  const int64_t k_step = a.ks[2] * 2, v_step = a.vs[2] * 2;
  const uint16_t *q = row_of(a.q, a.qs, b, hq, qi), *g = row_of(a.g, a.gs, b, hq, qi);
  uint16_t* const dq = a.dq + ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D;
  const float factor = hi - lo == 1 ? 0.f : a.scale * ldexpf(1.f, -kUp<DT>);
  float shifted = lse - kUp<DT>, back = 1.f;
  // the slopes of keys k0 .. + 31, zeros for what is not seen and for other rows
  auto in = [&](int k0, int i) { return min(i, a.n_keys - 1 - k0); };  // (a key past the last is the last, and not seen)
  auto slopes = [&](int k0, f32x16& s, uint32_t& seen) {
    const char *kr = kp + k0 * k_step + in(k0, lane & 31) * static_cast<int>(k_step), *vr = vp + k0 * v_step + in(k0, lane & 31) * static_cast<int>(v_step);
    f32x16 dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      s = mfma<DT>(*reinterpret_cast<const u32x4*>(kr + (16 * t + 8 * h) * 2), *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h), s);
      dp = mfma<DT>(*reinterpret_cast<const u32x4*>(vr + (16 * t + 8 * h) * 2), *reinterpret_cast<const u32x4*>(g + 16 * t + 8 * h), dp);
      in_order();
    }
    seen = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = k0 + 8 * (r / 4) + 4 * h + r % 4;
      const bool sees = redo && key >= lo && key < hi;
      s[r] = sees ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -shifted)) * (dp[r] - delta) : 0.f;
      seen |= sees ? 1u << r : 0u;
    }
  };
  if constexpr (DT == WX_F16) {
    float top = 0.f;
    for (int k0 = from; k0 < up_to; k0 += 32) {
      f32x16 s;
      uint32_t seen;
      slopes(k0, s, seen);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (fabsf(s[r]) < kInf) top = fmaxf(top, fabsf(s[r]));
    }
    const int less = slopes_less(top);
    shifted += static_cast<float>(less), back = ldexpf(1.f, less);
  }
  for (int o = 0; o < T::kOut; ++o) {
    f32x16 sum = {};
    const int c = 32 * o + (lane & 31);
    for (int k0 = from; k0 < up_to; k0 += 32) {
      f32x16 s;
      uint32_t seen;
      slopes(k0, s, seen);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Odd odd;
        const u32x4 x = gather_cols<DT>(t, h, odd, [&](int i) -> uint32_t {
          return D % 32 != 0 && c >= D ? 0u : *reinterpret_cast<const uint16_t*>(kp + k0 * k_step + (in(k0, i) * static_cast<int>(k_step) + 2 * c));
        });
        in_order();
        sum = mfma<DT>(x, pack_step<DT>(s, t), sum);
        odd.nan |= odd.plus | odd.minus, odd.plus = odd.minus = 0;
        add_odd<DT>(sum, odd, seen, 0, t);
        in_order();
      }
    }
    if constexpr (DT == WX_F16)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[r] *= back;
    store_cols<DT, D>(sum, o, factor, redo ? dq : nullptr, lane);
  }
}

template <int DT, int D, int RW>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(BwdArgs a) {
  using T = AttnTile<D>;
  constexpr int KB = 64, KW = 4 / RW, kTileBytes = KB * T::kPitch;
  static_assert(KW == 1 || (KW == 2 && RW * T::kOut * 16 * 64 * 4 <= 2 * kTileBytes), "the second key group's sums fit a slot");
  unsigned char *const lds0 = lds_slot<2 * kTileBytes, 0>(), *const lds1 = lds_slot<2 * kTileBytes, 1>();
  __shared__ int2 s_bounds[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int rw = wave % RW, kw = wave / RW;
  int pair, tile;
  a.spread.place(blockIdx.x, pair, tile);
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int row = (tile * RW + rw) * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int in_row = live ? row : 0, qi = a.by_group.div(in_row), hq = hk * a.group + in_row - qi * a.group;
  const MaskRow row_mask = mask_row(a.mask, b, qi, a.n_queries, a.n_keys);
  in_order();
  u32x2 rf[T::kSteps] = {};
  u32x4 qf[T::kSteps], gf[T::kSteps], of[T::kSteps];  // (asked for behind the mask and before anything that waits for it; a row past the last reads the first)
  {
    const uint16_t* q = row_of(a.q, a.qs, b, hq, qi);
    const uint16_t* g = row_of(a.g, a.gs, b, hq, qi);
    const uint16_t* o = a.out + ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D;
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      qf[t] = *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h);
      gf[t] = *reinterpret_cast<const u32x4*>(g + 16 * t + 8 * h);
      of[t] = *reinterpret_cast<const u32x4*>(o + 16 * t + 8 * h);
      if (a.rest != nullptr) rf[t] = *reinterpret_cast<const u32x2*>(a.rest + (o - a.out) + 16 * t + 8 * h);
    }
  }
  float lse = a.lse[static_cast<int64_t>(pair) * a.rows + in_row];
  in_order();
  int lo = 0, hi = 0;
  if (live) key_range(a.mask, row_mask, qi, a.n_queries, a.n_keys, lo, hi);
  const bool some = hi > lo;
  int w_lo = wave_extreme<false>(some ? lo : 0x7fffffff);
  const int w_hi = wave_extreme<true>(hi);
  const int f_lo = wave_extreme<true>(some ? lo : 0), f_hi = wave_extreme<false>(some ? hi : 0x7fffffff);
  w_lo = min(w_lo, w_hi);
  if (lane == 0) s_bounds[wave] = int2{w_hi > w_lo ? w_lo : 0x7fffffff, w_hi};
  attn_lds_barrier();
  int g_lo = 0x7fffffff, g_hi = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    g_lo = min(g_lo, s_bounds[u].x);
    g_hi = max(g_hi, s_bounds[u].y);
  }
  g_hi = __builtin_amdgcn_readfirstlane(g_hi);
  g_lo = __builtin_amdgcn_readfirstlane(min(g_lo, g_hi));
  const int iters = (g_hi - g_lo + KB - 1) / KB;

  const char* kp = reinterpret_cast<const char*>(a.k + b * a.ks[0] + hk * a.ks[1]);
  const char* vp = reinterpret_cast<const char*>(a.v + b * a.vs[0] + hk * a.vs[1]);
  const int64_t k_step = a.ks[2] * 2, v_step = a.vs[2] * 2;
  uint32_t k_off[T::kChunks / 4], v_off[T::kChunks / 4];
#pragma unroll
  for (int i = 0; i < T::kChunks / 4; ++i) {
    k_off[i] = stage_offset<D>(i, lane, [&](int r) { return static_cast<uint32_t>((wave * 16 + r) * static_cast<int>(k_step)); });
    v_off[i] = stage_offset<D>(i, lane, [&](int r) { return static_cast<uint32_t>((wave * 16 + r) * static_cast<int>(v_step)); });
  }
  auto fetch = [&](int it, unsigned char* slot) {
    const int k0 = g_lo + it * KB, left = g_hi - k0, r0 = wave * 16;
    const auto rk = attn_rsrc(kp + k0 * k_step, kRsrcBytes), rv = attn_rsrc(vp + k0 * v_step, kRsrcBytes);
    if (left >= KB) {
      stage16<D>(rk, slot + r0 * T::kPitch, k_off);
      stage16<D>(rv, slot + kTileBytes + r0 * T::kPitch, v_off);
    } else {
      stage16<D>(rk, slot + r0 * T::kPitch, lane, [&](int r) { return r0 + r < left ? static_cast<uint32_t>((r0 + r) * static_cast<int>(k_step)) : kOutside; });
      stage16<D>(rv, slot + kTileBytes + r0 * T::kPitch, lane, [&](int r) { return r0 + r < left ? static_cast<uint32_t>((r0 + r) * static_cast<int>(v_step)) : kOutside; });
    }
  };
  if (iters > 0) fetch(0, lds0);

  float sums[2] = {0.f, 0.f}, rests = 0.f;
#pragma unroll
  for (int t = 0; t < T::kSteps; ++t) {
#pragma unroll
    for (int u = 0; u < 4; ++u) sums[u & 1] = dot2<DT>(gf[t][u], of[t][u], sums[u & 1]);
#pragma unroll
    for (int u = 0; u < 2; ++u) rests = dot2<DT>(gf[t][2 * u + 1], widen_rest2<DT, true>(rf[t][u]), dot2<DT>(gf[t][2 * u], widen_rest2<DT, false>(rf[t][u]), rests));
  }
  rests = both_sum(rests) * (1.f / kRestUp<DT>);
  // (rests that e5m2 does not hold are left out)
  const float delta = some ? both_sum(sums[0] + sums[1]) + (fabsf(rests) < kInf ? rests : 0.f) : 0.f;
  lse = some ? lse : kInf;
  constexpr bool kFit = DT == WX_F16;
  int up = kUp<DT>;  // this row's slopes are formed times 2^up
  float shifted = lse - kUp<DT>;
  float l_info = shifted;
  if (__any(delta != delta)) {  // a row whose gradient is NaN throughout makes all of dV NaN as well: said by its L, so that nothing is done again for it
    bool all = delta != delta;
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x = Elem<DT>::load(gf[t][u] & 0xffffu), y = Elem<DT>::load(gf[t][u] >> 16);
        all = all && x != x && y != y;
      }
    const uint64_t rows = __ballot(all);
    if ((rows & rows >> 32) >> (lane & 31) & 1) l_info = __builtin_nanf("");
  }
  const int block = tile * RW + rw, one = __any(hi - lo == 1);
  if (kw == 0 && block < a.row_blocks) {
    const int64_t at = static_cast<int64_t>(pair) * a.row_blocks + block;
    uint32_t* info = a.info + at * kInfoWords;
    info[(h ? 64 : 0) + (lane & 31)] = h ? static_cast<uint32_t>(lo) : __float_as_uint(l_info);
    info[(h ? 96 : 32) + (lane & 31)] = h ? static_cast<uint32_t>(hi) : __float_as_uint(delta);
    if (lane == 0) {
      *reinterpret_cast<int4*>(info + 128) = int4{f_lo, f_hi, one, 0};
      a.bounds[at] = int2{w_lo, w_hi};
    }
  }

  f32x16 acc[T::kOut];
#pragma unroll
  for (int o = 0; o < T::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[o][r] = 0.f;
  // Keeps the row's slopes in fp16's range: `top` is the largest of what this lane is about to round.
  auto fit = [&](f32x16& s, int from, float top) {
    if (!__any(top > kMostSlope && top < kInf)) return;
    const int less = slopes_less(top);
    const float f = ldexpf(1.f, -less);
    up -= less;
    shifted += static_cast<float>(less);
#pragma unroll
    for (int r = 0; r < 8; ++r) s[from + r] *= f;
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[o][r] *= f;
  };
  const int rows_first = rows_base<D>(lane), cols_first = cols_base<D>(lane);
  auto turn = [&](int it, unsigned char* tk, unsigned char* other) {
    wait_loads();
    attn_barrier();
    if (it + 1 < iters) fetch(it + 1, other);
    const unsigned char* tv = tk + kTileBytes;
#pragma unroll
    for (int i = 0; i < KB / 32 / KW; ++i) {
      const int n = KW == 1 ? i : kw, k0 = g_lo + it * KB + 32 * n;
      if (k0 >= w_hi || k0 + 32 <= w_lo) continue;
      // A product's operand is asked for kAhead products before it; the second half's powers are found under the first half's products.
      constexpr int kAhead = D == 80 ? 2 : 3, kScores = 2 * T::kSteps, kProducts = 2 * T::kOut;
      int rows_at = rows_first, cols_at = cols_first;
      asm volatile("" : "+v"(rows_at), "+v"(cols_at));
      auto read_s = [&](int i) { return read_rows<D>(i % 2 == 0 ? tk : tv, 32 * n, i / 2, rows_at); };
      auto read_k = [&](int i) { return read_cols<D>(tk, 32 * n, i / T::kOut, i % T::kOut, cols_at); };
      f32x16 s, dp;
      u32x4 f[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) f[i] = read_s(i);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
      in_order();
#pragma unroll
      for (int i = 0; i < kScores; ++i) {
        if (i % 2 == 0) s = mfma<DT>(f[i % kAhead], qf[i / 2], s);
        else dp = mfma<DT>(f[i % kAhead], gf[i / 2], dp);
        if (i + kAhead < kScores) f[i % kAhead] = read_s(i + kAhead);
        in_order();
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) f[i] = read_k(i);
      in_order();
      if (k0 < f_lo || k0 + 32 > f_hi) {
        const uint32_t span = static_cast<uint32_t>(hi - lo);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = static_cast<uint32_t>(k0 + 4 * h + 8 * (r / 4) + r % 4 - lo) < span ? s[r] : -kInf;
      }
      float top = 0.f;
      auto slope = [&](int r) {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -shifted)) * (dp[r] - delta);
        if constexpr (kFit) top = fmaxf(top, fabsf(s[r]));
      };
#pragma unroll
      for (int r = 0; r < 8; ++r) slope(r);
      if constexpr (kFit) {
        fit(s, 0, top);
        top = 0.f;
      }
      u32x4 ds = pack_step<DT>(s, 0);
      in_order();
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        if (i == T::kOut) {
          if constexpr (kFit) fit(s, 8, top);
          ds = pack_step<DT>(s, 1);
        }
        acc[i % T::kOut] = mfma<DT>(f[i % kAhead], ds, acc[i % T::kOut]);
        if (i + kAhead < kProducts) f[i % kAhead] = read_k(i + kAhead);
        if (i < T::kOut) {
          constexpr int each = (8 + T::kOut - 1) / T::kOut;
#pragma unroll
          for (int r = 8 + i * each; r < 8 + (i + 1) * each && r < 16; ++r) slope(r);
        }
        in_order();
      }
    }
  };
  for (int it = 0; it < iters; it += 2) {
    turn(it, lds0, lds1);
    if (it + 1 < iters) turn(it + 1, lds1, lds0);
  }
  int block_up = kUp<DT>;
  if constexpr (kFit) {
    block_up = wave_extreme<false>(up);
    if (block_up < kUp<DT>) {  // (of the wavefront's rows: the sums of all in the same power again)
      const float f = ldexpf(1.f, kUp<DT> - up);
#pragma unroll
      for (int o = 0; o < T::kOut; ++o)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[o][r] *= f;
    }
  }
  if constexpr (KW == 2) {  // the second key group's sums to the first
    float* const at = reinterpret_cast<float*>(lds0) + rw * (T::kOut * 16 * 64) + lane;
    __syncthreads();
    if (kw == 1) {
#pragma unroll
      for (int o = 0; o < T::kOut; ++o)
#pragma unroll
        for (int r = 0; r < 16; ++r) at[(16 * o + r) * 64] = acc[o][r];
      if (kFit && lane == 0) s_bounds[rw].x = block_up;
    }
    __syncthreads();
    if (kw == 1) return;
    if constexpr (kFit) block_up = min(block_up, s_bounds[rw].x);
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[o][r] += at[(16 * o + r) * 64];
  }
  if (kFit && lane == 0 && block < a.row_blocks) a.info[(static_cast<int64_t>(pair) * a.row_blocks + block) * kInfoWords + 131] = static_cast<uint32_t>(block_up);
  const uint32_t again = columns(not_numbers<D>(acc) && some && lse == lse && delta == delta);
  if (!some) {
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[o][r] = 0.f;
  }
  // (a row of one key has no slope: its sum is what rounding left of dP - delta)
  const float factor = hi - lo == 1 ? 0.f : a.scale * ldexpf(1.f, -kUp<DT>);
  uint16_t* const dq = a.dq + ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D;
  store_row<DT, D>(acc, factor, live ? dq : nullptr, lane);
  if (again != 0) dq_again<DT, D, RW>(a, again, lse, delta);
}

// What the workgroups of the next kernel do (attention_plan.h): a workgroup per pair, a lane per key tile, the row blocks dealt to 16
// wavefronts.
__global__ __launch_bounds__(1024) void attn_plan_kernel(BwdArgs a) {
  constexpr int kChunk = 4096;
  __shared__ int s_first[kPlanTiles], s_last[kPlanTiles];
  __shared__ int2 s_bounds[kChunk];
  const int pair = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int2* bounds = a.bounds + static_cast<int64_t>(pair) * a.row_blocks;
  int4* list = a.list + static_cast<int64_t>(pair) * a.units;
  for (int c0 = 0; c0 < a.key_tiles; c0 += kPlanTiles) {
    const int n_tiles = min(a.key_tiles - c0, kPlanTiles);
    s_first[tid] = 0x7fffffff, s_last[tid] = -1;
    for (int t0 = 0; t0 < a.row_blocks; t0 += kChunk) {
      const int n = min(a.row_blocks - t0, kChunk);
      if (t0 > 0) __syncthreads();
      for (int t = tid; t < n; t += 1024) s_bounds[t] = bounds[t0 + t];
      __syncthreads();
      for (int c = 0; c < n_tiles; c += 64) {
        const int k0 = (c0 + c + lane) * kKeyTile;
        int first = 0x7fffffff, last = -1;
#pragma unroll 4
        for (int t = tid >> 6; t < n; t += 16) {
          const int2 x = s_bounds[t];
          const bool sees = x.x < k0 + kKeyTile && x.y > k0 && x.y > x.x;
          first = sees ? min(first, t0 + t) : first;
          last = sees ? t0 + t : last;
        }
        if (last >= 0) {
          atomicMin(&s_first[c + lane], first);
          atomicMax(&s_last[c + lane], last);
        }
      }
    }
    __syncthreads();
    if (a.more == 0) {  // every tile is a unit
      if (tid < n_tiles) list[c0 + tid] = int4{c0 + tid, s_last[tid] < 0 ? 0 : s_first[tid], s_last[tid] + 1, -1};
      __syncthreads();
    }
  }
  if (a.more == 0 || tid >= 64) return;
  int2* tiles = a.tiles + static_cast<int64_t>(pair) * a.key_tiles;
  int64_t work = 0;
  for (int t = lane; t < a.key_tiles; t += 64) work += max(s_last[t] - s_first[t] + 1, 0);
#pragma unroll
  for (int n = 1; n < 64; n *= 2) work += __shfl_xor(static_cast<long long>(work), n);
  const int unit = unit_blocks(work, a.aim);
  int next = 0;  // (never past a.units)
  for (int c = 0; c < a.key_tiles; c += 64) {
    const bool is = c + lane < a.key_tiles;
    const int from = is ? s_first[c + lane] : 0, blocks = is ? max(s_last[c + lane] - from + 1, 0) : 0;
    const int units = is ? tile_units(blocks, unit) : 0;
    int up_to = units;
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
      const int x = __shfl_up(up_to, n);
      if (lane >= n) up_to += x;
    }
    const int at = next + up_to - units;
    const int each = units > 0 ? (blocks + units - 1) / units : 0;
    for (int u = 0; u < units; ++u)
      list[at + u] = int4{c + lane, blocks > 0 ? from + min(blocks, u * each) : 0, blocks > 0 ? from + min(blocks, (u + 1) * each) : 0, units > 1 ? at + u : -1};
    if (is) tiles[c + lane] = int2{units, at};
    next += __shfl(up_to, 63);
  }
  for (int u = next + lane; u < a.units; u += 64) list[u] = int4{-1, 0, 0, -1};
}

// The pair of a workgroup of the next kernel, and which of its units it takes.  (The pair varies fastest: dealt to the XCDs by their unit, a
// tile's first units all went to a few.)
__device__ __forceinline__ int todo_pair(const BwdArgs& a, int* unit = nullptr) {
  const int pairs = a.batch * a.n_kv, id = blockIdx.x, from = pairs % 8 == 0 ? id >> 3 : id, per = pairs % 8 == 0 ? pairs >> 3 : pairs;
  const int u = a.by_pairs.div(from);
  if (unit != nullptr) *unit = u;
  return pairs % 8 == 0 ? (id & 7) * per + (from - u * per) : from - u * per;
}

// Keys whose sum is not a number: again (see Odd, attention.h), those of this wavefront's that `again` has a bit for, over all rows of its
// unit, dK's slopes times `of`, unless a row that sees the key makes the whole sum NaN (by its L, or for dK by its delta).  (A query that is not finite has no
// probability where its L is a number, so that its slope times it is NaN.)  The place is found once more, as in dq_again.
template <int DT, int D>
__device__ __forceinline__ void dkv_again(const BwdArgs& a, uint32_t again, int4 todo, float of) {
  using T = AttnTile<D>;
  int tid = threadIdx.x, pair = todo_pair(a), tile = __builtin_amdgcn_readfirstlane(todo.x), first = __builtin_amdgcn_readfirstlane(todo.y);
  const int last = __builtin_amdgcn_readfirstlane(todo.z);
  asm volatile("" : "+v"(tid), "+s"(pair), "+s"(tile), "+s"(first));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, half = wave & 1, rg = wave >> 1;
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int k0 = tile * kKeyTile, key = k0 + half * 32 + (lane & 31);
  const uint16_t* qb = a.q + b * a.qs[0] + static_cast<int64_t>(hk) * a.group * a.qs[1];
  const uint16_t* gb = a.g + b * a.gs[0] + static_cast<int64_t>(hk) * a.group * a.gs[1];
  const uint32_t* info_base = a.info + static_cast<int64_t>(pair) * a.row_blocks * kInfoWords;
  for (int t = last - 1; t >= first && again != 0; --t) {  // (the last rows first: under a causal mask they see the most)
    const uint32_t* info = info_base + static_cast<int64_t>(t) * kInfoWords;
    const float l = __uint_as_float(info[lane & 31]), delta = __uint_as_float(info[32 + (lane & 31)]);
    for (uint32_t rows = columns(l != l || (rg == 0 && delta != delta)); rows != 0 && again != 0; rows &= rows - 1) {
      const int i = __builtin_ctz(rows);
      again &= ~columns(key >= static_cast<int>(info[64 + i]) && key < static_cast<int>(info[96 + i]));
    }
  }
  if (again == 0) return;
  const bool redo = again >> (lane & 31) & 1, whole = todo.w < 0;
  const int in_key = key < a.n_keys ? key : 0;
  const uint16_t *k = row_of(a.k, a.ks, b, hk, in_key), *v = row_of(a.v, a.vs, b, hk, in_key);
  const float scale = rg == 0 ? a.scale : 1.f;
  uint16_t* const grad = rg == 0 ? a.dk : a.dv;
  float* const part = a.part + (static_cast<int64_t>(pair) * a.units + todo.w) * (kKeyTile * 2 * D) + rg * D;
  auto row_at = [&](const uint16_t* base, const int64_t* st, int t, int i) {  // (a row past the last is the last, and sees nothing here)
    const int row = min(t * 32 + i, a.rows - 1), at = a.by_group.div(row);
    return base + at * st[2] + (row - at * a.group) * st[1];
  };
  const float back = ldexpf(1.f, -kUp<DT>) / of;
  for (int o = 0; o < T::kOut; ++o) {
    f32x16 sum = {};
    const int c = 32 * o + (lane & 31);
    for (int t = first; t < last; ++t) {
      const uint32_t* info = info_base + static_cast<int64_t>(t) * kInfoWords;
      const uint16_t *q = row_at(qb, a.qs, t, lane & 31), *g = row_at(gb, a.gs, t, lane & 31);
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int u = 0; u < T::kSteps; ++u) {
        s = mfma<DT>(*reinterpret_cast<const u32x4*>(q + 16 * u + 8 * h), *reinterpret_cast<const u32x4*>(k + 16 * u + 8 * h), s);
        dp = mfma<DT>(*reinterpret_cast<const u32x4*>(g + 16 * u + 8 * h), *reinterpret_cast<const u32x4*>(v + 16 * u + 8 * h), dp);
        in_order();
      }
      uint32_t seen = 0, zero = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 8 * (r / 4) + 4 * h + r % 4, lo = static_cast<int>(info[64 + i]), hi = static_cast<int>(info[96 + i]);
        const bool sees = redo && key >= lo && key < hi;
        float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -__uint_as_float(info[i])));
        if (rg == 0) {
          const float delta = __uint_as_float(info[32 + i]);
          x *= ((hi - lo == 1 ? delta : dp[r]) - delta) * of;
        }
        s[r] = sees ? x : 0.f;
        seen |= sees ? 1u << r : 0u;
        zero |= sees && x == 0.f ? 1u << r : 0u;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        Odd odd;
        const u32x4 x = gather_cols<DT>(u, h, odd, [&](int i) -> uint32_t {
          return D % 32 != 0 && c >= D ? 0u : *((rg == 0 ? row_at(qb, a.qs, t, i) : row_at(gb, a.gs, t, i)) + c);
        });
        in_order();
        sum = mfma<DT>(x, pack_step<DT>(s, u), sum);
        if (rg == 0) odd.nan |= odd.plus | odd.minus, odd.plus = odd.minus = 0;
        add_odd<DT>(sum, odd, seen, rg == 0 ? 0u : zero, u);
        in_order();
      }
    }
    if constexpr (DT == WX_F16)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[r] *= back;
    if (whole) store_cols<DT, D>(sum, o, scale, redo ? grad + ((static_cast<int64_t>(b) * a.n_keys + key) * a.n_kv + hk) * D : nullptr, lane);
    else if (redo) store_sums<D>(sum, o, part + (key - k0) * 2 * D, lane);
  }
}

// A wavefront holds 32 keys (K and V as B operands, dK^T and dV^T as accumulators) and takes every second block of 32 rows of Q and dO
// of the workgroup's unit; two such wavefronts make the 64 keys of a workgroup, and the other two take the blocks in between.  S has
// rows in its registers here and a key per column, so that P and dS are the B operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
// A tile of one unit writes its gradients, the others' units write their sums, which attn_dkv_join_kernel adds up.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(BwdArgs a) {
  using T = AttnTile<D>;
  constexpr int kTileBytes = 32 * T::kPitch, kInfoBytes = (kInfoWords * 4 + 63) / 64 * 64, kSlot = 2 * kTileBytes + kInfoBytes;
  constexpr int kSums = T::kOut * 16 * 64 * 4;  // one wavefront's sums of one gradient
  unsigned char* const lds0 = lds_slot<(2 * kSlot > 2 * kSums ? 2 * kSlot : 2 * kSums), 0>();
  unsigned char* const lds1 = lds_slot<(2 * kSlot > 2 * kSums ? 2 * kSlot : 2 * kSums), 1>();
  __shared__ u32x4 s_offsets[256];
  __shared__ float s_slope[DT == WX_F16 ? 4 : 1][32];
  // (D = 128: two of V's operands stand in LDS, read in front of their products; with all in registers one was spilled, and the wait
  // for its memory was a wait for the next block's as well)
  constexpr int kHeld = D == 128 ? T::kSteps - 2 : T::kSteps;
  __shared__ u32x4 s_v[kHeld < T::kSteps ? T::kSteps - kHeld : 1][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int half = wave & 1, rg = wave >> 1;
  int unit;
  const int pair = todo_pair(a, &unit);
  const int4 todo = a.list[static_cast<int64_t>(pair) * a.units + unit];
  const int tile = __builtin_amdgcn_readfirstlane(todo.x), first = __builtin_amdgcn_readfirstlane(todo.y), last = __builtin_amdgcn_readfirstlane(todo.z);
  if (tile < 0) return;
  const bool whole = todo.w < 0;
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int k0 = tile * kKeyTile, wk = k0 + half * 32, key = wk + (lane & 31);
  const bool live = key < a.n_keys;

  const uint16_t* qb = a.q + b * a.qs[0] + static_cast<int64_t>(hk) * a.group * a.qs[1];
  const uint16_t* gb = a.g + b * a.gs[0] + static_cast<int64_t>(hk) * a.group * a.gs[1];
  const char* src = reinterpret_cast<const char*>(half == 0 ? qb : gb);  // this wavefront loads its group's queries, or their gradients
  const int64_t pos_step = (half == 0 ? a.qs[2] : a.gs[2]) * 2;
  const int head_step = static_cast<int>((half == 0 ? a.qs[1] : a.gs[1]) * 2), pos_step32 = static_cast<int>(pos_step);
  const uint32_t* info_base = a.info + static_cast<int64_t>(pair) * a.row_blocks * kInfoWords;
  // Offsets of a block's rows from its first: the same for every block where the group divides 32 or 32 the group.  They are kept in
  // LDS, for want of registers.
  const bool regular = 32 % a.group == 0 || a.group % 32 == 0;
  const int in_group = a.group < 32 ? a.group : 32;
  const int second = in_group == 32 ? 16 * head_step : a.by_in_group.div(16) * pos_step32;  // from the first 16 rows to the others
  {
    uint32_t off[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < T::kChunks / 4; ++i)
      off[i] = stage_offset<D>(i, lane, [&](int r) {
        const int di = a.by_in_group.div(r), hd = r - di * in_group;
        return static_cast<uint32_t>(di * pos_step32 + hd * head_step);
      });
    s_offsets[tid] = u32x4{off[0], off[1], off[2], off[3]};
  }
  auto fetch = [&](int t, unsigned char* slot) {
    const int row0 = t * 32, i0 = a.by_group.div(row0), rem = row0 - i0 * a.group;
    const char* base = src + __builtin_amdgcn_readfirstlane(i0) * pos_step;
    unsigned char* to = slot + half * kTileBytes;
    if (regular && row0 + 32 <= a.rows) {
      const auto r = attn_rsrc(base + __builtin_amdgcn_readfirstlane(rem) * static_cast<int64_t>(head_step), kRsrcBytes);
      const u32x4 o = s_offsets[tid];
      const uint32_t off[4] = {o[0], o[1], o[2], o[3]};
      stage16<D>(r, to, off);
      stage16<D>(r, to + 16 * T::kPitch, off, second);
    } else {
      int here = lane;
      asm volatile("" : "+v"(here));  // (what this path needs is made here, not kept over the loop)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        stage16<D>(attn_rsrc(base, kRsrcBytes), to + u * 16 * T::kPitch, here, [&](int r) {
          const uint32_t x = static_cast<uint32_t>(rem + 16 * u + r), di = static_cast<uint32_t>(a.by_group.div(static_cast<int>(x))), hd = x - di * a.group;
          return row0 + 16 * u + r < a.rows ? di * static_cast<uint32_t>(pos_step32) + hd * static_cast<uint32_t>(head_step) : kOutside;
        });
    }
    if (half == 1 && lane < kInfoWords / 4)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(attn_rsrc(info_base + static_cast<int64_t>(t) * kInfoWords, kInfoWords * 4), WX_LDS(slot + 2 * kTileBytes), 16,
                                               lane * 16, 0, 0, 0);
  };
  unsigned char *mine = lds0 + rg * kSlot, *other = lds1 + rg * kSlot;
  if (first + rg < last) fetch(first + rg, mine);

  u32x4 kf[T::kSteps], vf[kHeld];
  {
    const uint16_t* k = row_of(a.k, a.ks, b, hk, live ? key : 0);
    const uint16_t* v = row_of(a.v, a.vs, b, hk, live ? key : 0);
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      kf[t] = live ? *reinterpret_cast<const u32x4*>(k + 16 * t + 8 * h) : u32x4{0u, 0u, 0u, 0u};
      const u32x4 x = live ? *reinterpret_cast<const u32x4*>(v + 16 * t + 8 * h) : u32x4{0u, 0u, 0u, 0u};
      if (t < kHeld) vf[t] = x;
      else s_v[t - kHeld][tid] = x;
    }
  }
  f32x16 dk[T::kOut], dv[T::kOut];
#pragma unroll
  for (int o = 0; o < T::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[o][r] = dv[o][r] = 0.f;

  constexpr bool kFit = DT == WX_F16;
  // dk holds its sums times 2^kUp and, for each key, s_slope's power of two, dv times 2^kUp.  (In LDS, for want of registers.)
  if constexpr (kFit) s_slope[wave][lane & 31] = 1.f;
  bool scaled = false;  // one of them is not 1
  const int rows_first = rows_base<D>(lane), cols_first = cols_base<D>(lane);
  auto turn = [&](int t, unsigned char* tq, unsigned char* next) {
    wait_loads();
    attn_barrier();
    if (t + 2 < last) fetch(t + 2, next);
    if (t >= last) return;
    const unsigned char* tg = tq + kTileBytes;
    const float* info = reinterpret_cast<const float*>(tq + 2 * kTileBytes);
    const int4 full = *reinterpret_cast<const int4*>(info + 128);
    const int f_lo = __builtin_amdgcn_readfirstlane(full.x), f_hi = __builtin_amdgcn_readfirstlane(full.y), one = __builtin_amdgcn_readfirstlane(full.z);
    const bool large = kFit && __builtin_amdgcn_readfirstlane(full.w) < kUp<DT>;
    // (an exclusive-or per read in place of an address register for each: the accumulators leave none)
    int rows_at = rows_first, cols_at = cols_first;
    asm volatile("" : "+v"(rows_at), "+v"(cols_at));
    // A product's operand is asked for kAhead products before it; the second half's powers are found under the first half's products.
    constexpr int kAhead = 2, kScores = 2 * T::kSteps, kProducts = 4 * T::kOut;
    auto read_s = [&](int i) { return read_rows<D>(i % 2 == 0 ? tq : tg, 0, i / 2, rows_at); };
    auto read_g = [&](int i) { return read_cols<D>(i % 2 == 0 ? tg : tq, 0, i / (2 * T::kOut), i / 2 % T::kOut, cols_at); };
    f32x16 s, dp;
    u32x4 f[kAhead], w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_s(i);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
    in_order();
#pragma unroll
    for (int i = 0; i < kScores; ++i) {
      if (i % 2 == 0) s = mfma<DT>(f[i % kAhead], kf[i / 2], s);
      else dp = mfma<DT>(f[i % kAhead], i / 2 < kHeld ? vf[i / 2 < kHeld ? i / 2 : 0] : w, dp);
      if (i + kAhead < kScores) f[i % kAhead] = read_s(i + kAhead);
      if (i % 2 == 1 && i / 2 + 1 >= kHeld && i / 2 + 1 < T::kSteps) w = s_v[i / 2 + 1 - kHeld][tid];
      in_order();
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_g(i);
    in_order();
    if (wk < f_lo || wk + 32 > f_hi) {  // some row does not see all of the keys
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int4 lo = *reinterpret_cast<const int4*>(info + 64 + 8 * g + 4 * h), hi = *reinterpret_cast<const int4*>(info + 96 + 8 * g + 4 * h);
        const int l4[4] = {lo.x, lo.y, lo.z, lo.w}, h4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g + i] = ((key >= l4[i]) & (key < h4[i])) ? s[4 * g + i] : -kInf;
      }
    }
    if (one != 0) {  // some row sees one key: its slope is none
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 8 * (r / 4) + 4 * h + r % 4;
        const int keys = __float_as_int(info[96 + at]) - __float_as_int(info[64 + at]);
        const float delta = info[32 + at];
        dp[r] = keys == 1 ? delta : dp[r];
        in_order();
      }
    }
    auto slope = [&](int g) {  // P and dS of registers 4 g .. + 3
      const float4 lse = *reinterpret_cast<const float4*>(info + 8 * g + 4 * h), delta = *reinterpret_cast<const float4*>(info + 32 + 8 * g + 4 * h);
      const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, de[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -ls[i]));
        dp[r] = s[r] * (dp[r] - de[i]);
      }
    };
    auto fit = [&](int from) {  // as in the first kernel, of this lane's key
      if (!scaled && !large) return;
      in_order();
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) top = fmaxf(top, fabsf(dp[from + r]));
      in_order();
      int at = lane;
      asm volatile("" : "+v"(at));
      float of = s_slope[wave][at & 31];
      top *= of;
      if (__any(top > kMostSlope && top < kInf)) {
        const float f = ldexpf(1.f, -slopes_less(top));
        of *= f;
        s_slope[wave][at & 31] = of;
        scaled = true;
#pragma unroll
        for (int o = 0; o < T::kOut; ++o)
#pragma unroll
          for (int r = 0; r < 16; ++r) dk[o][r] *= f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) dp[from + r] *= of;
      in_order();
    };
    slope(0);
    slope(1);
    if constexpr (kFit) fit(0);
    u32x4 p = pack_step<DT>(s, 0), ds = pack_step<DT>(dp, 0);
    in_order();
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int o = i / 2 % T::kOut;
      if (i == 2 * T::kOut) {
        if constexpr (kFit) fit(8);
        p = pack_step<DT>(s, 1), ds = pack_step<DT>(dp, 1);
      }
      if (i % 2 == 0) dv[o] = mfma<DT>(f[i % kAhead], p, dv[o]);
      else dk[o] = mfma<DT>(f[i % kAhead], ds, dk[o]);
      if (i + kAhead < kProducts) f[i % kAhead] = read_g(i + kAhead);
      if (i == 0) slope(2);
      if (i == T::kOut) slope(3);
      in_order();
    }
  };
  for (int t = first; t < last; t += 4) {
    turn(t + rg, mine, other);
    if (t + 2 < last) turn(t + 2 + rg, other, mine);
  }

  if constexpr (kFit) {
    const float fv = ldexpf(1.f, -kUp<DT>), fk = fv / s_slope[wave][lane & 31];
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[o][r] *= fk, dv[o][r] *= fv;
  }
  // The two row groups' sums: the first gets the others' dK and finishes it, the second dV.
  __syncthreads();
  {
    float* give = reinterpret_cast<float*>(rg == 0 ? lds1 : lds0) + half * (kSums / 4) + lane;
    const float* take = reinterpret_cast<const float*>(rg == 0 ? lds0 : lds1) + half * (kSums / 4) + lane;
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) give[(16 * o + r) * 64] = rg == 0 ? dv[o][r] : dk[o][r];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[o][r] = (rg == 0 ? dk[o][r] : dv[o][r]) + take[(16 * o + r) * 64];  // (from here on: what this group finishes)
  }
  const float scale = rg == 0 ? a.scale : 1.f;
  uint16_t* const grad = rg == 0 ? a.dk : a.dv;
  // (of this unit's first key)
  float* const part = a.part + (static_cast<int64_t>(pair) * a.units + todo.w) * (kKeyTile * 2 * D) + rg * D;
  uint32_t again = columns(live && not_numbers<D>(dk));
  if (whole) {
    store_row<DT, D>(dk, scale, live ? grad + ((static_cast<int64_t>(b) * a.n_keys + key) * a.n_kv + hk) * D : nullptr, lane);
  } else if (live) {
#pragma unroll
    for (int o = 0; o < T::kOut; ++o) store_sums<D>(dk[o], o, part + (key - k0) * 2 * D, lane);
  }

  if (again != 0) dkv_again<DT, D>(a, again, todo, kFit && rg == 0 ? fminf(s_slope[half][lane & 31], s_slope[half + 2][lane & 31]) : 1.f);
}

// dK and dV of the keys of a tile of several units, from the units' sums: four workgroups per tile, a thread per 4 channels (one
// workgroup took 13 us for 316 tiles of 6 units and head size 64, four take 7).
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(BwdArgs a) {
  const int at = blockIdx.x >> 2, pair = a.by_tiles.div(at), tile = at - pair * a.key_tiles;
  const int2 of_tile = a.tiles[static_cast<int64_t>(pair) * a.key_tiles + tile];
  if (of_tile.x <= 1) return;
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const float* part = a.part + (static_cast<int64_t>(pair) * a.units + of_tile.y) * (kKeyTile * 2 * D);
  constexpr int kMine = kKeyTile * (2 * D / 4) / 4;
  for (int i = (blockIdx.x & 3) * kMine + threadIdx.x; i < ((blockIdx.x & 3) + 1) * kMine; i += 256) {
    const int key = tile * kKeyTile + i / (2 * D / 4), e = i % (2 * D / 4) * 4;
    if (key >= a.n_keys) break;
    const float* src = part + i * 4;
    float4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int u = 0; u < of_tile.x; ++u) {
      const float4 x = *reinterpret_cast<const float4*>(src + u * (kKeyTile * 2 * D));
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    const float f = e < D ? a.scale : 1.f;
    uint16_t* dst = (e < D ? a.dk + e : a.dv + e - D) + ((static_cast<int64_t>(b) * a.n_keys + key) * a.n_kv + hk) * D;
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<DT>(s.x * f, s.y * f), pack2<DT>(s.z * f, s.w * f)};
  }
}

struct Workspace {
  size_t info, bounds, tiles, list, part, total;
};
Workspace layout(int64_t pairs, int64_t rows, int64_t n_keys, int head_dim) {
  const size_t blocks = static_cast<size_t>(pairs) * ((rows + 31) / 32), tiles = static_cast<size_t>(pairs) * ((n_keys + kKeyTile - 1) / kKeyTile);
  const size_t more = static_cast<size_t>(pairs) * more_units(pairs, rows, n_keys, device_cu_count());
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  Workspace w{};
  w.info = 0;
  w.bounds = up(blocks * kInfoWords * 4);
  w.tiles = w.bounds + up(blocks * sizeof(int2));
  w.list = w.tiles + up(tiles * sizeof(int2));
  w.part = w.list + up((tiles + more) * sizeof(int4));
  w.total = w.part + (more > 0 ? (tiles + more) * kKeyTile * 2 * head_dim * sizeof(float) : 0);
  return w;
}

template <int DT, int D>
int launch_bwd(BwdArgs& a, hipStream_t s) {
  const int64_t pairs = static_cast<int64_t>(a.batch) * a.n_kv;
  // Rows that fill 128-row workgroups two to a CU take those, fewer take 64-row ones, whose wavefronts share the keys.  Forward and backward
  // with 64 / 128: 5003 packed tokens 123 / 133 us, 4096 causal tokens of 8 heads 256 / 281 (472 and 256 large workgroups); 16 x 912 tokens
  // 410 / 376, 4096 tokens of 16 heads that see all 629 / 610 (1824 and 512).
  const int row_waves = pairs * ((a.row_blocks + 3) / 4) < 2 * device_cu_count() ? 2 : 4;
  const int64_t row_tiles = pairs * ((a.row_blocks + row_waves - 1) / row_waves), units = pairs * a.units;
  if (too_many_blocks(row_tiles, 256) || (a.key_tiles > 0 && (too_many_blocks(units, 256) || too_many_blocks(pairs, 1024))))
    return fail(WX_ERR_UNSUPPORTED, "wx_attention_bwd: too many rows or keys");
  const int all = static_cast<int>(pairs);
  a.by_kv = Divider(a.n_kv), a.by_group = Divider(a.group), a.by_in_group = Divider(a.group < 32 ? a.group : 32);
  a.by_pairs = Divider(all % 8 == 0 ? all / 8 : all), a.by_tiles = Divider(a.key_tiles > 0 ? a.key_tiles : 1);
  const dim3 block(256);
  if (row_tiles > 0) {
    a.spread = Spread(all, (a.row_blocks + row_waves - 1) / row_waves);
    if (row_waves == 2) hipLaunchKernelGGL((attn_dq_kernel<DT, D, 2>), dim3(static_cast<unsigned>(row_tiles)), block, 0, s, a);
    else hipLaunchKernelGGL((attn_dq_kernel<DT, D, 4>), dim3(static_cast<unsigned>(row_tiles)), block, 0, s, a);
    if (int rc = check_launch("attn_dq_kernel")) return rc;
  }
  if (a.key_tiles > 0) {
    hipLaunchKernelGGL(attn_plan_kernel, dim3(static_cast<unsigned>(pairs)), dim3(1024), 0, s, a);
    if (int rc = check_launch("attn_plan_kernel")) return rc;
    hipLaunchKernelGGL((attn_dkv_kernel<DT, D>), dim3(static_cast<unsigned>(units)), block, 0, s, a);
    if (int rc = check_launch("attn_dkv_kernel")) return rc;
  }
  if (a.more > 0) {
    hipLaunchKernelGGL((attn_dkv_join_kernel<DT, D>), dim3(static_cast<unsigned>(pairs * a.key_tiles * 4)), block, 0, s, a);
    return check_launch("attn_dkv_join_kernel");
  }
  return WX_OK;
}

}  // namespace
}  // namespace wx

using namespace wx;

extern "C" size_t wx_attention_bwd_workspace_bytes(int64_t batch, int n_q_heads, int n_kv_heads, int64_t n_queries, int64_t n_keys,
                                                   int head_dim) {
  if (batch <= 0 || n_q_heads < 0 || n_kv_heads <= 0 || n_queries < 0 || n_keys < 0 || head_dim <= 0) return 0;
  return layout(batch * n_kv_heads, n_queries * (n_q_heads / n_kv_heads), n_keys, head_dim).total;
}

extern "C" int wx_attention_bwd(const void* q, const void* k, const void* v, const void* out, const float* lse, const void* rest,
                                const void* grad_out, void* grad_q, void* grad_k, void* grad_v, const int32_t* key_ranges, const int32_t* key_lengths,
                                int causal, int64_t batch, int n_q_heads, int n_kv_heads, int64_t n_queries, int64_t n_keys,
                                int head_dim, const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                                const int64_t grad_strides[3], float scale, int dtype, void* workspace, size_t workspace_bytes,
                                wx_stream_t stream) {
  const char* who = "wx_attention_bwd";
  if (int rc = attention_check(who, batch, n_q_heads, n_kv_heads, n_queries, n_keys, head_dim, dtype, scale)) return rc;
  if (!q_strides || !k_strides || !v_strides || !grad_strides) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null strides", who);
  if (batch == 0 || n_kv_heads == 0) return WX_OK;
  const int group = std::max(n_q_heads / n_kv_heads, 1);
  const int64_t rows = n_queries * (n_q_heads / n_kv_heads);  // (none without query heads: the keys' gradients are zeros then, as without queries)
  if ((rows > 0 && (!q || !out || !lse || !grad_out || !grad_q)) || (n_keys > 0 && (!k || !v || !grad_k || !grad_v)))
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  for (const void* p : {q, k, v, out, rest, grad_out, static_cast<const void*>(grad_q), static_cast<const void*>(grad_k), static_cast<const void*>(grad_v),
                        static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(key_ranges) & 7) return fail(WX_ERR_INVALID_ARGUMENT, "%s: key_ranges must be 8-byte aligned", who);
  if (int rc = attention_check_strides(who, "q", q_strides, 2, 34, group)) return rc;
  if (int rc = attention_check_strides(who, "k", k_strides, 2, 64, 1)) return rc;
  if (int rc = attention_check_strides(who, "v", v_strides, 2, 64, 1)) return rc;
  if (int rc = attention_check_strides(who, "grad_out", grad_strides, 2, 34, group)) return rc;
  BwdArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v), a.g = static_cast<const uint16_t*>(grad_out);
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.ks[i] = k_strides[i], a.vs[i] = v_strides[i], a.gs[i] = grad_strides[i];
  a.out = static_cast<const uint16_t*>(out), a.rest = static_cast<const uint8_t*>(rest), a.lse = lse;
  a.dq = static_cast<uint16_t*>(grad_q), a.dk = static_cast<uint16_t*>(grad_k), a.dv = static_cast<uint16_t*>(grad_v);
  a.mask = {reinterpret_cast<const int2*>(key_ranges), key_lengths, causal};
  a.batch = static_cast<int>(batch), a.n_q = n_q_heads, a.n_kv = n_kv_heads, a.n_queries = static_cast<int>(n_queries), a.n_keys = static_cast<int>(n_keys);
  a.group = group, a.rows = static_cast<int>(rows), a.row_blocks = (a.rows + 31) / 32;
  a.c = scale * kLog2e, a.scale = scale;
  const int64_t pairs = batch * n_kv_heads;
  a.key_tiles = (a.n_keys + kKeyTile - 1) / kKeyTile;
  a.aim = aim_units(pairs, n_keys, device_cu_count()), a.more = more_units(pairs, a.rows, n_keys, device_cu_count());
  a.units = a.key_tiles + a.more;
  const Workspace w = layout(pairs, a.rows, n_keys, head_dim);
  if (w.total > 0 && (!workspace || workspace_bytes < w.total)) return fail(WX_ERR_WORKSPACE, "%s: workspace too small (see wx_attention_bwd_workspace_bytes)", who);
  char* ws = static_cast<char*>(workspace);
  a.info = reinterpret_cast<uint32_t*>(ws + w.info), a.bounds = reinterpret_cast<int2*>(ws + w.bounds), a.tiles = reinterpret_cast<int2*>(ws + w.tiles), a.list = reinterpret_cast<int4*>(ws + w.list);
  a.part = reinterpret_cast<float*>(ws + w.part);
  hipStream_t s = as_stream(stream);
  if (dtype == WX_BF16) {
    if (head_dim == 64) return launch_bwd<WX_BF16, 64>(a, s);
    if (head_dim == 80) return launch_bwd<WX_BF16, 80>(a, s);
    return launch_bwd<WX_BF16, 128>(a, s);
  }
  if (head_dim == 64) return launch_bwd<WX_F16, 64>(a, s);
  if (head_dim == 80) return launch_bwd<WX_F16, 80>(a, s);
  return launch_bwd<WX_F16, 128>(a, s);
}
