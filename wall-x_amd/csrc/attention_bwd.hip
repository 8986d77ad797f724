// Attention backward (gfx950): with P = exp2(c S - L) recomputed from the scores and the forward's base-2 log-sum-exp L,
//   delta = rowsum(dO O),  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two kernels, seven matrix products in place of the five that share one pass: the first walks the keys of a tile of rows (dQ),
// the second the rows of a tile of keys (dK, dV, all heads of the group in turn).  Every sum is then one wavefront's own, in a
// fixed order: no atomics, the same gradients every time.
//
// 16 rows of 912 causal tokens of 16 / 2 heads of 128 (72 GFLOP in three products, 96 in four): dQ 124 us, 0.58 PFLOP/s, matrix units busy
// 31 % (the rows' four operands are on their way for a third of it); the plan 5; dK and dV 153 us, 0.63 PFLOP/s, 40 %, reading 0.6 GB of
// which half is in L2; the join 15.  5003 packed tokens of 12 / 4 heads of 64: 29, 8, 39 and 7 us.
#include <algorithm>

#include "attention.h"

namespace wx {

int attention_check(const char* who, int64_t batch, int n_q, int n_kv, int64_t n_queries, int64_t n_keys, int head_dim, int dtype, float scale);
int attention_check_strides(const char* who, const char* name, const int64_t* st, int elem_bytes, int64_t span, int64_t heads);

namespace {

struct BwdArgs {
  const uint16_t *q, *k, *v, *g;  // g = dO
  int64_t qs[3], ks[3], vs[3], gs[3];
  const uint16_t* out;            // [batch, n_queries, n_q, D]
  const uint8_t* rest;            // like out: what its rounding left (rest_of), or null
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
// sees a single one, and (fp16) the power of two that the slopes of all its rows fit fp16 with.
constexpr int kInfoWords = 4 * 32 + 4;

// fp16's range is too short for probabilities of many keys and for their slopes: P is 1 / keys, dS as much smaller again as the gradient
// that comes in, and beyond 65504 where few keys meet a large one.  P enters its product times 2^15, which it cannot leave the range with.  dS of
// a row is formed times 2^15 as well (both are one subtraction from L), until a slope passes 2^15 (kMostSlope): then by as much less as
// takes the largest to below 2^10, and the sums so far with it.  The second kernel, whose products sum over rows, takes the least of the
// powers of the rows that it has met.  Powers of two are exact, and taken back from the sums.  Forward and backward of 16 x 912 tokens in fp16
// 378 us, 368 with P and dS as they are; dQ's error for gradients of 0.001 over 8192 keys 0.096 % of its length (0.094 of it the result's own
// rounding), 0.76 with them.
template <int DT>
constexpr int kUp = DT == WX_F16 ? 15 : 0;
constexpr float kMostSlope = 32768.f;
constexpr int kSlopeTo = 9;

constexpr int kKeyTile = 64;

__device__ __forceinline__ const uint16_t* row_of(const uint16_t* p, const int64_t* st, int b, int h, int i) {
  return p + b * st[0] + h * st[1] + i * st[2];
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
  rests = both_sum(rests);
  // (a rest that e5m2 does not hold, of outputs of 10^7 and more, is left out)
  const float delta = some ? both_sum(sums[0] + sums[1]) + (fabsf(rests) < kInf ? rests : 0.f) : 0.f;
  lse = some ? lse : kInf;
  constexpr bool kFit = DT == WX_F16;
  int up = kUp<DT>;  // this row's slopes are formed times 2^up
  float shifted = lse - kUp<DT>;
  const int block = tile * RW + rw, one = __any(hi - lo == 1);
  if (kw == 0 && block < a.row_blocks) {
    const int64_t at = static_cast<int64_t>(pair) * a.row_blocks + block;
    uint32_t* info = a.info + at * kInfoWords;
    info[(h ? 64 : 0) + (lane & 31)] = h ? static_cast<uint32_t>(lo) : __float_as_uint(shifted);
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
    top = both_max(top);
    const int less = top > kMostSlope && top < kInf ? static_cast<int>(__float_as_uint(top) >> 23) - 127 - kSlopeTo : 0;
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

  bool bad = false;
#pragma unroll
  for (int o = 0; o < T::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (32 * o + 8 * (r / 4) < D) bad = bad || acc[o][r] != acc[o][r];
  if (!some) {
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[o][r] = 0.f;
  }
  // (a row of one key has no slope: its sum is what rounding left of dP - delta)
  store_row<DT, D>(acc, hi - lo == 1 ? 0.f : a.scale * ldexpf(1.f, -kUp<DT>), live ? a.dq + ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D : nullptr, lane);
  // Rows whose sum is not a number, in plain loops over the keys that they see: 0 * inf may have come from one that they do not.
  uint64_t redo = __ballot(bad && some);
  redo = (redo | redo >> 32) & 0xffffffffull;
  while (redo != 0) {
    const int r = __builtin_ctzll(redo);
    redo &= redo - 1;
    const int row_r = __shfl(row, r), lo_r = __shfl(lo, r), hi_r = __shfl(hi, r);
    const float lse_r = __shfl(lse, r), delta_r = __shfl(delta, r);
    const int i_r = row_r / a.group, hq_r = hk * a.group + row_r % a.group;
    const uint16_t *q = row_of(a.q, a.qs, b, hq_r, i_r), *g = row_of(a.g, a.gs, b, hq_r, i_r);
    float sum[2] = {0.f, 0.f};
    for (int first = lo_r; first < hi_r; first += 64) {
      const int key = first + lane;
      float ds = 0.f;
      if (key < hi_r) {
        const uint16_t *kr = row_of(a.k, a.ks, b, hk, key), *vr = row_of(a.v, a.vs, b, hk, key);
        float s = 0.f, dp = 0.f;
        for (int d = 0; d < D; ++d) {
          s = __builtin_fmaf(Elem<DT>::load(q[d]), Elem<DT>::load(kr[d]), s);
          dp = __builtin_fmaf(Elem<DT>::load(g[d]), Elem<DT>::load(vr[d]), dp);
        }
        ds = exp2f(s * a.c - lse_r) * (dp - delta_r);
      }
      const int n = min(64, hi_r - first);
      for (int j = 0; j < n; ++j) {
        const float x = __shfl(ds, j);
        const uint16_t* kr = row_of(a.k, a.ks, b, hk, first + j);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (lane + 64 * u < D) sum[u] = __builtin_fmaf(x, Elem<DT>::load(kr[lane + 64 * u]), sum[u]);
      }
    }
    uint16_t* dst = a.dq + ((static_cast<int64_t>(b) * a.n_queries + i_r) * a.n_q + hq_r) * D;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 64 * u < D) dst[lane + 64 * u] = static_cast<uint16_t>(Elem<DT>::store(sum[u] * (hi_r - lo_r == 1 ? 0.f : a.scale)));
  }
}

// What the workgroups of the next kernel do: a workgroup per pair, a lane per key tile, the row blocks dealt to 16 wavefronts.
//
// Under a causal mask the first keys are seen by all rows and the last by few, and of a row of packed sequences a tile is seen by those
// of its own: a tile's row blocks, from the first to the last that sees it, are cut evenly into units of at most as many as make a pair's
// units about `aim` in all (kLeast where that is fewer), so that the longest workgroup is a unit and not a tile.
constexpr int kLeast = 16;
constexpr int kPlanTiles = 1024;
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
  int work = 0;
  for (int t = lane; t < a.key_tiles; t += 64) work += max(s_last[t] - s_first[t] + 1, 0);
#pragma unroll
  for (int n = 1; n < 64; n *= 2) work += __shfl_xor(work, n);
  const int unit = max(kLeast, (work + a.aim - 1) / a.aim);
  int next = 0;  // (never past a.units: the full units are no more than a.aim, the last ones of the tiles no more than those; and see more_units)
  for (int c = 0; c < a.key_tiles; c += 64) {
    const bool is = c + lane < a.key_tiles;
    const int from = is ? s_first[c + lane] : 0, blocks = is ? max(s_last[c + lane] - from + 1, 0) : 0;
    const int units = is ? max((blocks + unit - 1) / unit, 1) : 0;  // (a tile that nothing sees: one of no blocks, which writes zeros)
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
  // (D = 128: two of V's operands stand in LDS, read in front of their products; with all in registers one was spilled, and the wait
  // for its memory was a wait for the next block's as well)
  constexpr int kHeld = D == 128 ? T::kSteps - 2 : T::kSteps;
  __shared__ u32x4 s_v[kHeld < T::kSteps ? T::kSteps - kHeld : 1][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int half = wave & 1, rg = wave >> 1;
  const int pairs = a.batch * a.n_kv;
  // (the pair varies fastest: dealt to the XCDs by their unit, a tile's first units all went to a few)
  int pair;
  int4 todo;
  {
    const int id = blockIdx.x, from = pairs % 8 == 0 ? id >> 3 : id, per = pairs % 8 == 0 ? pairs >> 3 : pairs;
    const int unit = a.by_pairs.div(from);
    pair = pairs % 8 == 0 ? (id & 7) * per + (from - unit * per) : from - unit * per;
    todo = a.list[static_cast<int64_t>(pair) * a.units + unit];
  }
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
  int up = kUp<DT>;         // dk holds its sums times 2^up, dv times 2^kUp
  float of_slope = 1.f;     // 2^(up - kUp)
  const int rows_first = rows_base<D>(lane), cols_first = cols_base<D>(lane);
  auto turn = [&](int t, unsigned char* tq, unsigned char* next) {
    wait_loads();
    attn_barrier();
    if (t + 2 < last) fetch(t + 2, next);
    if (t >= last) return;
    const unsigned char* tg = tq + kTileBytes;
    const float* info = reinterpret_cast<const float*>(tq + 2 * kTileBytes);
    const int4 full = *reinterpret_cast<const int4*>(info + 128);
    const int f_lo = __builtin_amdgcn_readfirstlane(full.x), f_hi = __builtin_amdgcn_readfirstlane(full.y);
    if constexpr (kFit) {
      const int here = __builtin_amdgcn_readfirstlane(full.w);
      if (here < up) {
        const float f = ldexpf(1.f, here - up);
        up = here;
        of_slope = ldexpf(1.f, up - kUp<DT>);
#pragma unroll
        for (int o = 0; o < T::kOut; ++o)
#pragma unroll
          for (int r = 0; r < 16; ++r) dk[o][r] *= f;
      }
    }
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
    if (__builtin_amdgcn_readfirstlane(full.z) != 0) {  // some row sees one key: its slope is none
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
        if constexpr (kFit) dp[r] *= of_slope;
      }
    };
    slope(0);
    slope(1);
    u32x4 p = pack_step<DT>(s, 0), ds = pack_step<DT>(dp, 0);
    in_order();
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int o = i / 2 % T::kOut;
      if (i == 2 * T::kOut) p = pack_step<DT>(s, 1), ds = pack_step<DT>(dp, 1);
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
    const float fk = ldexpf(1.f, -up), fv = ldexpf(1.f, -kUp<DT>);
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
  bool bad = false;
#pragma unroll
  for (int o = 0; o < T::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (32 * o + 8 * (r / 4) < D) bad = bad || dk[o][r] != dk[o][r];
  const float scale = rg == 0 ? a.scale : 1.f;
  uint16_t* const grad = rg == 0 ? a.dk : a.dv;
  // (of this unit's first key)
  float* const part = a.part + (static_cast<int64_t>(pair) * a.units + todo.w) * (kKeyTile * 2 * D) + rg * D;
  if (whole) {
    store_row<DT, D>(dk, scale, live ? grad + ((static_cast<int64_t>(b) * a.n_keys + key) * a.n_kv + hk) * D : nullptr, lane);
  } else if (live) {
    float* dst = part + (key - k0) * 2 * D;
#pragma unroll
    for (int o = 0; o < T::kOut; ++o)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * o + 8 * g < D) *reinterpret_cast<float4*>(dst + 32 * o + 8 * g + 4 * h) = float4{dk[o][4 * g], dk[o][4 * g + 1], dk[o][4 * g + 2], dk[o][4 * g + 3]};
  }
  // Keys whose sums are not numbers, in plain loops over the rows that see them.
  uint64_t redo = __ballot(bad && live);
  redo = (redo | redo >> 32) & 0xffffffffull;
  while (redo != 0) {
    const int r = __builtin_ctzll(redo);
    redo &= redo - 1;
    const int key_r = wk + r;
    const uint16_t *kr = row_of(a.k, a.ks, b, hk, key_r), *vr = row_of(a.v, a.vs, b, hk, key_r);
    float sum[2] = {0.f, 0.f};
    for (int t = first * 32; t < min(last * 32, a.rows); t += 64) {
      const int row = t + lane;
      float x = 0.f;  // the row's P, or its dS
      bool see = false;
      if (row < a.rows && row < last * 32) {
        const uint32_t* info = info_base + static_cast<int64_t>(row / 32) * kInfoWords + row % 32;
        see = key_r >= static_cast<int>(info[64]) && key_r < static_cast<int>(info[96]);
        if (see) {
          const int hq = hk * a.group + row % a.group;
          const uint16_t *q = row_of(a.q, a.qs, b, hq, row / a.group), *g = row_of(a.g, a.gs, b, hq, row / a.group);
          float s = 0.f, d = 0.f;
          for (int e = 0; e < D; ++e) {
            s = __builtin_fmaf(Elem<DT>::load(q[e]), Elem<DT>::load(kr[e]), s);
            d = __builtin_fmaf(Elem<DT>::load(g[e]), Elem<DT>::load(vr[e]), d);
          }
          x = exp2f(s * a.c - (__uint_as_float(info[0]) + kUp<DT>));
          if (rg == 0) x *= (info[96] - info[64] == 1 ? __uint_as_float(info[32]) : d) - __uint_as_float(info[32]);
        }
      }
      uint64_t seen = __ballot(see);
      while (seen != 0) {
        const int j = __builtin_ctzll(seen);
        seen &= seen - 1;
        const float xj = __shfl(x, j);
        const int hq = hk * a.group + (t + j) % a.group;
        const uint16_t* w = rg == 0 ? row_of(a.q, a.qs, b, hq, (t + j) / a.group) : row_of(a.g, a.gs, b, hq, (t + j) / a.group);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (lane + 64 * u < D) sum[u] = __builtin_fmaf(xj, Elem<DT>::load(w[lane + 64 * u]), sum[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 64 * u < D) {
        if (whole) grad[((static_cast<int64_t>(b) * a.n_keys + key_r) * a.n_kv + hk) * D + lane + 64 * u] = static_cast<uint16_t>(Elem<DT>::store(sum[u] * scale));
        else part[(key_r - k0) * 2 * D + lane + 64 * u] = sum[u];
      }
  }
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

// Units that a pair's key tiles are cut into beyond one to each: about kUnits workgroups to each place on the chip (two to a CU) of all
// pairs', where the tiles alone are fewer.  More units end more evenly, fewer write and join fewer sums (64 KB a unit of head size 128).
// Forward and backward with 1 / 2 / 3 / 4 / 6: 8192 causal tokens of 16 / 2 heads 1464 / 1344 / 1321 / 1339 / 1372 us, 4096 tokens of 16 / 16
// heads that see all 593 / 594 / 643 / 648 / 672, 16 rows of 912 causal tokens 379 / 384 / 404 / 413 / 442.
constexpr int kUnits = 2;
int aim_units(int64_t pairs, int64_t n_keys) {
  const int64_t tiles = pairs * ((n_keys + kKeyTile - 1) / kKeyTile), places = 2 * device_cu_count();
  return tiles == 0 || tiles >= kUnits * places || tiles > pairs * kPlanTiles ? 0 : static_cast<int>((kUnits * places + pairs - 1) / pairs);
}
// No tile makes more than its rows' blocks do in units of the least length.
int more_units(int64_t pairs, int64_t rows, int64_t n_keys) {
  const int64_t of_tile = ((rows + 31) / 32 + kLeast - 1) / kLeast, most = (n_keys + kKeyTile - 1) / kKeyTile * std::max<int64_t>(of_tile - 1, 0);
  return static_cast<int>(std::min<int64_t>(aim_units(pairs, n_keys), most));
}

struct Workspace {
  size_t info, bounds, tiles, list, part, total;
};
Workspace layout(int64_t pairs, int64_t rows, int64_t n_keys, int head_dim) {
  const size_t blocks = static_cast<size_t>(pairs) * ((rows + 31) / 32), tiles = static_cast<size_t>(pairs) * ((n_keys + kKeyTile - 1) / kKeyTile);
  const size_t more = static_cast<size_t>(pairs) * more_units(pairs, rows, n_keys);
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
  if (row_tiles > 0x7fffffffll || units > 0x7fffffffll) return fail(WX_ERR_UNSUPPORTED, "wx_attention_bwd: too many rows");
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
  if (batch <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_queries < 0 || n_keys < 0 || head_dim <= 0) return 0;
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
  if (batch == 0 || n_q_heads == 0) return WX_OK;
  const int group = n_q_heads / n_kv_heads;
  if ((n_queries > 0 && (!q || !out || !lse || !grad_out || !grad_q)) || (n_keys > 0 && (!k || !v || !grad_k || !grad_v)))
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
  a.group = group, a.rows = static_cast<int>(n_queries) * group, a.row_blocks = (a.rows + 31) / 32;
  a.c = scale * kLog2e, a.scale = scale;
  const int64_t pairs = batch * n_kv_heads;
  a.key_tiles = (a.n_keys + kKeyTile - 1) / kKeyTile;
  a.aim = aim_units(pairs, n_keys), a.more = more_units(pairs, a.rows, n_keys);
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
