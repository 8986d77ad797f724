// Attention forward: O = softmax(scale Q K^T over the keys of each query's range) V, one pass over the keys with a running
// maximum and sum, for keys and values in the queries' type or quantised to e4m3 with a scale per token (gfx950).
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace wx {
namespace {

struct FwdArgs {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];   // strides in elements: batch, head, position
  const float *k_scale, *v_scale;  // e4m3: [batch, n_kv, n_keys]
  uint16_t* out;                 // [batch, n_queries, n_q, D]
  float* lse;                    // [batch, n_kv, n_queries * group], base 2, or null
  uint8_t* rest;                 // with lse: what out's rounding left times kRestUp, like out, or null
  AttnMask mask;
  int batch, n_q, n_kv, n_queries, n_keys, group;
  int rows, row_tiles, splits;
  Divider by_splits, by_kv, by_group, by_rows;
  Spread spread;
  float c;                       // scale * log2(e)
  float* part;                   // splits > 1: [pair, split, rows, D] sums, then [pair, split, rows] (maximum, sum)
};

__device__ __forceinline__ float2* part_stats(const FwdArgs& a, int d) {
  return reinterpret_cast<float2*>(a.part + static_cast<int64_t>(a.batch) * a.n_kv * a.splits * a.rows * d);
}

// two e4m3 values, times a power of two, to two of the compute type (exact for a power of 1)
template <int DT, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t x, float power = 1.0f) {
  if constexpr (DT == WX_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, power, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, power, HI));
}

// fp16's range is too short for a probability times its key's scale: of values of 0.01 the scales are about 2^-13, and most of the products
// would be below 2^-24.  So a value's code takes the power of two of its scale as it is widened (no instruction more) and the probability
// the rest, between 1 and 2.  What a value loses there, 2^-25 if it is below 2^-14, is half a step of such a result.  Scales above 2^7, whose
// largest code would be beyond fp16, leave what is above it with the probability; should that be beyond fp16 too, the sum is not finite
// and the row is done again.  64 x 32 queries over 800 to 912 cached keys: 37 us, 36 with the scale at the probability alone (whose error is 2.5 %
// of the result for values of 0.001, against 0.03 %).
__device__ __forceinline__ uint32_t scale_power(float scale) { return min(__float_as_uint(scale) & 0x7f800000u, 134u << 23); }

// The keys of this workgroup's split.
__device__ __forceinline__ int2* split_share() {
  __shared__ int2 s;
  return &s;
}

// ---- Rows again (see Odd, attention.h), of this wavefront's those that `again` has a bit for, with the maximum and the sum that they ended
// with.  Their place is found once more: kept over the kernel's loops for this rare case it costs them registers.
template <int DT, int D, bool F8, int RW>
__device__ __forceinline__ void rows_again(const FwdArgs& a, uint32_t again, float m, float l) {
  using T = AttnTile<D>;
  constexpr int KW = RW == 8 ? 1 : 4 / RW, kElem = F8 ? 1 : 2;
  constexpr bool kPowers = F8 && DT == WX_F16;
  int id = blockIdx.x, tid = threadIdx.x;
  asm volatile("" : "+s"(id), "+v"(tid));
  const int lane = tid & 63, rw = __builtin_amdgcn_readfirstlane(tid >> 6) % RW, h = lane >> 5;
  const int rest = a.by_splits.div(id), split = id - rest * a.splits;
  int pair, tile;
  a.spread.place(rest, pair, tile);
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int row = tile * 32 * RW + rw * 32 + (lane & 31), in_row = row < a.rows ? row : 0, qi = a.by_group.div(in_row), hq = hk * a.group + in_row - qi * a.group;
  const bool redo = again >> (lane & 31) & 1;
  int lo = 0, hi = 0;
  if (redo) key_range(a.mask, b, qi, a.n_queries, a.n_keys, lo, hi);
  if constexpr (KW > 1) {
    const int2 share = *split_share();
    lo = max(lo, share.x), hi = min(hi, share.y);
  }
  const int from = wave_extreme<false>(redo ? lo : 0x7fffffff), up_to = wave_extreme<true>(hi);
  const float mc = m == -kInf ? 0.f : m * a.c;
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.qs[0] + hq * a.qs[1] + qi * a.qs[2];
  const int64_t to = ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D;
  const char* kp = static_cast<const char*>(a.k) + (b * a.ks[0] + hk * a.ks[1]) * kElem;
  const char* vp = static_cast<const char*>(a.v) + (b * a.vs[0] + hk * a.vs[1]) * kElem;
  const int64_t k_step = a.ks[2] * kElem, v_step = a.vs[2] * kElem;
  const float* ksc = F8 ? a.k_scale + (static_cast<int64_t>(b) * a.n_kv + hk) * a.n_keys : nullptr;
  const float* vsc = F8 ? a.v_scale + (static_cast<int64_t>(b) * a.n_kv + hk) * a.n_keys : nullptr;
  auto in = [&](int k0, int i) { return min(i, a.n_keys - 1 - k0); };  // (a key past the last is the last, and not seen)
  // the probabilities (times what scale their values do not carry) of keys k0 .. + 31, zeros for what is not seen and for other rows
  auto powers = [&](int k0, f32x16& s, uint32_t& seen) {
    const char* kr = kp + k0 * k_step + in(k0, lane & 31) * static_cast<int>(k_step);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) {
      u32x4 x;
      if constexpr (F8) {
        const u32x2 y = *reinterpret_cast<const u32x2*>(kr + 16 * t + 8 * h);
        x = u32x4{widen2<DT, false>(y[0]), widen2<DT, true>(y[0]), widen2<DT, false>(y[1]), widen2<DT, true>(y[1])};
      } else {
        x = *reinterpret_cast<const u32x4*>(kr + (16 * t + 8 * h) * 2);
      }
      s = mfma<DT>(x, *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h), s);
      in_order();
    }
    seen = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = 8 * (r / 4) + 4 * h + r % 4, key = k0 + i;
      const bool sees = redo && key >= lo && key < hi;
      if constexpr (F8) {
        const int at = k0 + in(k0, i);
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r] * ksc[at], a.c, -mc)) * (kPowers ? vsc[at] * __uint_as_float((254u << 23) - scale_power(vsc[at])) : vsc[at]);
      } else {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -mc));
      }
      s[r] = sees ? s[r] : 0.f;
      seen |= sees ? 1u << r : 0u;
    }
  };
  int less = 0;  // (fp16 codes) a power of two that brings the row's largest probability times scale into fp16
  if constexpr (kPowers) {
    float top = 0.f;
    for (int k0 = from; k0 < up_to; k0 += 32) {
      f32x16 s;
      uint32_t seen;
      powers(k0, s, seen);
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[r]));
    }
    top = both_max(top);
    less = top < kInf ? max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, 0) : 0;
  }
  const float f = ldexpf(1.f, -less), back = ldexpf(1.f, less);
  for (int o = 0; o < T::kOut; ++o) {
    f32x16 sum = {};
    const int c = 32 * o + (lane & 31);
    for (int k0 = from; k0 < up_to; k0 += 32) {
      f32x16 s;
      uint32_t seen, zero = 0;
      powers(k0, s, seen);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        zero |= s[r] == 0.f ? seen & 1u << r : 0u;
        if constexpr (kPowers) s[r] *= f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Odd odd;
        const u32x4 x = gather_cols<DT>(t, h, odd, [&](int i) -> uint32_t {
          if (D % 32 != 0 && c >= D) return 0;
          const char* v = vp + k0 * v_step + (in(k0, i) * static_cast<int>(v_step) + c * kElem);
          if constexpr (F8) return widen2<DT, false>(*reinterpret_cast<const uint8_t*>(v), kPowers ? __uint_as_float(scale_power(vsc[k0 + in(k0, i)])) : 1.f) & 0xffffu;
          else return *reinterpret_cast<const uint16_t*>(v);
        });
        in_order();
        sum = mfma<DT>(x, pack_step<DT>(s, t), sum);
        add_odd<DT>(sum, odd, seen, zero, t);
        in_order();
      }
    }
    if constexpr (kPowers)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[r] *= back;
    if (KW > 1 && a.splits > 1) {
      if (redo) store_sums<D>(sum, o, a.part + ((static_cast<int64_t>(pair) * a.splits + split) * a.rows + row) * D, lane);
    } else if (!F8 && a.rest != nullptr) {
      store_cols<DT, D, true>(sum, o, 1.f / l, redo ? a.out + to : nullptr, lane, redo ? a.rest + to : nullptr);
    } else {
      store_cols<DT, D>(sum, o, 1.f / l, redo ? a.out + to : nullptr, lane);
    }
  }
}

// RW of the workgroup's four wavefronts take 32 rows each; the other factor, KW = 4 / RW, shares the keys: wavefront group kw
// takes every KW-th tile of KB keys, and the groups' sums are joined in LDS at the end.
// Many rows (RW = 4): a tile of 64 keys serves 128 rows.  Fewer (RW = 2): two tiles of 32 keys at a time serve 64 rows each.  Long ones
// (RW = 8): eight wavefronts, 256 rows, in two groups half a step apart (below; plan() has the rule and what each takes).  Tiles
// are loaded one ahead, straight to LDS; e4m3 ones through registers, where they are widened to the compute type (exactly); their
// scales multiply the scores and the probabilities, a value per key.  (A form whose four wavefronts each walked tiles of their own for 32
// rows, without a barrier, was no faster for single queries: 38 against 35 us over 8 x 32768 cached keys.)
//
// What bounds it: 16384 causal tokens of 16 / 2 heads of 128 take 0.97 to 1.01 ms, 1.13 to 1.09 PFLOP/s (a large library product in the same type: 1.36
// PFLOP/s), without bank conflicts, at a clock that the power holds near 1.9 GHz.  Half a step of the two groups takes 1400 to 1800
// cycles, in which a SIMD's products need 1024, the other group's powers some 930 (one is four passes) and the tiles' way out of
// LDS, 128 KB, as long as the products.  With 128 rows, each wavefront at its own pace: 1.03 ms, matrix units busy 58 % of the time, vector
// units 56 %.  16 rows of 912 tokens: 71 to 80 us, 0.65 PFLOP/s; of a workgroup's time a quarter lies
// before its first product.  48 x 1024 patches in windows of 64, 16 heads of 80: 119 us, 4.2 TB/s.  64 x 32 queries over 800 to 912 cached
// keys: 34 us, by the vector units (46 %) and the widening's way through LDS.  Single queries of 8 sequences over 20 to 32 thousand
// cached keys: 112 MB in 28 us, 4.0 TB/s, and 4 for the join.
// (Heads of 80: 168 registers, one less than it would take, let three workgroups share a CU: 48 x 1024 patches in windows 131 us
// instead of 136, 8 x 2000 causal tokens 126 instead of 132.  The others' sums and tiles leave two.)
template <int DT, int D, bool F8, int RW>
__global__ __launch_bounds__(RW == 8 ? 512 : 256, D == 80 && !F8 && RW == 4 ? 3 : 2) void attn_fwd_kernel(FwdArgs a) {
  using T = AttnTile<D>;
  constexpr int KW = RW == 8 ? 1 : 4 / RW, KB = RW == 2 ? 32 : 64, NT = KB / 32;  // (one or two key groups)
  constexpr bool kDirect = !F8;
  constexpr int kTileBytes = KB * T::kPitch;
  constexpr int kScaleBytes = F8 ? 2 * KB * 4 : 0;
  constexpr int kSlot = 2 * kTileBytes + kScaleBytes;
  constexpr int kTiles = KW * kSlot;                                      // of one buffer
  constexpr int kJoinStats = 4 * 32 * (64 + 4) * 4, kJoin = KW > 1 ? kJoinStats + 4 * 32 * 8 : 0;  // 64 channels at a time
  constexpr int kFirst = kTiles > kJoin ? kTiles : kJoin;
  unsigned char* const lds = lds_slot<RW == 8 ? 16 : kFirst, 0>();
  unsigned char* const lds1 = lds_slot<RW == 8 ? 16 : kTiles, 1>();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kw = wave / RW, h = lane >> 5;

  int pair, tile, split;
  {
    int id = blockIdx.x;
    const int rest = a.by_splits.div(id);
    split = id - rest * a.splits;
    id = rest;
    a.spread.place(id, pair, tile);
  }
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int row = tile * 32 * RW + rw * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int in_row = live ? row : 0, qi = a.by_group.div(in_row), hq = hk * a.group + in_row - qi * a.group;

  const MaskRow row_mask = mask_row(a.mask, b, qi, a.n_queries, a.n_keys);
  in_order();
  u32x4 qf[T::kSteps];  // (asked for behind the mask and before anything that waits for it)
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.qs[0] + hq * a.qs[1] + qi * a.qs[2];
#pragma unroll
    for (int t = 0; t < T::kSteps; ++t) qf[t] = *reinterpret_cast<const u32x4*>(q + 16 * t + 8 * h);  // (a row past the last reads the first)
  }
  in_order();
  int lo = 0, hi = 0;
  if (live) key_range(a.mask, row_mask, qi, a.n_queries, a.n_keys, lo, hi);
  const bool some = hi > lo;
  int w_lo = wave_extreme<false>(some ? lo : 0x7fffffff), w_hi = wave_extreme<true>(hi);   // any row of the wavefront sees [w_lo, w_hi)
  const int f_lo = wave_extreme<true>(some ? lo : 0), f_hi = wave_extreme<false>(some ? hi : 0x7fffffff);  // every row that sees something sees [f_lo, f_hi)
  if (w_lo > w_hi) w_lo = w_hi;
  // the workgroup's keys
  __shared__ int2 bounds[RW];
  if (kw == 0 && lane == 0) bounds[rw] = int2{w_hi > w_lo ? w_lo : 0x7fffffff, w_hi};
  attn_lds_barrier();
  int g_lo = 0x7fffffff, g_hi = 0;
#pragma unroll
  for (int u = 0; u < RW; ++u) {
    g_lo = min(g_lo, bounds[u].x);
    g_hi = max(g_hi, bounds[u].y);
  }
  g_lo = __builtin_amdgcn_readfirstlane(min(g_lo, g_hi));
  g_hi = __builtin_amdgcn_readfirstlane(g_hi);
  {  // this split's share of the tiles
    const int n = (g_hi - g_lo + KB - 1) / KB;
    const int each = a.by_splits.div(n), more = n - each * a.splits;  // the first `more` splits take one more
    const int t0 = split * each + min(split, more), t1 = t0 + each + (split < more ? 1 : 0);
    g_hi = min(g_hi, g_lo + t1 * KB);
    g_lo += t0 * KB;
  }
  if (KW > 1 && tid == 0) *split_share() = int2{g_lo, g_hi};  // (behind the first of many barriers)
  const int s_lo = max(lo, g_lo), s_hi = min(hi, g_hi);
  const int tiles = __builtin_amdgcn_readfirstlane((g_hi - g_lo + KB - 1) / KB), iters = (tiles + KW - 1) / KW;

  constexpr int kElem = F8 ? 1 : 2;
  const char* kp = static_cast<const char*>(a.k) + (b * a.ks[0] + hk * a.ks[1]) * kElem;
  const char* vp = static_cast<const char*>(a.v) + (b * a.vs[0] + hk * a.vs[1]) * kElem;
  const int64_t k_step = a.ks[2] * kElem, v_step = a.vs[2] * kElem;  // (KB of them fit 31 bits: checked on the host)
  const float* ksc = F8 ? a.k_scale + (static_cast<int64_t>(b) * a.n_kv + hk) * a.n_keys : nullptr;
  const float* vsc = F8 ? a.v_scale + (static_cast<int64_t>(b) * a.n_kv + hk) * a.n_keys : nullptr;

  // ---- staging
  constexpr int kChunk = F8 ? D / 16 : D / 8;                      // 16-byte pieces of a row in memory
  constexpr int kLoaders = RW * 64;                                // threads of one key group
  constexpr int kPieces = (KB * kChunk + kLoaders - 1) / kLoaders; // per thread
  const int gt = rw * 64 + lane;
  constexpr bool kPowers = F8 && DT == WX_F16;
  u32x4 pk[kDirect ? 1 : kPieces], pv[kDirect ? 1 : kPieces];
  float pks = 0.f, pvs = 0.f, pvp[kPowers ? kPieces : 1];  // pvp: the scales of the pieces' values
  uint32_t k_off[kDirect ? T::kChunks / 4 : 1], v_off[kDirect ? T::kChunks / 4 : 1];
  if constexpr (kDirect) {
#pragma unroll
    for (int i = 0; i < T::kChunks / 4; ++i) {
      k_off[i] = stage_offset<D>(i, lane, [&](int r) { return static_cast<uint32_t>((rw * 16 + r) * static_cast<int>(k_step)); });
      v_off[i] = stage_offset<D>(i, lane, [&](int r) { return static_cast<uint32_t>((rw * 16 + r) * static_cast<int>(v_step)); });
    }
  }
  const int rows_at = rows_base<D>(lane), cols_at = cols_base<D>(lane);
  auto key0 = [&](int it) { return g_lo + (it * KW + kw) * KB; };
  auto fetch = [&](int it, unsigned char* slot) {  // a tile on its way: to LDS, or into registers
    const int k0 = key0(it), left = g_hi - k0;  // (may be <= 0: zeros)
    const int64_t at = left > 0 ? k0 : 0;
    const auto rk = attn_rsrc(kp + at * k_step, kRsrcBytes), rv = attn_rsrc(vp + at * v_step, kRsrcBytes);
    if constexpr (kDirect) {
      static_assert(RW == 8 || KB == 16 * RW, "a wavefront loads 16 rows");
      const int r0 = rw * 16;
      if (left >= KB) {  // all rows are there: the offsets stay the same from tile to tile
        stage16<D>(rk, slot + r0 * T::kPitch, k_off);
        stage16<D>(rv, slot + kTileBytes + r0 * T::kPitch, v_off);
      } else {
        stage16<D>(rk, slot + r0 * T::kPitch, lane, [&](int r) { return r0 + r < left ? static_cast<uint32_t>((r0 + r) * static_cast<int>(k_step)) : kOutside; });
        stage16<D>(rv, slot + kTileBytes + r0 * T::kPitch, lane, [&](int r) { return r0 + r < left ? static_cast<uint32_t>((r0 + r) * static_cast<int>(v_step)) : kOutside; });
      }
    } else {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int n = u * kLoaders + gt, r = n / kChunk, c = n % kChunk;
        const bool in = r < left && r < KB;
        pk[u] = __builtin_amdgcn_raw_buffer_load_b128(rk, in ? r * static_cast<int>(k_step) + c * 16 : static_cast<int>(kOutside), 0, 0);
        pv[u] = __builtin_amdgcn_raw_buffer_load_b128(rv, in ? r * static_cast<int>(v_step) + c * 16 : static_cast<int>(kOutside), 0, 0);
        if constexpr (kPowers) pvp[u] = in ? vsc[k0 + r] : 0.f;
      }
      if constexpr (F8) {
        const bool in = gt < left && gt < KB;
        pks = in ? ksc[k0 + gt] : 0.f;
        pvs = in ? vsc[k0 + gt] : 0.f;
      }
    }
  };
  auto put = [&](unsigned char* slot) {  // registers -> LDS
    if constexpr (!kDirect) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int n = u * kLoaders + gt, r = n / kChunk, c = n % kChunk;
        if (KB * kChunk % kLoaders != 0 && r >= KB) continue;
        if constexpr (F8) {
          const float power = kPowers ? __uint_as_float(scale_power(pvp[u])) : 1.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x0 = pk[u][2 * half], x1 = pk[u][2 * half + 1], y0 = pv[u][2 * half], y1 = pv[u][2 * half + 1];
            *reinterpret_cast<u32x4*>(slot + T::at(r, 2 * c + half)) = u32x4{widen2<DT, false>(x0), widen2<DT, true>(x0), widen2<DT, false>(x1), widen2<DT, true>(x1)};
            *reinterpret_cast<u32x4*>(slot + kTileBytes + T::at(r, 2 * c + half)) = u32x4{widen2<DT, false>(y0, power), widen2<DT, true>(y0, power), widen2<DT, false>(y1, power), widen2<DT, true>(y1, power)};
          }
        } else {
          *reinterpret_cast<u32x4*>(slot + T::at(r, c)) = pk[u];
          *reinterpret_cast<u32x4*>(slot + kTileBytes + T::at(r, c)) = pv[u];
        }
      }
      if constexpr (F8)
        if (gt < KB) {
          reinterpret_cast<float*>(slot + 2 * kTileBytes)[gt] = pks;
          reinterpret_cast<float*>(slot + 2 * kTileBytes)[KB + gt] = kPowers ? pvs * __uint_as_float((254u << 23) - scale_power(pvs)) : pvs;
        }
    }
  };

  // ---- the sums
  f32x16 acc[T::kOut];
#pragma unroll
  for (int o = 0; o < T::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[o][r] = 0.f;
  float m = -kInf, l = 0.f;  // running maximum (both halves alike) and this lane's share of the sum

  // The mask on a tile's scores, and the running maximum.
  auto soften = [&](f32x16 (&s)[NT], int k0) {
    if (k0 < f_lo || k0 + KB > f_hi || k0 + KB > g_hi) {  // some row does not see all of the tile
      const uint32_t span = static_cast<uint32_t>(s_hi > s_lo ? s_hi - s_lo : 0);
      const int first = k0 + 4 * h - s_lo;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t at = static_cast<uint32_t>(first + 32 * n + 8 * (r / 4) + r % 4);
          s[n][r] = at < span ? s[n][r] : -kInf;
        }
    }
    float tops[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 2) tops[r / 2 % 4] = fmaxf(fmaxf(tops[r / 2 % 4], s[n][r]), s[n][r + 1]);
    const float top = both_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    // The maximum is only there to keep the powers in range: it moves (and the sums are rescaled) when a score exceeds it
    // by more than 2^8, not with every new maximum.
    if (__any((top - m) * a.c > 8.f)) {
      const float mn = fmaxf(m, top), alpha = mn == -kInf ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int o = 0; o < T::kOut; ++o)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[o][r] *= alpha;
    }
  };

  // One tile: the scores, then the powers and the products with the values.  A product's operand is asked for kAhead products
  // before it, and the second half's powers are found under the first half's products.
  auto step = [&](const unsigned char* tk, int k0) {
    constexpr int kAhead = D == 80 ? 3 : 4, kScores = NT * T::kSteps, kProducts = NT * 2 * T::kOut;
    const unsigned char* tv = tk + kTileBytes;
    const float* scales = reinterpret_cast<const float*>(tk + 2 * kTileBytes);
    int rows_here = rows_at, cols_here = cols_at;  // (the addresses are made from these here: kept over the loop they would be spilled)
    asm volatile("" : "+v"(rows_here), "+v"(cols_here));
    auto read_k = [&](int i) { return read_rows<D>(tk, 32 * (i % NT), i / NT, rows_here); };
    auto read_v = [&](int i) { return read_cols<D>(tv, 32 * (i / (2 * T::kOut)), i / T::kOut % 2, i % T::kOut, cols_here); };
    f32x16 s[NT];
    u32x4 f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_k(i);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
    in_order();
#pragma unroll
    for (int i = 0; i < kScores; ++i) {
      s[i % NT] = mfma<DT>(f[i % kAhead], qf[i / NT], s[i % NT]);
      if (i + kAhead < kScores) f[i % kAhead] = read_k(i + kAhead);
      in_order();
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = read_v(i);
    in_order();
    if constexpr (F8) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 x = *reinterpret_cast<const float4*>(scales + 32 * n + 8 * g + 4 * h);
          s[n][4 * g] *= x.x, s[n][4 * g + 1] *= x.y, s[n][4 * g + 2] *= x.z, s[n][4 * g + 3] *= x.w;
        }
    }
    soften(s, k0);
    const float mc = m == -kInf ? 0.f : m * a.c;
    float sums[2] = {0.f, 0.f};
    auto power = [&](int n, int r) {  // of registers r and r + 1
      s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.c, -mc));
      s[n][r + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r + 1], a.c, -mc));
      sums[0] += s[n][r];
      sums[1] += s[n][r + 1];
      if constexpr (F8) {
        const float2 x = *reinterpret_cast<const float2*>(scales + KB + 32 * n + 8 * (r / 4) + 4 * h + r % 4);
        s[n][r] *= x.x, s[n][r + 1] *= x.y;
      }
    };
#pragma unroll
    for (int u = 0; u < 8; ++u) power(0, 2 * u);
    u32x4 p[2] = {pack_step<DT>(s[0], 0), pack_step<DT>(s[0], 1)};
    in_order();
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int n = i / (2 * T::kOut), t = i / T::kOut % 2, o = i % T::kOut, at = i % (2 * T::kOut);
      if (n > 0 && at == 0) p[0] = pack_step<DT>(s[n], 0), p[1] = pack_step<DT>(s[n], 1);
      acc[o] = mfma<DT>(f[i % kAhead], p[t], acc[o]);
      if (i + kAhead < kProducts) f[i % kAhead] = read_v(i + kAhead);
      if (n + 1 < NT) {
        const int each = (8 + 2 * T::kOut - 1) / (2 * T::kOut);
#pragma unroll
        for (int u = at * each; u < (at + 1) * each && u < 8; ++u) power(n + 1, 2 * u);
      }
      in_order();
    }
    l += sums[0] + sums[1];
  };

  if constexpr (RW == 8) {
    static_assert(!F8 && D == 128, "");
    // Two groups of four wavefronts, one of each on every SIMD, half a step apart: while one group's matrix units work -- P V of the last
    // tile, then the scores of the next -- the other finds its powers.  The first group loads the keys of the next tile, the second the
    // values; a barrier ends each half.
    unsigned char *const k_even = lds_slot<kTileBytes, 2>(), *const k_odd = lds_slot<kTileBytes, 3>(), *const v_even = lds_slot<kTileBytes, 4>(),
                  *const v_odd = lds_slot<kTileBytes, 5>();
    const bool late = rw >= 4;
    const int r0 = (rw & 3) * 16, my_step = static_cast<int>(late ? v_step : k_step);
    const char* const my = late ? vp : kp;
    uint32_t my_off[T::kChunks / 4];
#pragma unroll
    for (int i = 0; i < T::kChunks / 4; ++i) my_off[i] = stage_offset<D>(i, lane, [&](int r) { return static_cast<uint32_t>((r0 + r) * my_step); });
    auto load = [&](int t, unsigned char* slot) {
      const int k0 = g_lo + t * KB, left = g_hi - k0;
      const auto rs = attn_rsrc(my + static_cast<int64_t>(k0) * my_step, kRsrcBytes);
      if (left >= KB) stage16<D>(rs, slot + r0 * T::kPitch, my_off);
      else stage16<D>(rs, slot + r0 * T::kPitch, lane, [&](int r) { return r0 + r < left ? static_cast<uint32_t>((r0 + r) * my_step) : kOutside; });
    };
    auto visible = [&](int t) { const int k0 = g_lo + t * KB; return t < tiles && k0 < w_hi && k0 + KB > w_lo; };
    f32x16 sc[NT];
    u32x4 pr[2 * NT];
    bool before = false;  // there are powers of the last tile
    auto products = [&](int t, const unsigned char* tk, const unsigned char* tv) {
      constexpr int kAhead = 4, kScores = NT * T::kSteps, kProducts = NT * 2 * T::kOut;
      int rows_here = rows_at, cols_here = cols_at;
      asm volatile("" : "+v"(rows_here), "+v"(cols_here));
      auto read_k = [&](int i) { return read_rows<D>(tk, 32 * (i % NT), i / NT, rows_here); };
      auto read_v = [&](int i) { return read_cols<D>(tv, 32 * (i / (2 * T::kOut)), i / T::kOut % 2, i % T::kOut, cols_here); };
      u32x4 f[kAhead];
      if (before) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = read_v(i);
        in_order();
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
          acc[i % T::kOut] = mfma<DT>(f[i % kAhead], pr[i / T::kOut], acc[i % T::kOut]);
          if (i + kAhead < kProducts) f[i % kAhead] = read_v(i + kAhead);
          else f[i % kAhead] = read_k(i + kAhead - kProducts);  // (of no use behind the last tile)
          in_order();
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = read_k(i);
      }
      if (!visible(t)) return;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[n][r] = 0.f;
      in_order();
#pragma unroll
      for (int i = 0; i < kScores; ++i) {
        sc[i % NT] = mfma<DT>(f[i % kAhead], qf[i / NT], sc[i % NT]);
        if (i + kAhead < kScores) f[i % kAhead] = read_k(i + kAhead);
        in_order();
      }
    };
    auto powers = [&](int t) {
      before = visible(t);
      if (!before) return;
      const int k0 = g_lo + t * KB;
      soften(sc, k0);
      const float mc = m == -kInf ? 0.f : m * a.c;
      float sums[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          sc[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][r], a.c, -mc));
          sc[n][r + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][r + 1], a.c, -mc));
          sums[0] += sc[n][r];
          sums[1] += sc[n][r + 1];
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) pr[2 * n] = pack_step<DT>(sc[n], 0), pr[2 * n + 1] = pack_step<DT>(sc[n], 1);
      l += sums[0] + sums[1];
    };
    auto turn = [&](int t, unsigned char* k_this, unsigned char* k_next, unsigned char* v_last, unsigned char* v_next) {
      if (!late && t + 1 < tiles) load(t + 1, k_next);
      products(t, k_this, v_last);
      in_order();
      if (late) wait_loads();
      attn_barrier();
      if (late && t + 1 < tiles) load(t + 1, v_next);
      powers(t);
      in_order();
      if (!late) wait_loads();
      attn_barrier();
    };
    if (!late && tiles > 0) {
      load(0, k_even);
      wait_loads();
    }
    attn_barrier();
    if (late) {
      if (tiles > 0) load(0, v_even);
      attn_barrier();
    }
    for (int t = 0; t <= tiles; t += 2) {
      turn(t, k_even, k_odd, v_odd, v_odd);
      if (t + 1 <= tiles) turn(t + 1, k_odd, k_even, v_even, v_even);
    }
    if (!late) attn_barrier();
  }
  unsigned char *mine = lds + kw * kSlot, *other_slot = lds1 + kw * kSlot;
  if (RW != 8 && iters > 0) fetch(0, mine);
  auto turn = [&](int it, unsigned char* slot, unsigned char* other) {
    const int k0 = key0(it);
    if constexpr (kDirect) {
      wait_loads();
      attn_barrier();
      if (it + 1 < iters) fetch(it + 1, other);
    } else {
      put(slot);
      if (it + 1 < iters) fetch(it + 1, other);
      wait_lds();
      attn_barrier();
    }
    if (k0 < w_hi && k0 + KB > w_lo && k0 < g_hi) step(slot, k0);
  };
  if constexpr (RW != 8)
    for (int it = 0; it < iters; it += 2) {
      turn(it, mine, other_slot);
      if (it + 1 < iters) turn(it + 1, other_slot, mine);
    }
  l = both_sum(l);
  // ---- the result: joined over the key groups, then either the row itself or this split's part of it
  // Rows whose sum is not a number though the sum of their powers is are made again at the end; of fp16 codes also rows whose probabilities
  // times scales went beyond fp16.
  uint32_t again = columns(not_numbers<D, kPowers>(acc) && s_hi > s_lo);
  uint16_t* out = a.out + ((static_cast<int64_t>(b) * a.n_queries + qi) * a.n_q + hq) * D;
  const int64_t stat = static_cast<int64_t>(pair) * a.rows + row;
  if constexpr (KW == 1) {
    const float inv = some && l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    if (!F8 && a.rest != nullptr) store_row<DT, D, true>(acc, some ? inv : 0.f, live ? out : nullptr, lane, live ? a.rest + (out - a.out) : nullptr);
    else store_row<DT, D>(acc, some ? inv : 0.f, live ? out : nullptr, lane);
    if (!some && live) {  // (0 * NaN above)
#pragma unroll
      for (int c = 0; c < D / 8; c += 2) *reinterpret_cast<u32x4*>(out + 8 * (c + h)) = u32x4{0u, 0u, 0u, 0u};
    }
    again &= columns(l == l);
    if (a.lse != nullptr && live && h == 0) a.lse[stat] = some ? __builtin_fmaf(m, a.c, __builtin_amdgcn_logf(l)) : kInf;
  } else {
    // Every key group's sums to LDS, 64 channels at a time, scaled to the common maximum; then a thread adds up 8 channels of a row.
    float2* stats = reinterpret_cast<float2*>(lds + kJoinStats);
    float* sums = reinterpret_cast<float*>(lds);
    __shared__ uint32_t s_again[4];
    __syncthreads();
    if (h == 0) stats[wave * 32 + lane] = float2{m, l};
    if (lane == 0) s_again[wave] = again;
    __syncthreads();
    float top = -kInf, l_all = 0.f;
#pragma unroll
    for (int u = 0; u < KW; ++u) top = fmaxf(top, stats[(u * RW + rw) * 32 + (lane & 31)].x);
    again = __builtin_amdgcn_readfirstlane(s_again[rw] | s_again[rw + RW * (KW - 1)]);
    if (again != 0) {
#pragma unroll
      for (int u = 0; u < KW; ++u) {
        const float2 st = stats[(u * RW + rw) * 32 + (lane & 31)];
        l_all += st.x == -kInf ? 0.f * st.y : st.y * __builtin_amdgcn_exp2f((st.x - top) * a.c);
      }
      again &= columns(l_all == l_all);
    }
    const float f = m == -kInf ? 0.f : __builtin_amdgcn_exp2f((m - top) * a.c);
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += 64) {
      if (c0 > 0) __syncthreads();
#pragma unroll
      for (int o = c0 / 32; o < (c0 + 64) / 32 && o < T::kOut; ++o)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * o + 8 * g < D)
            *reinterpret_cast<float4*>(sums + (wave * 32 + (lane & 31)) * 68 + 32 * o - c0 + 8 * g + 4 * h) =
                float4{acc[o][4 * g] * f, acc[o][4 * g + 1] * f, acc[o][4 * g + 2] * f, acc[o][4 * g + 3] * f};
      __syncthreads();
      // wavefront (kw, rw) finishes rows rw * 32 + kw * (32 / KW) ..., 8 lanes a row
      constexpr int kMine = 32 / KW, kLanes = 8;
#pragma unroll
      for (int first = 0; first < kMine; first += 64 / kLanes) {
        const int r = kw * kMine + first + lane / kLanes, ch = c0 / 8 + lane % kLanes;
        const int row_r = tile * 32 * RW + rw * 32 + r;
        const bool mine_r = row_r < a.rows && ch < D / 8;
        float top_r = -kInf, l_r = 0.f;
#pragma unroll
        for (int u = 0; u < KW; ++u) top_r = fmaxf(top_r, stats[(u * RW + rw) * 32 + r].x);
#pragma unroll
        for (int u = 0; u < KW; ++u) {
          const float2 st = stats[(u * RW + rw) * 32 + r];
          l_r += st.x == -kInf ? 0.f * st.y : st.y * __builtin_amdgcn_exp2f((st.x - top_r) * a.c);
        }
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ch < D / 8)
#pragma unroll
          for (int u = 0; u < KW; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += sums[((u * RW + rw) * 32 + r) * 68 + (ch * 8 - c0) + e];
        const int i_r = row_r < a.rows ? a.by_group.div(row_r) : 0;
        int lo_r = 0, hi_r = 0;
        if (row_r < a.rows) key_range(a.mask, b, i_r, a.n_queries, a.n_keys, lo_r, hi_r);
        const bool some_r = hi_r > lo_r;
        const int64_t to = ((static_cast<int64_t>(b) * a.n_queries + i_r) * a.n_q + hk * a.group + row_r - i_r * a.group) * D;
        const int64_t to_part = (static_cast<int64_t>(pair) * a.splits + split) * a.rows + row_r;
        const bool store_r = !(again >> r & 1);
        if (mine_r) {
          if (a.splits > 1) {
            float4* dst = reinterpret_cast<float4*>(a.part + to_part * D + ch * 8);
            if (store_r) {
              dst[0] = float4{v[0], v[1], v[2], v[3]};
              dst[1] = float4{v[4], v[5], v[6], v[7]};
            }
            if (ch == 0) part_stats(a, D)[to_part] = float2{top_r, l_r};
          } else {
            const float inv = some_r ? 1.f / l_r : 0.f;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = some_r ? v[e] * inv : 0.f;
            if (store_r) *reinterpret_cast<u32x4*>(a.out + to + ch * 8) = pack16<DT>(w);
            if (store_r && a.rest != nullptr)
              *reinterpret_cast<u32x2*>(a.rest + to + ch * 8) = u32x2{pack_rest_of<DT>(w[0], w[1], w[2], w[3]), pack_rest_of<DT>(w[4], w[5], w[6], w[7])};
            if (ch == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(pair) * a.rows + row_r] = some_r ? __builtin_fmaf(top_r, a.c, __builtin_amdgcn_logf(l_r)) : kInf;
          }
        }
      }
    }
    if (kw != 0) return;
    m = top, l = l_all;
  }
  if (again != 0) rows_again<DT, D, F8, RW>(a, again, m, l);
}

constexpr int kMaxSplits = 256;

// Joins the splits of a row, lane l channels l and l + 64.  ROWS = 4: a wavefront per row, for a few splits of many rows (a workgroup per
// row took 26 us for 8000 rows of 3 splits).  ROWS = 1: a workgroup per row, every wavefront a quarter of the splits, for many (a
// wavefront per row took 24 us for 128 rows of 32 splits: one dependent load after the other).
template <int DT, int D, int ROWS>
__global__ __launch_bounds__(256) void attn_join_kernel(FwdArgs a) {
  __shared__ float s_top[4], s_sum[4], s_weight[kMaxSplits], s_out[4][128];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * ROWS + (ROWS == 4 ? wave : 0);
  if (at >= static_cast<int64_t>(a.batch) * a.n_kv * a.rows) return;
  const int pair = a.by_rows.div(static_cast<int>(at)), row = static_cast<int>(at) - pair * a.rows;
  const float2* stats = part_stats(a, D) + static_cast<int64_t>(pair) * a.splits * a.rows + row;
  const float* part = a.part + (static_cast<int64_t>(pair) * a.splits * a.rows + row) * D;
  const int mine = ROWS == 4 ? lane : tid;
  const float2 st = mine < a.splits ? stats[static_cast<int64_t>(mine) * a.rows] : float2{-kInf, 0.f};
  const int b = a.by_kv.div(pair), hk = pair - b * a.n_kv;
  const int i = a.by_group.div(row), hq = hk * a.group + row - i * a.group;
  int lo, hi;
  key_range(a.mask, b, i, a.n_queries, a.n_keys, lo, hi);
  float top = wave_max(st.x);
  if constexpr (ROWS == 1) {
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  }
  // (a split that the row sees nothing of has no part, whatever stands in its place)
  const float f = st.x == -kInf ? 0.f : __builtin_amdgcn_exp2f((st.x - top) * a.c);
  float l = wave_sum(st.y * f);
  if constexpr (ROWS == 1) {
    s_weight[tid] = f;
    if (lane == 0) s_sum[wave] = l;
    __syncthreads();
    l = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  }
  float o[2] = {0.f, 0.f};
  constexpr int kStep = ROWS == 4 ? 1 : 4, kBatch = ROWS == 4 ? 4 : 8;
  for (int s0 = ROWS == 4 ? 0 : wave; s0 < a.splits; s0 += kBatch * kStep) {
    float x[kBatch][2], w[kBatch];  // (of splits past the last: the last one's, without weight)
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int s = min(s0 + n * kStep, a.splits - 1);
      w[n] = ROWS == 4 ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s)) : s_weight[s];
      if (s0 + n * kStep >= a.splits) w[n] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) x[n][u] = lane + 64 * u < D ? part[static_cast<int64_t>(s) * a.rows * D + lane + 64 * u] : 0.f;
    }
#pragma unroll
    for (int n = 0; n < kBatch; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) o[u] += w[n] == 0.f ? 0.f : x[n][u] * w[n];
  }
  const int64_t to = ((static_cast<int64_t>(b) * a.n_queries + i) * a.n_q + hq) * D;
  auto store = [&](int c, float sum) {
    const float x = hi > lo ? sum / l : 0.f;
    a.out[to + c] = static_cast<uint16_t>(Elem<DT>::store(x));
    if (a.rest != nullptr) a.rest[to + c] = static_cast<uint8_t>(pack_rest(rest_of<DT>(x), 0.f, 0.f, 0.f));
  };
  if constexpr (ROWS == 4) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 64 * u < D) store(lane + 64 * u, o[u]);
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u) s_out[wave][lane + 64 * u] = o[u];
    __syncthreads();
    if (tid < D) store(tid, (s_out[0][tid] + s_out[1][tid]) + (s_out[2][tid] + s_out[3][tid]));
  }
  if (a.lse != nullptr && (ROWS == 4 ? lane : tid) == 0) a.lse[at] = hi > lo ? __builtin_fmaf(top, a.c, __builtin_amdgcn_logf(l)) : kInf;
}

// How a call is spread over the chip: wavefronts of the workgroup that take rows (4, 2 or 1), and splits of the keys.
struct FwdPlan {
  int row_waves, splits;
};
FwdPlan plan(int64_t pairs, int64_t rows, int64_t keys, int head_dim, bool f8) {
  const int cus = device_cu_count();
  FwdPlan p{4, 1};
  // Rows that fill 128-row workgroups two to a CU take those, fewer take 64-row ones, whose two pairs of wavefronts share the keys.  With
  // 64 / 128: 5003 packed tokens of 12 / 4 heads of 64 28 / 38 us (472 large workgroups); 16 x 912 tokens of 16 / 2 heads of 128 107 / 74,
  // 48 x 1024 patches of 16 heads of 80 in windows 203 / 131 (1824 and 6144).
  if (rows <= 64 || pairs * ((rows + 127) / 128) < 2 * cus) p.row_waves = 2;
  // Heads of 128 over many keys, of more rows than a 256-row workgroup to a CU takes: two groups of wavefronts in step with each other.
  // Its start is not under another workgroup's work, so that it pays for long rows only.  128 / 256 rows: 8192 causal tokens of 16 / 2 heads
  // 287 / 255 us, 2 x 4096 that see all 265 / 250, 16384 causal ones 1028 / 977, 4 x 8192 packed ones 301 / 309; 8 x 2048 causal ones 147 /
  // 148, 4 x 2900 146 / 150, 16 x 912 73 / 82.
  else if (head_dim == 128 && !f8 && keys >= 4096 && pairs * ((rows + 255) / 256) >= cus) p.row_waves = 8;
  const int64_t groups = pairs * ((rows + 32 * p.row_waves - 1) / (32 * p.row_waves));
  if (p.row_waves == 2 && groups > 0 && groups < 2 * cus) {
    // Too few workgroups for the chip: the keys in n parts, up to two workgroups to a CU, of at least a tile for each key group.  A tile
    // of 64 keys takes about 0.8 us, the join 4, and writing and reading the parts of n splits n times what one's take at 3 TB/s: the n of
    // the least sum, if that is less than without.  Measured without / with: one query of 8 heads over 8 x 32768 cached keys of 2 heads 35 us
    // in 32 parts, 40 over 64; 4 x 300 causal tokens of 16 / 2 heads 11 / 28 (2 parts), 2000 tokens 37 / 48 (2), 32 x 5 queries over 2400
    // to 3000 cached keys of 8 heads of 64 45 / 33 (2).
    const double tiles = 0.8 * (keys / 64.0), each = static_cast<double>(pairs) * rows * head_dim * 8 / 3e6;
    const int64_t want = (2 * cus + groups - 1) / groups, most = keys / 64;
    int64_t n = static_cast<int64_t>(std::sqrt(tiles / each));
    n = std::min({n, want, most, static_cast<int64_t>(kMaxSplits)});
    if (n > 1 && tiles / n + 4 + n * each < tiles) p.splits = static_cast<int>(n);
  }
  return p;
}

template <int DT, int D, bool F8>
int launch_fwd(FwdArgs& a, const FwdPlan& p, hipStream_t s) {
  a.splits = p.splits;
  a.row_tiles = (a.rows + 32 * p.row_waves - 1) / (32 * p.row_waves);
  const int pairs = a.batch * a.n_kv;
  a.by_splits = Divider(p.splits), a.by_kv = Divider(a.n_kv), a.by_group = Divider(a.group);
  a.spread = Spread(pairs, a.row_tiles);
  const int64_t blocks = static_cast<int64_t>(a.batch) * a.n_kv * a.row_tiles * a.splits;
  const int64_t all_rows = static_cast<int64_t>(a.batch) * a.n_kv * a.rows, joins = a.splits <= 8 ? (all_rows + 3) / 4 : all_rows;
  if (too_many_blocks(blocks, p.row_waves == 8 ? 512 : 256) || (a.splits > 1 && too_many_blocks(joins, 256))) return fail(WX_ERR_UNSUPPORTED, "attention: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  if (p.row_waves == 2) {
    hipLaunchKernelGGL((attn_fwd_kernel<DT, D, F8, 2>), grid, block, 0, s, a);
  } else if (p.row_waves == 4) {
    hipLaunchKernelGGL((attn_fwd_kernel<DT, D, F8, 4>), grid, block, 0, s, a);
  } else if constexpr (D == 128 && !F8) {
    hipLaunchKernelGGL((attn_fwd_kernel<DT, D, F8, 8>), grid, dim3(512), 0, s, a);
  }
  if (int rc = check_launch("attn_fwd_kernel")) return rc;
  if (a.splits > 1) {
    a.by_rows = Divider(a.rows);
    if (a.splits <= 8) hipLaunchKernelGGL((attn_join_kernel<DT, D, 4>), dim3(static_cast<unsigned>(joins)), block, 0, s, a);
    else hipLaunchKernelGGL((attn_join_kernel<DT, D, 1>), dim3(static_cast<unsigned>(joins)), block, 0, s, a);
    return check_launch("attn_join_kernel");
  }
  return WX_OK;
}

template <bool F8>
int dispatch_fwd(FwdArgs& a, const FwdPlan& p, int head_dim, int dtype, hipStream_t s) {
  if (dtype == WX_BF16) {
    if (head_dim == 64) return launch_fwd<WX_BF16, 64, F8>(a, p, s);
    if (head_dim == 80) return launch_fwd<WX_BF16, 80, F8>(a, p, s);
    return launch_fwd<WX_BF16, 128, F8>(a, p, s);
  }
  if (head_dim == 64) return launch_fwd<WX_F16, 64, F8>(a, p, s);
  if (head_dim == 80) return launch_fwd<WX_F16, 80, F8>(a, p, s);
  return launch_fwd<WX_F16, 128, F8>(a, p, s);
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

// Shared by the forward and the backward: sizes, types and strides that the kernels take.
int attention_check(const char* who, int64_t batch, int n_q, int n_kv, int64_t n_queries, int64_t n_keys, int head_dim, int dtype,
                    float scale) {
  if (batch < 0 || n_q < 0 || n_kv < 0 || n_queries < 0 || n_keys < 0) return fail(WX_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (head_dim != 64 && head_dim != 80 && head_dim != 128)
    return fail(WX_ERR_UNSUPPORTED, "%s: head_dim %d must be 64, 80 or 128", who, head_dim);
  if (dtype != WX_BF16 && dtype != WX_F16) return fail(WX_ERR_UNSUPPORTED, "%s: dtype %d must be bf16 or fp16", who, dtype);
  if (n_kv == 0 ? n_q != 0 : n_q % n_kv != 0)
    return fail(WX_ERR_INVALID_ARGUMENT, "%s: %d query heads are no multiple of %d key / value heads", who, n_q, n_kv);
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", who);
  const int64_t group = n_kv ? n_q / n_kv : 0;
  if (group > 1024) return fail(WX_ERR_UNSUPPORTED, "%s: more than 1024 query heads to a key / value head", who);
  if (n_keys > 0x3fffffffll || (group && n_queries > 0x3fffffffll / group) || batch > 0x7fffffffll / (n_kv ? n_kv : 1))
    return fail(WX_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 rows or keys", who);
  return WX_OK;
}

// 16-byte rows, and `span` positions and `heads` heads of 2 (1) byte elements within 31 bits of a tile's first byte
int attention_check_strides(const char* who, const char* name, const int64_t* st, int elem_bytes, int64_t span, int64_t heads) {
  const int64_t unit = 16 / elem_bytes;
  for (int i = 0; i < 3; ++i)
    if (st[i] % unit != 0 || st[i] < 0) return fail(WX_ERR_UNSUPPORTED, "%s: %s's strides must be positive and keep rows 16-byte aligned", who, name);
  const int64_t most = 0x7ff00000ll / elem_bytes;
  if (st[2] > most / span || (heads > 1 && st[1] > (most - st[2] * span) / (heads - 1)))
    return fail(WX_ERR_UNSUPPORTED, "%s: %s's strides are too large", who, name);
  return WX_OK;
}

}  // namespace wx

using namespace wx;

extern "C" size_t wx_attention_workspace_bytes(int64_t batch, int n_q_heads, int n_kv_heads, int64_t n_queries, int64_t n_keys,
                                               int head_dim) {
  if (batch <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_queries <= 0 || n_keys < 0 || head_dim <= 0) return 0;
  const int64_t rows = n_queries * (n_q_heads / n_kv_heads);
  const FwdPlan p = plan(batch * n_kv_heads, rows, n_keys, head_dim, false);  // (of the splits, which do not depend on the type)
  return p.splits == 1 ? 0 : static_cast<size_t>(batch) * n_kv_heads * p.splits * rows * (head_dim + 2) * sizeof(float);
}

static int forward(const char* who, const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, bool f8,
                   void* out, float* lse, void* rest, const int32_t* key_ranges, const int32_t* key_lengths, int causal, int64_t batch,
                   int n_q, int n_kv, int64_t n_queries, int64_t n_keys, int head_dim, const int64_t* qs, const int64_t* ks,
                   const int64_t* vs, float scale, int dtype, void* workspace, size_t workspace_bytes, wx_stream_t stream) {
  if (int rc = attention_check(who, batch, n_q, n_kv, n_queries, n_keys, head_dim, dtype, scale)) return rc;
  if (!qs || !ks || !vs) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null strides", who);
  if (batch == 0 || n_q == 0 || n_queries == 0) return WX_OK;
  if (!q || !out || (n_keys > 0 && (!k || !v || (f8 && (!k_scale || !v_scale))))) return fail(WX_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(rest)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(key_ranges) & 7) return fail(WX_ERR_INVALID_ARGUMENT, "%s: key_ranges must be 8-byte aligned", who);
  const int group = n_q / n_kv;
  if (int rc = attention_check_strides(who, "q", qs, 2, 1, 1)) return rc;
  if (int rc = attention_check_strides(who, "k", ks, f8 ? 1 : 2, 64, 1)) return rc;
  if (int rc = attention_check_strides(who, "v", vs, f8 ? 1 : 2, 64, 1)) return rc;
  FwdArgs a{};
  a.q = q, a.k = k, a.v = v;
  for (int i = 0; i < 3; ++i) a.qs[i] = qs[i], a.ks[i] = ks[i], a.vs[i] = vs[i];
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.out = static_cast<uint16_t*>(out), a.lse = lse, a.rest = static_cast<uint8_t*>(rest);
  a.mask = {reinterpret_cast<const int2*>(key_ranges), key_lengths, causal};
  a.batch = static_cast<int>(batch), a.n_q = n_q, a.n_kv = n_kv, a.n_queries = static_cast<int>(n_queries), a.n_keys = static_cast<int>(n_keys);
  a.group = group, a.rows = static_cast<int>(n_queries) * group;
  a.c = scale * kLog2e;
  const FwdPlan p = plan(batch * n_kv, a.rows, n_keys, head_dim, f8);
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < wx_attention_workspace_bytes(batch, n_q, n_kv, n_queries, n_keys, head_dim))
      return fail(WX_ERR_WORKSPACE, "%s: workspace too small (see wx_attention_workspace_bytes)", who);
    if (misaligned(workspace)) return fail(WX_ERR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
    a.part = static_cast<float*>(workspace);
  }
  return f8 ? dispatch_fwd<true>(a, p, head_dim, dtype, as_stream(stream)) : dispatch_fwd<false>(a, p, head_dim, dtype, as_stream(stream));
}

extern "C" int wx_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* rest, const int32_t* key_ranges,
                                const int32_t* key_lengths, int causal, int64_t batch, int n_q_heads, int n_kv_heads,
                                int64_t n_queries, int64_t n_keys, int head_dim, const int64_t q_strides[3], const int64_t k_strides[3],
                                const int64_t v_strides[3], float scale, int dtype, void* workspace, size_t workspace_bytes,
                                wx_stream_t stream) {
  return forward("wx_attention_fwd", q, k, v, nullptr, nullptr, false, out, lse, rest, key_ranges, key_lengths, causal, batch, n_q_heads,
                 n_kv_heads, n_queries, n_keys, head_dim, q_strides, k_strides, v_strides, scale, dtype, workspace, workspace_bytes, stream);
}

extern "C" int wx_cached_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                   void* out, const int32_t* key_ranges, const int32_t* key_lengths, int causal, int64_t batch,
                                   int n_q_heads, int n_kv_heads, int64_t n_queries, int64_t capacity, int head_dim,
                                   const int64_t q_strides[3], float scale, int dtype, void* workspace, size_t workspace_bytes,
                                   wx_stream_t stream) {
  const int64_t st[3] = {n_kv_heads * capacity * head_dim, capacity * head_dim, head_dim};
  return forward("wx_cached_attention", q, k_cache, v_cache, k_scale, v_scale, true, out, nullptr, nullptr, key_ranges, key_lengths, causal, batch,
                 n_q_heads, n_kv_heads, n_queries, capacity, head_dim, q_strides, st, st, scale, dtype, workspace, workspace_bytes, stream);
}
