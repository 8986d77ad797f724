// Shared device code of the attention kernels (attention_fwd.hip, attention_bwd.hip), gfx950.
//
// Rows.  The G = Hq / Hkv query heads that share a key / value head are packed beside each other: row r of a
// (sequence, key / value head) pair is query r / G of head hkv * G + r % G.  A tile of rows then covers few queries, so a
// causal tile wastes little past the diagonal, one read of a key tile serves all heads of the group, and a single
// query fills G rows of a matrix product instead of one.
//
// Products.  All run on v_mfma_f32_32x32x16 with the scores transposed, S^T = K Q^T: the accumulator's column is the row
// (lane & 31) and its registers are keys 8 g + 4 h + i (register 4 g + i, h = lane >> 5).  The softmax of a row is then
// a reduction over a lane's own registers and one exchange between the lane halves, and the probabilities are already
// the B operand of O^T = V^T P^T if the contraction takes its 16 keys of step t in the order 16 t + 8 (j / 4) + 4 h + j % 4:
// nothing crosses lanes, the A operand is read in that order by transposing LDS reads.
//
// LDS tiles hold a row of D 2-byte values per key (query), in chunks of 16 bytes, pitch 128 (D = 64), 192 (80) or 256 bytes
// (128).  chunk c of row r is kept at chunk c ^ swizzle(r): 16 consecutive rows read at one chunk (b128) and 4 rows read at
// four neighbouring chunks (transposing b64) fall into different banks.
#pragma once

#include "common.h"

namespace wx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 att_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 att_bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 att_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 att_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 att_f16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();

struct AttnMask {
  const int2* ranges;   // [batch, n_queries] (lo, hi) or null
  const int32_t* lens;  // [batch] or null
  int causal;
};

// [lo, hi) of the keys that query i of sequence b sees; lo = hi = 0 when there are none.  What the mask holds in memory is asked
// for first (mask_row), so that it does not wait behind what is asked for in between.
struct MaskRow {
  int len;
  int2 range;
};
__device__ __forceinline__ MaskRow mask_row(const AttnMask& m, int b, int i, int n_queries, int n_keys) {
  MaskRow r{n_keys, int2{0, n_keys}};
  if (m.ranges != nullptr) r.range = m.ranges[static_cast<int64_t>(b) * n_queries + i];
  if (m.lens != nullptr) r.len = m.lens[b];
  return r;
}
__device__ __forceinline__ void key_range(const AttnMask& m, const MaskRow& r, int i, int n_queries, int n_keys, int& lo, int& hi) {
  const int len = r.len < 0 ? 0 : (r.len > n_keys ? n_keys : r.len);
  lo = max(0, r.range.x);
  hi = min(len, r.range.y);
  if (m.causal) hi = min(hi, len - n_queries + i + 1);
  if (hi <= lo) lo = hi = 0;
}
__device__ __forceinline__ void key_range(const AttnMask& m, int b, int i, int n_queries, int n_keys, int& lo, int& hi) {
  key_range(m, mask_row(m, b, i, n_queries, n_keys), i, n_queries, n_keys, lo, hi);
}

// n / d for n < 2^31 by a multiplication: the host makes the factor (a division by a number from memory is some 20 instructions,
// and a workgroup's coordinates take half a dozen).
struct Divider {
  uint32_t d, factor, shift;
  Divider() = default;
  explicit Divider(uint32_t by) : d(by) {
    shift = 0;
    while ((1ull << shift) < by) ++shift;
    factor = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), factor) + static_cast<uint32_t>(n)) >> shift);
  }
};

// Workgroup -> (pair, tile of it), the last tiles first: under a causal mask they are the longest.  Where the pairs divide by 8 every XCD
// gets an eighth of them, in a row: their keys are read into one L2, and heads of 80, whose rows share cache lines with the next
// head's, into no second one (48 x 1024 patches in windows 120 us; 132 with the pairs dealt round).  Of many pairs `wide` at a time, so that
// their keys stay in that L2.
struct Spread {
  int pairs, wide, tiles;
  Divider by_pass, by_wide;
  Spread() = default;
  Spread(int pairs_, int tiles_) : pairs(pairs_), wide(pairs_ % 8 == 0 ? pairs_ / 8 : pairs_), tiles(tiles_) {
    if (pairs % 8 == 0 && wide > 8)
      for (int n = 8; n >= 4; --n)
        if (wide % n == 0) {
          wide = n;
          break;
        }
    by_pass = Divider(static_cast<uint32_t>(wide) * tiles), by_wide = Divider(wide);
  }
  __device__ __forceinline__ void place(int id, int& pair, int& tile) const {
    const bool dealt = pairs % 8 == 0;
    const int j = dealt ? id >> 3 : id, pass = by_pass.div(j), rest = j - pass * static_cast<int>(by_pass.d), t = by_wide.div(rest);
    pair = (dealt ? (id & 7) * (pairs >> 3) : 0) + pass * wide + rest - t * wide;
    tile = tiles - 1 - t;
  }
};

template <int D>
struct AttnTile {
  static constexpr int kPitch = D == 64 ? 128 : (D == 80 ? 192 : 256);
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kSteps = D / 16;         // contraction steps over the head
  static constexpr int kOut = (D + 31) / 32;    // 32-channel tiles of an output (the last one of D = 80 is half padding)
  __device__ static __forceinline__ int swizzle(int row) {
    if constexpr (kPitch == 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (kPitch == 128) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
  }
  __device__ static __forceinline__ int at(int row, int chunk) { return row * kPitch + ((chunk ^ swizzle(row)) << 4); }
};

#define WX_LDS(p) ((__attribute__((address_space(3))) void*)(p))

__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_rsrc(const void* base, uint32_t bytes) {
  const uint64_t v = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  void* p = reinterpret_cast<void*>((static_cast<uint64_t>(hi) << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, static_cast<int>(bytes), 0x00020000);
}
constexpr uint32_t kRsrcBytes = 0x7ffffff0u;  // offsets from here on read as zero
constexpr uint32_t kOutside = 0x80000000u;

template <int DT>
__device__ __forceinline__ f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (DT == WX_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(att_bf16x8, a), __builtin_bit_cast(att_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(att_f16x8, a), __builtin_bit_cast(att_f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == WX_BF16) {
    const att_bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const att_f16x2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};  // (to nearest; the packed convert rounds to zero)
    return __builtin_bit_cast(uint32_t, v);
  }
}

// B operand of contraction step t (keys 16 t .. 16 t + 15 in the order above) from the accumulator registers of 32 keys.
template <int DT>
__device__ __forceinline__ u32x4 pack_step(const f32x16& p, int t) {
  const int r = 8 * t;
  return u32x4{pack2<DT>(p[r], p[r + 1]), pack2<DT>(p[r + 2], p[r + 3]), pack2<DT>(p[r + 4], p[r + 5]), pack2<DT>(p[r + 6], p[r + 7])};
}

// The value of this lane's partner in the other half (lane ^ 32) and its own: max / sum of the two in both.
__device__ __forceinline__ float both_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
// Smallest / largest of the 32 values that a wavefront's halves both hold, the same in all lanes: rotations inside each row of 16
// lanes, then the first lanes of two rows.
template <bool MAX>
__device__ __forceinline__ int wave_extreme(int x) {
#define WX_STEP(N)                                                           \
  {                                                                          \
    const int y = __builtin_amdgcn_update_dpp(x, x, 0x120 + N, 0xF, 0xF, false); \
    x = MAX ? max(x, y) : min(x, y);                                         \
  }
  WX_STEP(8)
  WX_STEP(4)
  WX_STEP(2)
  WX_STEP(1)
#undef WX_STEP
  const int a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  return MAX ? max(a, b) : min(a, b);
}

__device__ __forceinline__ int wave_prefix(int x) {  // inclusive, over the wavefront's lanes
#define WX_ADD(CTRL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false)
  WX_ADD(0x111, 0xF);
  WX_ADD(0x112, 0xF);
  WX_ADD(0x114, 0xF);
  WX_ADD(0x118, 0xF);
  WX_ADD(0x142, 0xA);  // (the last lane of a row of 16 to the next row, of 32 to the next half)
  WX_ADD(0x143, 0xC);
#undef WX_ADD
  return x;
}

// Byte offsets, in a tile, of what a lane reads of its first block: the other blocks lie at constant distances and exclusive-ors.
//   rows  A operand, contraction over the head: row lane & 31 of 32 rows, channels 16 t + 8 h .. + 7 of step t
//   cols  A operand, contraction over the tile's rows: channel 32 o + (lane & 31), rows 16 t + 8 (j / 4) + 4 h + j % 4
template <int D>
__device__ __forceinline__ int rows_base(int lane) {
  return AttnTile<D>::at(lane & 31, lane >> 5);
}
// (ds_read_b64_tr_b16: lane j of 16 gives the address of 4 consecutive channels of row j >> 2 and receives channel j of the 4 rows)
template <int D>
__device__ __forceinline__ int cols_base(int lane) {
  return AttnTile<D>::at(4 * (lane >> 5) + ((lane >> 2) & 3), 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);
}
template <int D>
__device__ __forceinline__ u32x4 read_rows(const unsigned char* tile, int row0, int t, int base) {
  using T = AttnTile<D>;
  // chunk 2 t + h of a swizzled row: 2 t is an exclusive-or of the bits that the swizzle reaches and a sum above them
  constexpr int kXor = T::kPitch == 256 ? 255 : (T::kPitch == 128 ? 127 : 63);
  const int c = 32 * t;
  return *reinterpret_cast<const u32x4*>(tile + (base ^ (c & kXor)) + (c & ~kXor) + row0 * T::kPitch);  // (row0: a multiple of 16)
}
template <int D>
__device__ __forceinline__ u32x4 read_cols(const unsigned char* tile, int row0, int t, int o, int base) {
  using T = AttnTile<D>;
  constexpr int kXor = T::kPitch == 256 ? 255 : (T::kPitch == 128 ? 127 : 63);
  const int c = 64 * o;
  typedef __attribute__((address_space(3))) att_bf16x4* P;
  const unsigned char* at = tile + (row0 + 16 * t) * T::kPitch + (c & ~kXor);
  const att_bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((P)(at + (base ^ (c & kXor))));
  const att_bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((P)(at + 8 * T::kPitch + (base ^ (c & kXor) ^ 32)));  // 8 rows on: swizzle ^ 2
  const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
  return u32x4{x[0], x[1], y[0], y[1]};
}

// 16 consecutive rows of a tile, straight from global memory to LDS, by one wavefront: instruction i fills 1 KiB.  `offset(row)` is
// the byte offset of tile row `row` (0..15 from the wavefront's first) from the descriptor's base, or kOutside: such rows become zeros.
template <int D, class Offset>
__device__ __forceinline__ uint32_t stage_offset(int i, int lane, Offset offset) {
  using T = AttnTile<D>;
  const int n = i * 64 + lane, row = n / T::kChunks, chunk = (n % T::kChunks) ^ T::swizzle(row);
  const uint32_t off = offset(row);
  if (off == kOutside || (T::kChunks * 8 > D && chunk >= D / 8)) return kOutside;
  return off + static_cast<uint32_t>(chunk) * 16u;
}
template <int D, class Offset>
__device__ __forceinline__ void stage16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds, int lane, Offset offset) {
#pragma unroll
  for (int i = 0; i < AttnTile<D>::kChunks / 4; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, WX_LDS(lds + i * 1024), 16, static_cast<int>(stage_offset<D>(i, lane, offset)), 0, 0, 0);
}
// The same from offsets that were made before (all rows inside).
template <int D>
__device__ __forceinline__ void stage16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds, const uint32_t* offsets, int further = 0) {
#pragma unroll
  for (int i = 0; i < AttnTile<D>::kChunks / 4; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, WX_LDS(lds + i * 1024), 16, static_cast<int>(offsets[i]), further, 0, 0);
}

// One LDS array per (size, index).  A kernel's two slots for tiles are arrays of their own, at constant addresses in a loop unrolled
// by two: where both were parts of one array the compiler took the transposing reads of a tile for reads of what the loads in
// flight write, and waited for the next tile in the middle of every tile.
template <int BYTES, int ID>
__device__ __forceinline__ unsigned char* lds_slot() {
  __shared__ __attribute__((aligned(1024))) unsigned char s[BYTES];
  return s;
}

// Keeps the order in which the code stands.  Left to itself the scheduler asks for an operand from LDS right in front of the product
// that needs it and waits for each; the loops below ask a few products ahead and put other work between the products.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ void attn_barrier() {  // (no fences: they would drain the loads in flight)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
constexpr int attn_wait(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(attn_wait(0, 15));
  asm volatile("" ::: "memory");
}
// behind this wavefront's own LDS writes; loads from memory stay in flight
__device__ __forceinline__ void attn_lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(attn_wait(63, 0));
  attn_barrier();
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(attn_wait(63, 0));
  asm volatile("" ::: "memory");
}

// What rounding the output to its type leaves, as e5m2, for the backward's delta = rowsum(dO O): with O as rounded, delta's error is
// a quarter of dQ's, or most of it where the values differ by little of their size.  It is kept times a power of two that puts what
// outputs can leave into e5m2's range, 2^-16 to 57344: all of fp16's (2^-25 to 16), and what outputs of 2^-16 to 2^16 leave in bf16.  (Beyond that
// the backward leaves a row's rests out; below, they are zero.)
template <int DT>
constexpr float kRestUp = DT == WX_F16 ? 2048.f : 256.f;
__device__ __forceinline__ uint32_t pack_rest(float a, float b, float c, float d) {
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_bf8_f32(c, d, __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false), true));
}
template <int DT>
__device__ __forceinline__ float rest_of(float x, float rounded) { return (x - rounded) * kRestUp<DT>; }
template <int DT>
__device__ __forceinline__ float rest_of(float x) { return rest_of<DT>(x, Elem<DT>::round(x)); }
template <int DT>
__device__ __forceinline__ uint32_t pack_rest_of(float a, float b, float c, float d) {
  return pack_rest(rest_of<DT>(a), rest_of<DT>(b), rest_of<DT>(c), rest_of<DT>(d));
}

// Transposed accumulators (channel 32 o + 8 g + 4 h + i, row lane & 31) to one row of 2-byte values: the halves trade groups so
// that a lane stores 8 consecutive channels, 16 bytes, at a time.  `dst` is the lane's row or null; `rest` its row of rests or null.
template <int DT, int D, bool REST = false>
__device__ __forceinline__ void store_cols(const f32x16& acc, int o, float factor, uint16_t* dst, int lane, uint8_t* rest = nullptr) {
  const int h = lane >> 5;
#pragma unroll
  for (int g = 0; g < 4; g += 2) {
    if (D % 32 != 0 && 32 * o + 8 * g >= D) continue;
    float x[8];
    uint32_t a[4];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = acc[4 * g + u] * factor;
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = pack2<DT>(x[2 * u], x[2 * u + 1]);
    if constexpr (REST) {
      uint32_t r[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        r[u] = pack_rest(rest_of<DT>(x[4 * u], Elem<DT>::load(a[2 * u] & 0xffffu)), rest_of<DT>(x[4 * u + 1], Elem<DT>::load(a[2 * u] >> 16)),
                         rest_of<DT>(x[4 * u + 2], Elem<DT>::load(a[2 * u + 1] & 0xffffu)), rest_of<DT>(x[4 * u + 3], Elem<DT>::load(a[2 * u + 1] >> 16)));
      const auto y = __builtin_amdgcn_permlane32_swap(r[0], r[1], false, false);
      if (rest != nullptr) *reinterpret_cast<u32x2*>(rest + 32 * o + 8 * (g + h)) = u32x2{y[0], y[1]};
    }
    u32x4 v;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto r = __builtin_amdgcn_permlane32_swap(a[u], a[2 + u], false, false);
      v[u] = r[0];
      v[2 + u] = r[1];
    }
    if (dst != nullptr) *reinterpret_cast<u32x4*>(dst + 32 * o + 8 * (g + h)) = v;
  }
}
template <int DT, int D, bool REST = false>
__device__ __forceinline__ void store_row(const f32x16* acc, float factor, uint16_t* dst, int lane, uint8_t* rest = nullptr) {
#pragma unroll
  for (int o = 0; o < AttnTile<D>::kOut; ++o) store_cols<DT, D, REST>(acc[o], o, factor, dst, lane, rest);
}
// The same to a row of fp32 sums.
template <int D>
__device__ __forceinline__ void store_sums(const f32x16& acc, int o, float* dst, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (D % 32 == 0 || 32 * o + 8 * g < D) *reinterpret_cast<float4*>(dst + 32 * o + 8 * g + 4 * (lane >> 5)) = float4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
}

// ---- Sums that are not numbers.  A product over a tile multiplies what a row does not see by zero, which is NaN for values that are not
// finite.  Rows (keys) whose sums come out NaN are made again behind the others' stores, a wavefront for itself and 32 channels, 32 keys (rows)
// at a time, from operands that it gets straight from memory: values that are not finite are left out of the products, and added where
// they are seen.  16 rows of 912 causal tokens of 16 / 2 heads of 128, forward / backward: 75 / 320 us, with a NaN token in each row 77 / 316, with NaN
// in one channel of one value 710 / 480, as one row's gradient 76 / 1250, as all gradients 75 / 300 (in plain loops over rows and keys 4
// rows took 4 to 18 ms where they take 0.2).

// A 16-bit operand's 8 values with those that are not finite as zeros, and which those are, a bit each.
struct Odd {
  uint32_t nan = 0, plus = 0, minus = 0;
};
template <int DT>
__device__ __forceinline__ u32x4 finite8(const uint32_t (&x)[8], Odd& odd) {
  constexpr uint32_t kTop = DT == WX_BF16 ? 0x7f80u : 0x7c00u;
  uint32_t y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool is = (x[j] & kTop) == kTop, inf = (x[j] & 0x7fffu) == kTop;
    y[j] = is ? 0u : x[j];
    odd.nan |= is && !inf ? 1u << j : 0u;
    odd.plus |= inf && !(x[j] & 0x8000u) ? 1u << j : 0u;
    odd.minus |= inf && (x[j] & 0x8000u) ? 1u << j : 0u;
  }
  return u32x4{y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16};
}
// Ones where `bits` has its first 8 bits set.
template <int DT>
__device__ __forceinline__ u32x4 ones8(uint32_t bits) {
  constexpr uint32_t kOne = DT == WX_BF16 ? 0x3f80u : 0x3c00u;
  u32x4 v;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = (bits >> (2 * u) & 1u) * kOne | (bits >> (2 * u + 1) & 1u) * (kOne << 16);
  return v;
}
// Adds to the sums what finite8 left out of step t: `seen` and `zero` have a bit for each of the column's 16 registers, what it sees and
// what it sees with a factor of zero (then an infinity gives NaN).
template <int DT>
__device__ __forceinline__ void add_odd(f32x16& acc, const Odd& odd, uint32_t seen, uint32_t zero, int t) {
  if (!__any((odd.nan | odd.plus | odd.minus) != 0)) return;
  const f32x16 none = {};
  f32x16 x = mfma<DT>(ones8<DT>(odd.nan), ones8<DT>(seen >> (8 * t)), none);
  x = mfma<DT>(ones8<DT>(odd.plus | odd.minus), ones8<DT>(zero >> (8 * t)), x);
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] += x[r] > 0.f ? __builtin_nanf("") : 0.f;
#pragma unroll
  for (int sign = 0; sign < 2; ++sign) {
    x = mfma<DT>(ones8<DT>(sign ? odd.minus : odd.plus), ones8<DT>((seen & ~zero) >> (8 * t)), none);
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += x[r] > 0.f ? (sign ? -kInf : kInf) : 0.f;
  }
}
// The A operand over rows, of which `at(i)` is the 16-bit value of this lane's channel in row i of 32, in read_cols' order.
template <int DT, class At>
__device__ __forceinline__ u32x4 gather_cols(int t, int h, Odd& odd, At at) {
  uint32_t x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = at(16 * t + 8 * (j / 4) + 4 * h + j % 4);
  return finite8<DT>(x, odd);
}
// Whether one of a lane's sums is NaN (or, with INF, not finite).  (One comparison tells of two values.)
template <int D, bool INF = false>
__device__ __forceinline__ bool not_numbers(const f32x16* acc) {
  bool bad = false;
  float top = 0.f;
#pragma unroll
  for (int o = 0; o < AttnTile<D>::kOut; ++o)
#pragma unroll
    for (int r = 0; r < 16; r += 2)
      if (32 * o + 8 * (r / 4) < D) {
        bad = bad | __builtin_isunordered(acc[o][r], acc[o][r + 1]);
        if constexpr (INF) top = fmaxf(top, fmaxf(fabsf(acc[o][r]), fabsf(acc[o][r + 1])));
      }
  return bad || top == kInf;
}
// Which of the wavefront's 32 columns a predicate of its lanes holds for, in either half.
__device__ __forceinline__ uint32_t columns(bool x) {
  const uint64_t b = __ballot(x);
  return static_cast<uint32_t>(b | b >> 32);
}

// acc + the products of two pairs of 16-bit values, in fp32
template <int DT>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float acc) {
  if constexpr (DT == WX_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(att_bf16x2, a), __builtin_bit_cast(att_bf16x2, b), acc, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(att_f16x2, a), __builtin_bit_cast(att_f16x2, b), acc, false);
}
// two e5m2 values to two of the compute type (exact)
template <int DT, bool HI>
__device__ __forceinline__ uint32_t widen_rest2(uint32_t x) {
  if constexpr (DT == WX_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x, 1.0f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(x, 1.0f, HI));
}

}  // namespace wx
