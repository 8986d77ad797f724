// How paged attention's work is spread over the chip: the arithmetic by which the host sizes the launch and every workgroup finds its share of it
// (paged_attention.hip).  Plain C++: lane exchanges and memory are the kernel's, a reciprocal and a division by the group its arguments'.
//
// Items.  A (request, key / value head, tile of rows) is an item; rows are (query, head of the group) pairs as in attention.h.  Requests of up
// to 64 rows (single tokens, drafts) are one item a head, others tiles of 128 rows.  Every item has a measure, what it takes in keys: the
// keys that it sees and some for its start.  The launch has a fixed number of shares, two workgroups to a CU; each finds the sum of all
// measures for itself (a prefix sum over the requests) and takes an equal share of it, wherever in an item that begins or ends.  An item that lies
// in one share is finished there; of one that is cut every share leaves a part in a place of its own, 2 id + 1 of the item that begins in
// share id and 2 id of the one that began before it, which a second launch joins, in order.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define WX_PLAN __device__ __forceinline__
#else
#include <algorithm>
#define WX_PLAN inline
#endif

namespace wx {
namespace paged {

#ifndef __HIPCC__
using std::max;
using std::min;
#endif

constexpr int kFewLog = 6, kManyLog = 7, kFewRows = 1 << kFewLog, kManyRows = 1 << kManyLog;  // rows of an item of either kind
constexpr int kCut = 64;  // items are cut at multiples of so many keys
// What an item takes besides its keys, in keys: about 4.5 us where 64 keys take 1.2 to 2.5.  With 64 / 192 and 128: 64 single tokens over 800 to 912
// keys 23.5 / 22.0 us, 16 prompts of 912 tokens 123 / 111 (the items at a prompt's beginning are short).
constexpr int kStartFew = 192, kStartMany = 128;
// The least that a workgroup takes.  With 256 / 512 / 1024: 64 single tokens over 800 to 912 keys 35 / 39 / 48 us (when starts took longer).
constexpr int kLeast = 256;
// Tiles of few rows for everything where no request has more keys than this and either every item gets a like number of workgroups (see share_of()) or there
// are a quarter as many items as workgroups.  64 x 32 queries over 800 to 912 keys 45 us in tiles of many rows, 35 so; 512 queries over 2012 keys 44 and 40; but
// 2048 queries over themselves 53 and 59 (bf16 keys: 47 and 60), 2 x 1000 over 2000 43 and 47, 4 x 500 37 and 40, 2048 over 16384 keys 324 and 390.
constexpr int kShort = 2048;
// An item's end near to a share's end is the share's end: nearer than this in keys, which is about what a cut costs (a start, a part, its
// join), and than 3/8 of a share.  With 128 / 320: 64 mixed requests 64 / 67 us.  Items of up to half a share are not cut at all: 16 prompts of 912
// tokens 113 -> 100 us.
constexpr int kSnap = 128;
// What an e4m3 key takes of a tile of many rows, in those of few rows, which take their bytes' time; 16-bit keys take the same.  With 1 / 2 / 3, 62 single tokens
// and two chunks of 509: heads of 64 in fp16 59 / 53 / 54 us, of 128 in bf16 77 / 66 / 70, of 8 heads of their own with chunks of 200 55 / 44 / 43;
// 30 tokens over 8 to 16 thousand keys with two chunks of 128 96 / 90 / 91.  Of a bf16 cache 74 / 75 / 86, the long one 105 / 116 / 120.
constexpr float kManyToFew = 2.f;

constexpr int kMostMeasure = 0x3fffffff, kMostHigh = kMostMeasure >> 8;  // of all requests together (`shift` is chosen so)

// ---- the host's part
struct Launch {
  int shift;   // measures are in 2^shift keys, so that the sum of all fits 31 bits; 30: no such number
  int blocks;  // workgroups: the shares, and more where each may take an item
};
inline Launch launch_of(int64_t tokens, int group, int n_kv, int64_t requests, int64_t seq, int64_t most_keys, bool has_starts, int shares) {
  Launch l{0, shares};
  const int64_t rows = tokens * group, tiles = n_kv * (rows / kFewRows + requests);
  const int64_t keys = (most_keys > tokens ? most_keys : tokens) + 2 * kManyRows;
  if (tiles > kMostMeasure / (kStartFew + kStartMany)) l.shift = 30;  // (none will do, and the product below could pass 63 bits)
  while (l.shift < 30 && tiles * ((keys >> l.shift) + kStartFew + kStartMany) > kMostMeasure) ++l.shift;
  // Room for an item of many rows to a workgroup (see share_of()), where there may be so many; of more than four to a share (eight where the plan is a
  // wavefront's) the shares are as good, and a plan over more than 256 requests is too long to be made for an item: 1024 requests of 64 tokens 280 us so, 167 in shares.
  const int64_t at_least = rows / (kFewRows + 1), long_ones = has_starts ? (requests < at_least ? requests : at_least) : (seq * group > kFewRows ? requests : 0);
  const int64_t items = long_ones ? n_kv * (rows / kManyRows + long_ones) : 0;  // at most
  if (2 * items >= 3 * shares && requests <= 256) {
    const int64_t wide = (items + 7) / 8 * 8 + shares, most = static_cast<int64_t>(requests <= 64 ? 8 : 4) * shares;
    l.blocks = static_cast<int>(wide < most ? wide : most);
  }
  return l;
}

// ---- requests and their items.  A: lengths, starts (or null), tokens, seq, most_keys (to a request), group, by_group, n_kv, causal, shift, shares.
struct Request {
  int first, n, length;  // tokens first .. first + n - 1, `length` keys
  int rows;              // n * group
};
template <class A>
WX_PLAN Request request(const A& a, int r) {
  Request q;
  if (a.starts != nullptr) {
    q.first = min(max(a.starts[r], 0), a.tokens);
    q.n = min(max(a.starts[r + 1], q.first), a.tokens) - q.first;
  } else {
    q.first = r * a.seq, q.n = a.seq;
  }
  q.length = min(max(a.lengths[r], 0), a.most_keys);
  q.rows = q.n * a.group;
  return q;
}
// keys that the last of the rows up to `row` sees
template <class A>
WX_PLAN int keys_seen(const A& a, const Request& q, int row) {
  return a.causal ? min(max(q.length - q.n + a.by_group.div(row) + 1, 0), q.length) : q.length;
}
// Which requests: those of few rows, those of many, or all of them in tiles of few rows.
enum Kind { kFew, kMany, kAllFew };
// The items of one head of a request: tile t's measure is base + step (t + 1), which follows the diagonal.
struct Ramp {
  int base, step, tiles;
  WX_PLAN int before(int t) const { return t * base + static_cast<int>(step * (static_cast<int64_t>(t) * (t + 1) / 2)); }
  WX_PLAN int of(int t) const { return base + step * (t + 1); }
};
template <class A>
WX_PLAN int start_of(const A& a, bool few) { return max((few ? kStartFew : kStartMany) >> a.shift, 1); }
template <class A>
WX_PLAN Ramp ramp(const A& a, const Request& q, bool few) {
  const int log = few ? kFewLog : kManyLog, rows = 1 << log, tiles = (q.rows + rows - 1) >> log;
  const int step = a.causal && tiles > 1 ? a.by_group.div(rows) >> a.shift : 0;
  return {((step ? max(q.length - q.n, 0) : q.length) >> a.shift) + start_of(a, few), step, tiles};
}
// measure of one head of a request
template <class A>
WX_PLAN int measure(const A& a, const Request& q, int kind) {
  if (q.n == 0 || (kind != kAllFew && (q.rows <= kFewRows) != (kind == kFew))) return 0;
  const Ramp p = ramp(a, q, kind != kMany);
  return p.before(p.tiles);
}
WX_PLAN int tiles_of(const Request& q, bool few) {
  return few ? (q.rows + kFewRows - 1) >> kFewLog : (q.rows > kFewRows ? (q.rows + kManyRows - 1) >> kManyLog : 0);
}

// ---- sums over the requests: measures of each Kind, numbers of items of few rows (all requests') and of many (such requests'), and of the greater of a
// request's measures in few rows and in many (whose steps are rounded each for itself) a sum in 256ths that stays in range whatever starts hold; beside them
// the longest request
enum { kFewItems = 3, kManyItems, kHigh, kSums };
template <class A>
WX_PLAN void add_request(const A& a, const Request& q, int (&sums)[kSums], int& longest) {
  const bool few = q.rows <= kFewRows;
  const int m = measure(a, q, kAllFew) * a.n_kv, many = few ? 0 : measure(a, q, kMany) * a.n_kv;
  sums[kFew] += few ? m : 0;
  sums[kMany] += many;
  sums[kAllFew] += m;
  sums[kHigh] = min(sums[kHigh] + (max(m, many) >> 8), kMostHigh + 1);
  sums[kFewItems] += tiles_of(q, true) * a.n_kv;
  sums[kManyItems] += tiles_of(q, false) * a.n_kv;
  longest = max(longest, q.n == 0 ? 0 : q.length);
}

// ---- a workgroup's share: `size` of its kind's measures, from `x` into tile `tile` of `head` of request r; or part x of that item.
struct Share {
  int kind, id;    // id: below the launch's shares, unique over all kinds, wherever an item is cut
  int parts;       // not 0: every item is cut in so many parts, a share each
  int size, each;  // size 0: nothing; each: what a share of this kind takes
  int at, end;     // where in the requests' sums (see of_share()) it begins, and where it ends if another follows; -1: nowhere
  int r, head, tile, x;
  Request q;
};
// the sum that a share is in
WX_PLAN int of_share(const Share& s, const int (&sums)[kSums]) {
  if (s.parts) return s.kind != kMany ? sums[kFewItems] : sums[kManyItems];
  return s.kind == kAllFew ? sums[kAllFew] : (s.kind == kFew ? sums[kFew] : sums[kMany]);
}
// (quotients of whole numbers by way of floats, which take a tenth of an exact division's instructions; exact where both are below 1024: off by
// less than 1 / 1024 then, and so far from the next whole number)
template <class A>
WX_PLAN int quotient(const A& a, int x, int y) { return static_cast<int>(static_cast<float>(x) * a.reciprocal(static_cast<float>(y)) + 0x1p-11f); }
// (a little more than total / count)
template <class A>
WX_PLAN int each_of(const A& a, int total, int count) {
  return max(static_cast<int>(static_cast<float>(total) * a.reciprocal(static_cast<float>(count)) * 1.000001f) + 2, kLeast >> a.shift);
}
template <bool F8, class A>
WX_PLAN Share share_of(const A& a, int block, int blocks, const int (&all)[kSums], int longest) {
  Share s = {};
  s.end = -1;
  const int xcd = block & 7, j = block >> 3, per_xcd = a.shares / 8;
  if (all[kHigh] > kMostHigh) {  // (only of starts that do not ascend, whose requests overlap)
    s.id = block, s.at = -1;
    return s;
  }
  // Items of about one length, no more than there are workgroups: a like number of workgroups to each, without second items, where the longest
  // one's parts are no longer than shares are.  64 single tokens over 800 to 912 keys 22.1 -> 20.6 us.
  const int each_few = each_of(a, all[kAllFew], a.shares);
  int parts = 0;
  if (all[kFewItems] > 0 && all[kFewItems] <= a.shares) {
    parts = min(quotient(a, a.shares, all[kFewItems]), max((longest + kLeast - 1) / kLeast, 1));
    if (longest >> a.shift > static_cast<int64_t>(each_few) * parts) parts = 0;
  }
  const bool all_few = all[kMany] == 0 || (longest <= kShort && (parts != 0 || 4 * all[kFewItems] <= a.shares));
  // the kinds' workgroups, a like number of each on every XCD, neighbouring shares on the same
  int p = all_few ? per_xcd : 0;
  if (!all_few && all[kFew] != 0) {
    const float part = static_cast<float>(all[kFew]) / (static_cast<float>(all[kFew]) + (F8 ? kManyToFew : 1.f) * static_cast<float>(all[kMany]));
    p = a.uniform(min(max(static_cast<int>(part * per_xcd + 0.5f), 1), per_xcd - 1));
  }
  s.kind = all_few ? kAllFew : (j < p ? kFew : kMany);
  const int count = j < p ? 8 * p : 8 * (per_xcd - p);
  int w = j < p ? xcd * p + j : xcd * (per_xcd - p) + j - p;
  s.id = j < p ? w : 8 * p + w;
  const int total = of_share(s, all);
  s.each = a.uniform(all_few ? each_few : each_of(a, total, count));
  if (all_few) s.parts = a.uniform(parts);
  // Many items of many rows, three and more to two shares: a workgroup for each instead, where the launch has as many (an XCD has neighbouring ones), long
  // ones of a request first.  Which of the chip's places takes the next is found as they end: 16 prompts of 912 tokens 105 -> 97 us, 8 of them 68 -> 48;
  // from one to a share on 6 prompts 57 and 50, but 5 of 1000 behind as many 103 and 121.
  const int each_xcd = (all[kManyItems] + 7) / 8;
  bool none = false;
  if (s.kind == kMany && 2 * all[kManyItems] >= 3 * count && each_xcd <= (blocks >> 3) - p) {
    s.parts = 1;
    w = j - p < each_xcd ? xcd * each_xcd + j - p : all[kManyItems];
  } else {
    // The launch is wider than the shares for the sake of the items: of everything else, equal parts among it, the workgroups beyond the shares have
    // nothing.  (The host knows what room there is for tokens, not how many there are.)
    none = j >= per_xcd;
  }
  if (s.parts) {
    const int item = s.parts == 1 ? w : quotient(a, w, s.parts);
    s.x = w - item * s.parts;
    s.size = !none && item < of_share(s, all);
    s.at = item;
  } else {
    const int64_t at = static_cast<int64_t>(w) * s.each;
    s.size = !none && at < total ? min(total - static_cast<int>(at), s.each) : 0;
    s.at = s.size > 0 ? static_cast<int>(at) : -1, s.end = s.size == s.each ? s.at + s.each : -1;
  }
  return s;
}

// Where `at` of a request's measure lies, moved to an item's end if that is near.  Returns by how much it was moved.
struct Place {
  int head, tile, x;
};
template <class A>
WX_PLAN int snap_of(const A& a, int of_item, int each) {  // (at least 1: a share's end that is the item's own is no cut in it)
  const int most = each / 8 * 3;
  return max(2 * of_item <= each ? most : min(most, kSnap >> a.shift), 1);
}
template <class A>
WX_PLAN int locate(const A& a, const Request& q, int kind, int at, int each, Place& p) {
  const Ramp items = ramp(a, q, kind != kMany);
  const int of_head = items.before(items.tiles);
  p.head = at / of_head;
  p.x = at - p.head * of_head;
  int lo = 0, hi = items.tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (items.before(mid) <= p.x) lo = mid;
    else hi = mid - 1;
  }
  p.tile = lo;
  p.x -= items.before(lo);
  const int of_item = items.of(lo), snap = snap_of(a, of_item, each), to = p.x < snap ? 0 : (of_item - p.x < snap ? of_item : p.x), moved = to - p.x;
  p.x = to;
  return moved;
}
// What request q has of the sum that a share is in, and, `at` into that, the share's first item.  Returns by how much its begin was moved.
template <class A>
WX_PLAN int extent(const A& a, const Share& s, const Request& q) { return s.parts ? tiles_of(q, s.kind != kMany) * a.n_kv : measure(a, q, s.kind) * a.n_kv; }
template <class A>
WX_PLAN int begin_of(const A& a, const Share& s, const Request& q, int at, Place& p) {
  if (!s.parts) return locate(a, q, s.kind, at, s.each, p);
  const int tiles = tiles_of(q, s.kind != kMany);
  p.head = at / tiles, p.tile = tiles - 1 - (at - p.head * tiles);
  return 0;
}

// ---- a share's segments: rows row0 .. row0 + rows - 1 of a request over the keys lo .. hi - 1.
struct Segment {
  Request q;
  int r, head, row0, rows, lo, hi;
  bool whole;  // all of its item: the result itself
  int slot;    // otherwise its part's place
};
struct Part {  // of the item that begins in a share and ends in a later one
  int parts;   // 0: there is none
  int head;    // key / value head
  int first;   // the request's first token
  int row0, rows;
};  // (no arrays in it: they are put into LDS, at an address made from the dispatch packet, which lies in host memory: 12 us)

// run(few, segment) for each of them, in order; next(r, kind) is the next request of a kind from r on, -1 if there is none.
template <class A, class Next, class Run>
WX_PLAN Part segments(const A& a, const Share& s, Next next, Run run) {
  Part part = {};
  const bool few = s.kind != kMany;
  const int tile_rows = few ? kFewRows : kManyRows;
  int left = s.size, x = s.x, t = s.tile;
  Segment g;
  g.r = s.r, g.q = s.q, g.head = s.head;
  while (left > 0) {
    const Ramp items = ramp(a, g.q, few);
    for (; left > 0 && g.head < a.n_kv; ++g.head, t = 0)
      for (; left > 0 && t < items.tiles; ++t, x = 0) {
        g.row0 = t * tile_rows;
        g.rows = min(g.q.rows - g.row0, tile_rows);
        const int seen = keys_seen(a, g.q, g.row0 + g.rows - 1);
        int parts = s.parts, take = 1;
        if (s.parts) {
          const float each = static_cast<float>(seen) * (1.f / kCut) * a.reciprocal(static_cast<float>(s.parts));
          auto cut = [&](int i) { return i == s.parts ? seen : min(seen, static_cast<int>(each * static_cast<float>(i)) * kCut); };
          g.lo = cut(x), g.hi = cut(x + 1);
        } else {
          const int of_item = items.of(t), start = start_of(a, few);
          take = min(of_item - x, left);
          if (take <= 0) continue;  // (a share that begins at an item's end)
          auto cut = [&](int at) {
            if (at >= of_item) return seen;
            const int64_t key = static_cast<int64_t>(max(at - start, 0)) << a.shift;
            return key < seen ? static_cast<int>(key) / kCut * kCut : seen;
          };
          g.lo = cut(x), g.hi = cut(x + take);
          // (the shares' ends behind this one that are inside of the item and not near its end)
          parts = take == of_item ? 1 : 2 + (of_item - snap_of(a, of_item, s.each) - take) / s.each;
        }
        g.whole = parts == 1;
        g.slot = 2 * s.id + (x == 0);
        if (x == 0 && parts > 1) part.parts = parts, part.head = g.head, part.first = g.q.first, part.row0 = g.row0, part.rows = g.rows;
        run(few, g);
        left -= take;
      }
    if (left <= 0) break;
    g.r = next(g.r + 1, s.kind), g.head = 0;
    if (g.r < 0) break;
    g.q = request(a, g.r);
  }
  return part;
}

}  // namespace paged
}  // namespace wx
