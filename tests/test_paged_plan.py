"""Paged attention's schedule, without a GPU: the header by which every workgroup finds its share of the work, compiled for the CPU and run for all
workgroups of a launch.  Every item is covered once and in order, whole or in parts; parts have places of their own inside of the workspace and are
where the join looks for them; nothing is done twice, whatever room the call has beyond its requests' tokens."""

import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wall-x_amd", "csrc")
PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <tuple>
#include <vector>
#include "paged_plan.h"
using namespace wx::paged;

struct Args {
  const int *lengths, *starts;
  int tokens, seq, most_keys, group, n_kv, causal, shift, shares, requests, way;
  struct By { int d; int div(int n) const { return n / d; } } by_group;
  // the machine's reciprocal is within a unit of the last place: to nearest, the one above and the one below
  float reciprocal(float x) const { return way == 0 ? 1.f / x : std::nextafterf(1.f / x, way > 0 ? 1e30f : -1e30f); }
  int uniform(int x) const { return x; }
};

#define NEED(c, ...) do { if (!(c)) { std::printf("FAILED %s: ", #c); std::printf(__VA_ARGS__); std::printf("\n"); return 1; } } while (0)

// tokens seq requests most_keys group n_kv causal has_starts shares f8 way, then the lengths and (has_starts) the starts; prints
// "launched working cut" of a call in order
int one(bool f8, Args& a, bool has_starts) {
  const Launch l = launch_of(a.tokens, a.group, a.n_kv, a.requests, a.seq, a.most_keys, has_starts, a.shares);
  NEED(l.shift < 30 && l.blocks >= a.shares && l.blocks % 8 == 0, "%d %d", l.shift, l.blocks);
  a.shift = l.shift;
  int all[kSums] = {}, longest = 0;
  std::vector<Request> of(a.requests);
  for (int r = 0; r < a.requests; ++r) of[r] = request(a, r), add_request(a, of[r], all, longest);
  std::vector<Part> parts(a.shares);
  std::vector<int> written(a.shares), used(2 * a.shares);
  struct Piece { int lo, hi, row0, rows, whole, id, slot; };
  std::map<std::tuple<int, int, int>, std::vector<Piece>> items;  // (request, head, first row)
  int working = 0, cut = 0;
  for (int b = 0; b < l.blocks; ++b) {
    Share s = f8 ? share_of<true>(a, b, l.blocks, all, longest) : share_of<false>(a, b, l.blocks, all, longest);
    int moved[2] = {0, 0}, before = 0, found = 0;
    Place place = {}, other;
    for (int r = 0; s.size > 0 && r < a.requests; ++r) {
      const int m = extent(a, s, of[r]);
      if (before <= s.at && s.at < before + m) moved[0] = begin_of(a, s, of[r], s.at - before, place), s.r = r, s.q = of[r], ++found;
      if (before <= s.end && s.end < before + m) moved[1] = locate(a, of[r], s.kind, s.end - before, s.each, other);
      before += m;
    }
    NEED(s.size == 0 || found == 1, "block %d: %d requests", b, found);
    s.head = place.head, s.tile = place.tile;
    if (!s.parts) s.size += s.size > 0 ? moved[1] - moved[0] : 0, s.x = place.x;
    int bad = 0, n = 0;
    const Part part = segments(a, s,
        [&](int r, int kind) { for (; r < a.requests; ++r) if (measure(a, of[r], kind)) return r; return -1; },
        [&](bool few, const Segment& g) {
          const int tile_rows = few ? kFewRows : kManyRows;
          bad |= g.rows < 1 || g.rows > tile_rows || g.row0 % tile_rows || g.row0 + g.rows > g.q.rows || g.lo < 0 || g.lo > g.hi || (g.lo % kCut && g.lo != g.hi);
          if (!g.whole) {
            if (g.slot < 0 || g.slot >= 2 * a.shares) { bad |= 2; return; }
            bad |= 4 * (used[g.slot]++ != 0);
          }
          items[{g.r, g.head, g.row0}].push_back({g.lo, g.hi, g.row0, g.rows, g.whole, s.id, g.slot});
          ++n;
        });
    NEED(!bad, "block %d of %d: %s", b, l.blocks, bad & 2 ? "a part outside of the workspace" : (bad & 4 ? "a place taken twice" : "a segment out of range"));
    working += n > 0;
    if (b < a.shares) {
      NEED(s.id >= 0 && s.id < a.shares && !written[s.id]++, "block %d has id %d", b, s.id);
      parts[s.id] = part;
    }
  }
  bool ascend = true;
  for (int r = 1; r < a.requests; ++r) ascend &= of[r].first >= of[r - 1].first + of[r - 1].n;
  if (!ascend && all[kHigh] > kMostHigh) {  // requests that overlap, with more work than any others can ask for: nothing is done
    for (const Part& p : parts) NEED(p.parts == 0, "parts of nothing");
    NEED(items.empty(), "some of it is done");
    std::printf("%d %d 0\n", l.blocks, working);
    return 0;
  }
  NEED(all[kHigh] <= kMostHigh, "too much work");
  // every item, once and in order; parts where the join reads them
  std::vector<int> joined(a.shares);
  for (int r = 0; r < a.requests; ++r) {
    const Request& q = of[r];
    for (int h = 0; h < a.n_kv; ++h)
      for (int row = 0; row < q.rows;) {
        auto it = items.find({r, h, row});
        NEED(it != items.end(), "request %d head %d row %d is nobody's", r, h, row);
        const std::vector<Piece>& v = it->second;
        const int rows = v[0].rows, last = row + rows - 1;
        NEED(rows == std::min(q.rows - row, kFewRows) || rows == std::min(q.rows - row, kManyRows), "%d rows", rows);
        const int seen = a.causal ? std::max(0, std::min(q.length, q.length - q.n + last / a.group + 1)) : q.length;
        NEED((v.size() == 1) == (v[0].whole != 0), "request %d head %d row %d: %zu pieces", r, h, row, v.size());
        std::map<int, Piece> by_id;
        for (const Piece& p : v) {
          NEED(p.rows == rows && (v.size() == 1 || !p.whole), "pieces differ");
          NEED(by_id.emplace(p.id, p).second, "request %d head %d row %d twice in a share", r, h, row);
        }
        int key = 0, i = 0;
        const int id = by_id.begin()->first;
        for (const auto& [at, p] : by_id) {
          NEED(p.lo == key && at == id + i, "request %d head %d row %d: keys %d .. %d after %d", r, h, row, p.lo, p.hi, key);
          if (!p.whole) NEED(p.slot == (i == 0 ? 2 * id + 1 : 2 * at), "slot %d of share %d", p.slot, at);
          key = p.hi, ++i;
        }
        NEED(key == seen, "request %d head %d row %d: %d of %d keys", r, h, row, key, seen);
        if (v.size() > 1) {
          const Part& p = parts[id];
          NEED(p.parts == static_cast<int>(v.size()) && p.head == h && p.first == q.first && p.row0 == row && p.rows == rows, "request %d head %d row %d: its part has %d of %zu",
               r, h, row, p.parts, v.size());
          joined[id] = 1, ++cut;
        }
        items.erase(it);
        row += rows;
      }
  }
  NEED(items.empty(), "items of no request");
  for (int i = 0; i < a.shares; ++i) NEED((parts[i].parts != 0) == (joined[i] != 0), "share %d has parts of nothing", i);
  std::printf("%d %d %d\n", l.blocks, working, cut);
  return 0;
}

int main() {
  Args a = {};
  int has_starts, f8;
  while (std::scanf("%d %d %d %d %d %d %d %d %d %d %d", &a.tokens, &a.seq, &a.requests, &a.most_keys, &a.group, &a.n_kv, &a.causal, &has_starts, &a.shares, &f8, &a.way) == 11) {
    std::vector<int> lengths(a.requests + 1), starts(a.requests + 1);
    for (int r = 0; r < a.requests; ++r) if (std::scanf("%d", &lengths[r]) != 1) return 1;
    for (int r = 0; has_starts && r <= a.requests; ++r) if (std::scanf("%d", &starts[r]) != 1) return 1;
    a.lengths = lengths.data(), a.starts = has_starts ? starts.data() : nullptr, a.by_group.d = a.group;
    if (int rc = one(f8, a, has_starts)) return rc;
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    folder = tmp_path_factory.mktemp("plan")
    source, program = folder / "plan.cpp", folder / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-Wall", "-Werror", f"-I{CSRC}", str(source), "-o", str(program)], check=True)

    def run(cases):
        """(workgroups launched, with work, items cut) of each case (tokens, seq, group, Hkv, causal, starts or None, lengths, most keys of a request, shares, e4m3, way)."""
        lines = []
        for tokens, seq, group, n_kv, causal, starts, lengths, most_keys, shares, f8, way in cases:
            lines.append(" ".join(map(str, [tokens, seq, len(lengths), most_keys, group, n_kv, int(causal), int(starts is not None), shares, int(f8), way, *lengths, *(starts or [])])))
        done = subprocess.run([str(program)], input="\n".join(lines), capture_output=True, text=True)
        out = done.stdout.splitlines()
        assert done.returncode == 0, (out[-1], cases[len(out) - 1])
        assert len(out) == len(cases)
        return [tuple(map(int, line.split())) for line in out]

    return run


def packed(counts, lengths, room, front=0, group=8, n_kv=2, causal=True, most_keys=None, shares=512, f8=True, way=0):
    starts = [front]
    for n in counts:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + room
    return tokens, tokens, group, n_kv, causal, starts, lengths, most_keys or max([1, *lengths]), shares, f8, way


@pytest.mark.parametrize("way", [-1, 0, 1])
def test_a_step_in_a_wide_buffer(plan, way):
    """Few tokens where the call has room for prompts: the launch is wide for items that are not there."""
    cases = [packed([1] * 16, [912] * 16, 15 * 912, way=way), packed([1] * 64, [900] * 64, 8192 - 64, way=way), packed([1] * 64, [912] * 64, 5120 - 64, way=way),
             packed([1] * 32, [500] * 32, 1024 - 32, group=8, n_kv=8, way=way), packed([3, 5, 1, 0] * 8, [700] * 32, 16 * 912, way=way),
             packed([32] * 64, [880] * 64, 64 * 200, causal=False, way=way), packed([1] * 63 + [600], [4000] * 64, 16000, way=way),
             packed([1] * 30, [40000] * 30, 60000, way=way), packed([1] * 200, [300] * 200, 30000, way=way), packed([0] * 16, [912] * 16, 16 * 912, way=way)]
    for launched, working, _ in plan(cases):
        assert launched > 512 and working <= 512


def random_case(rng, widths=(None, 77)):
    R = int(2 ** rng.uniform(0, 8.5))
    kind = rng.choice(["steps", "drafts", "denoise", "chunks", "mixed", "any"])
    most = int(2 ** rng.uniform(0, 15))
    some = {"steps": lambda: 1, "drafts": lambda: rng.randint(0, 8), "denoise": lambda: 32, "chunks": lambda: int(2 ** rng.uniform(0, 10)),
            "mixed": lambda: rng.choice([1, 1, 1, 1, 1, 300]), "any": lambda: rng.choice([0, 1, int(2 ** rng.uniform(0, 9))])}[kind]
    counts = [some() for _ in range(R)]
    near = rng.random() < 0.5  # of about one length
    lengths = [max(0, (rng.randint(most - most // 8, most) if near else rng.randint(0, most)) + (n if rng.random() < 0.9 else -n // 2)) for n in counts]
    room = rng.choice([0, 5, int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(10, 16))])
    wide = rng.choice(widths)
    case = packed(counts, lengths, room, rng.choice([0, 0, 9]), rng.choice([1, 2, 3, 4, 7, 8, 24]), rng.choice([1, 2, 4, 8]), rng.random() < 0.7,
                  None if wide is None else max([1, *lengths]) + wide, rng.choice([512, 512, 512, 608, 128, 64]), rng.random() < 0.5, rng.choice([-1, 0, 1]))
    if rng.random() < 0.2:  # rows of q are requests
        n = counts[0] or 1
        case = (n * R, n, *case[2:5], None, *case[6:])
    return case


@pytest.mark.parametrize("seed", range(6))
def test_schedules(plan, seed):
    rng = random.Random(seed)
    cases = [random_case(rng) for _ in range(500)]
    done = plan(cases)
    assert sum(launched > case[8] for (launched, _, _), case in zip(done, cases)) > 50 and sum(cut > 0 for *_, cut in done) > 100


@pytest.mark.parametrize("seed", range(6))
def test_schedules_of_wide_tables(plan, seed):
    """Tables that could hold so many keys that measures are in hundreds of them, and a cut may fall on an item's end to the key."""
    rng = random.Random(100 + seed)
    done = plan([random_case(rng, (2 ** 20, 2 ** 25, 2 ** 28, 2 ** 30 - 2 ** 17)) for _ in range(300)])
    assert sum(cut > 0 for *_, cut in done) > 50


def test_schedules_of_many_query_heads_to_a_key_head(plan):
    """Rows of one query in several tiles; a diagonal that tiles are too short to count."""
    rng = random.Random(300)
    cases = []
    for _ in range(300):
        counts = [rng.choice([0, 1, 1, 2, 5]) for _ in range(rng.randint(1, 12))]
        lengths = [n + int(2 ** rng.uniform(0, 14)) for n in counts]
        cases.append(packed(counts, lengths, rng.choice([0, 3, 200]), 0, rng.choice([65, 100, 130, 1024]), rng.choice([1, 2]), rng.random() < 0.7, None, 512, rng.random() < 0.5, rng.choice([-1, 0, 1])))
    plan(cases)


def overlapping(rng, case):
    """Starts that do not ascend, or lie outside of the tokens."""
    return (*case[:5], [rng.randint(-5, case[0] + 5) for _ in range(len(case[6]) + 1)], *case[6:])


@pytest.mark.parametrize("seed", range(6))
def test_schedules_of_starts_that_descend(plan, seed):
    """Requests that claim the same tokens: each has its items all the same, or none has any."""
    rng = random.Random(200 + seed)
    done = plan([overlapping(rng, random_case(rng, (None, 77, 2 ** 25))) for _ in range(100)])
    assert sum(working > 0 for _, working, _ in done) > 40


def test_more_work_in_tiles_of_many_rows_than_of_few(plan):
    """Far more queries than keys and 24 heads to a key / value head: a diagonal that tiles of few rows are too short to count."""
    R, T = 199, 33336
    case = packed([1], [500] * R, T - 1, group=24, n_kv=8, most_keys=1518)
    assert plan([(*case[:5], [T // 50 * (r % 50) * (r % 2) for r in range(R + 1)], *case[6:])])


def test_requests_that_overlap(plan):
    """More work than requests that ascend can ask for: none of it is begun."""
    R, T = 4600, 4096
    assert plan([(T, T, 1, 1, False, [T * (r % 2) for r in range(R + 1)], [8192] * R, 8192, 512, True, 0)]) == [(512, 0, 0)]


LAUNCHES = r"""
#include <cstdio>
#include "paged_plan.h"
int main() {
  long long tokens, requests, seq, most_keys;
  int group, n_kv, has_starts;
  while (std::scanf("%lld %d %d %lld %lld %lld %d", &tokens, &group, &n_kv, &requests, &seq, &most_keys, &has_starts) == 7) {
    const wx::paged::Launch l = wx::paged::launch_of(tokens, group, n_kv, requests, seq, most_keys, has_starts, 512);
    std::printf("%d %d\n", l.shift, l.blocks);
  }
}
"""


def test_launches_of_the_largest_calls(tmp_path):
    """Measures are scaled so that all of them fit 31 bits, up to the sizes that a call is refused at and far beyond, against Python's integers."""
    (tmp_path / "launch.cpp").write_text(LAUNCHES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "launch.cpp"), "-o",
                    str(tmp_path / "launch")], check=True)
    rng = random.Random(1)
    most = 2 ** 30 - 1
    cases = [(1, 1, 64, most, 1, most, 1), (1, 1, most, most, 1, most, 1), (most, 1, 1, 1, most, most, 0), (2 ** 20, 1024, 1, 1, 2 ** 20, 1, 0), (4096, 1, 8, 3340000 // 8, 4096, 1, 1)]
    for _ in range(3000):
        n_kv, group = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 10))
        tokens = max(1, int(2 ** rng.uniform(0, 30)) // (n_kv * group))
        cases.append((tokens, group, n_kv, int(2 ** rng.uniform(0, 30)), tokens, int(2 ** rng.uniform(0, 30)), 1))
    out = subprocess.run([str(tmp_path / "launch")], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout.splitlines()
    fits = 0
    for (tokens, group, n_kv, requests, _, keys, _), line in zip(cases, out, strict=True):
        shift, blocks = map(int, line.split())
        tiles, keys = n_kv * (tokens * group // 64 + requests), max(keys, tokens) + 256
        need = next((s for s in range(30) if tiles * ((keys >> s) + 320) <= most), 30)
        assert shift == need and 512 <= blocks <= 4096, (tiles, keys, shift, need, blocks)
        fits += shift < 30
    assert 300 < fits < len(cases) - 300
