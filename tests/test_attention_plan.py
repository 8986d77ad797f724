"""The backward's plan never makes more units than its list has places, up to the largest sizes that the ops take (no GPU needed: the header
that the plan kernel and its host share, compiled for the CPU, against the plan in Python's integers)."""

import os
import random
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wall-x_amd", "csrc")
PROGRAM = """
#include <cstdio>
#include "attention_plan.h"
using namespace wx;
// a line each: pairs rows n_keys cus, then the number of tiles with work and their blocks (the same for all)
int main() {
  long long pairs, rows, n_keys, cus, seen, blocks;
  while (std::scanf("%lld %lld %lld %lld %lld %lld", &pairs, &rows, &n_keys, &cus, &seen, &blocks) == 6) {
    const int aim = aim_units(pairs, n_keys, cus), more = more_units(pairs, rows, n_keys, cus);
    if (more == 0) { std::printf("%d %d 0 0\\n", aim, more); continue; }
    const int unit = unit_blocks(static_cast<int64_t>(seen) * blocks, aim);
    std::printf("%d %d %d %d\\n", aim, more, unit, tile_units(static_cast<int>(blocks), unit));
  }
}
"""


def test_units_fit_their_list(tmp_path):
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    rng = random.Random(1)
    cases = [(1, 2 ** 30 - 1, 65472, 256), (1, 2 ** 27, 32768, 256), (3, 2 ** 29, 21000, 256), (1, 2 ** 30 - 1, 1, 256), (1, 1, 65472, 256)]
    for _ in range(3000):
        pairs, rows = int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 30))
        cases.append((pairs, rows, int(2 ** rng.uniform(0, 17)), rng.choice([1, 64, 256, 304])))
    lines = []
    for pairs, rows, n_keys, cus in cases:
        tiles, row_blocks = -(-n_keys // 64), -(-rows // 32)
        lines.append((pairs, rows, n_keys, cus, rng.choice([tiles, tiles, rng.randint(0, tiles)]), rng.choice([row_blocks, row_blocks, rng.randint(0, row_blocks)])))
    out = subprocess.run([str(program)], input="\n".join(" ".join(map(str, line)) for line in lines), capture_output=True, text=True, check=True).stdout
    planned = 0
    for (pairs, rows, n_keys, cus, seen, blocks), line in zip(lines, out.splitlines()):
        aim, more, unit, units = map(int, line.split())
        tiles = -(-n_keys // 64)
        if more == 0:
            continue
        planned += 1
        assert unit == max(16, -(-seen * blocks // aim)) and units == max(1, -(-blocks // unit))
        total = seen * units + (tiles - seen)
        assert total <= tiles + more, (pairs, rows, n_keys, cus, seen, blocks, total, tiles + more)
    assert planned > 300
