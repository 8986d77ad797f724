// How the backward's second kernel is spread over the chip: the arithmetic that its plan kernel and its host share (plain C++).
//
// Under a causal mask the first keys are seen by all rows and the last by few, and of a row of packed sequences a tile is seen by those
// of its own: a tile's blocks of 32 rows, from the first to the last that sees it, are cut evenly into units of at most as many as make a
// pair's units about `aim` in all (kLeast where that is fewer), so that the longest workgroup is a unit and not a tile.
#pragma once

#include <cstdint>

namespace wx {

constexpr int kKeyTile = 64;
constexpr int kLeast = 16;
constexpr int kPlanTiles = 1024;

// Units that a pair's key tiles are cut into beyond one to each: about kUnits workgroups to each place on the chip (two to a CU) of all
// pairs', where the tiles alone are fewer.  More units end more evenly, fewer write and join fewer sums (64 KB a unit of head size 128).
// Forward and backward with 1 / 2 / 3 / 4 / 6: 8192 causal tokens of 16 / 2 heads 1464 / 1344 / 1321 / 1339 / 1372 us, 4096 tokens of 16 / 16
// heads that see all 593 / 594 / 643 / 648 / 672, 16 rows of 912 causal tokens 379 / 384 / 404 / 413 / 442.
constexpr int kUnits = 2;
constexpr int aim_units(int64_t pairs, int64_t n_keys, int cus) {
  const int64_t tiles = pairs * ((n_keys + kKeyTile - 1) / kKeyTile), places = 2 * static_cast<int64_t>(cus);
  return tiles == 0 || tiles >= kUnits * places || tiles > pairs * kPlanTiles ? 0 : static_cast<int>((kUnits * places + pairs - 1) / pairs);
}
// No tile makes more than its rows' blocks do in units of the least length.
constexpr int more_units(int64_t pairs, int64_t rows, int64_t n_keys, int cus) {
  const int64_t of_tile = ((rows + 31) / 32 + kLeast - 1) / kLeast, most = (n_keys + kKeyTile - 1) / kKeyTile * (of_tile > 1 ? of_tile - 1 : 0);
  const int64_t aim = aim_units(pairs, n_keys, cus);
  return static_cast<int>(aim < most ? aim : most);
}

// Blocks of a unit at most, of `work` blocks of all of a pair's tiles (1024 tiles of 2^25 blocks pass 32 bits), and units of a tile of `blocks`: one
// of no blocks, which writes zeros, where nothing sees it.  Together never more than the tiles and more_units: the full units are no more
// than `aim`, the last ones of the tiles no more than those.
constexpr int unit_blocks(int64_t work, int aim) {
  const int64_t even = (work + aim - 1) / aim;
  return even > kLeast ? static_cast<int>(even) : kLeast;
}
constexpr int tile_units(int blocks, int unit) { return blocks > unit ? (blocks + unit - 1) / unit : 1; }

}  // namespace wx
