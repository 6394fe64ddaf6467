// The paged cache's index arithmetic, for the kernels and for host tests alike: plain C++, no HIP.  What it is given comes from arrays in
// device memory that nobody has checked, so everything is brought into its range first.
#pragma once
#include <stdint.h>

namespace pkh3 {

constexpr int kPageKeys = 64;
constexpr int at_most(int x, int y) { return x < y ? x : y; }
constexpr int at_least(int x, int y) { return x > y ? x : y; }

// One sequence of a batch: its rows first .. first + n - 1 of the call, its keys, the position of its first row (negative where it
// has more rows than keys).
struct Sequence {
  int first, n, keys;
  constexpr int position() const { return keys - n; }
};
constexpr Sequence make_sequence(int start, int end, int length, int rows, int table_pages) {
  const int at = at_most(at_least(start, 0), rows), to = at_most(at_least(end, 0), rows);
  return {at, at_least(to - at, 0), at_most(at_least(length, 0), table_pages * kPageKeys)};
}
// The same for writing, by the values as they are: brought into range, a row would come to another's place and take it.  Row r of the call stands at
// length - end + r; what is written are the rows whose place is in the table.  Their positions are from 0 on.
constexpr Sequence make_written(int start, int end, int length, int rows, int table_pages) {
  const int64_t row0 = (int64_t)end - length, behind = row0 + (int64_t)table_pages * kPageKeys;   // rows whose places would be 0 and the one past the table
  const int from = at_least(start, 0), until = at_most(end, rows);
  const int64_t at = row0 > from ? row0 : from, to = behind < until ? behind : until;
  return to > at ? Sequence{(int)at, (int)(to - at), (int)(to - row0)} : Sequence{0, 0, 0};
}
// .. and for attention: under the causal limit row r sees the keys up to length - end + r, those of its sequence that lie behind the table not among them, as
// if the table went on with pages that are not there.  `keys` is then the end of the call's last row, which nobody sees past (up to n past the table: the
// tiles end there).
constexpr Sequence make_attended(int start, int end, int length, int rows, int table_pages, int causal) {
  const int at = at_most(at_least(start, 0), rows), to = at_most(at_least(end, 0), rows), n = at_least(to - at, 0);
  const int last = at_least(length, 0) - (causal ? at_least(end, 0) - to : 0);
  return {at, n, at_most(at_least(last, 0), table_pages * kPageKeys + (causal ? n : 0))};
}
constexpr int page_in_pool(int id, int64_t n_pages) { return id >= 0 && id < n_pages ? id : -1; }

// ---- writing and reading: the tiles that a sequence's rows lie in, in front of position 0 too ----

constexpr int tiles_of_rows(const Sequence& s) { return s.n > 0 ? ((s.keys - 1) >> 6) - (s.position() >> 6) + 1 : 0; }

// the i-th of them, its places [p0, p1) that are rows of the call, and the call's row that place 0 would be
struct TileRows {
  int tile, p0, p1, row0;
};
constexpr TileRows tile_rows(const Sequence& s, int i) {
  const int tile = (s.position() >> 6) + i;
  return {tile, at_least(s.position() - tile * kPageKeys, 0), at_most(s.keys - tile * kPageKeys, kPageKeys), s.first + tile * kPageKeys - s.position()};
}
// Most tiles that `rows` rows of B sequences can lie in: n consecutive places touch at most floor((n + 62) / 64) + 1.
constexpr int64_t most_tiles(int64_t rows, int64_t B) {
  const int64_t used = B < rows ? B : rows;
  return (rows + 62 * used) / kPageKeys + used;
}

// ---- attention: blocks of rb query rows (a token's query heads of one kv head side by side), and the tiles they see ----

// The query heads of one kv head, and the token of a query row r, 0 <= r < 2^30: r / n by a multiplication.  With s the first power 2^s >= n and
// mul = ceil(2^(30+s) / n) (at most 2^31), r * mul / 2^(30+s) is over r / n by less than r / 2^30 / n, too little to reach the next whole number.
struct Group {
  int n;
  uint32_t mul;
  int shift;
  constexpr int token(int r) const { return (int)(uint32_t)(((uint64_t)((uint32_t)r << 2) * mul >> 32) >> shift); }
};
constexpr Group make_group(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return {n, (uint32_t)((((uint64_t)1 << (30 + s)) + n - 1) / n), s};
}

constexpr int blocks_of(const Sequence& s, const Group& G, int rb) { return (s.n * G.n + rb - 1) / rb; }
// keys that query row r sees; past the last row: what that one sees
constexpr int row_keys(const Sequence& s, const Group& G, int causal, int r) {
  if (!causal) return s.keys;
  return at_most(at_least(s.position() + G.token(at_most(r, s.n * G.n - 1)) + 1, 0), s.keys);
}
// tiles of block j: of its last row.  One at least: a block without keys writes zeros
constexpr int block_tiles(const Sequence& s, const Group& G, int causal, int rb, int j) {
  return at_least((row_keys(s, G, causal, (j + 1) * rb - 1) + kPageKeys - 1) >> 6, 1);
}
constexpr int block_tiles(const Sequence& s, const Group& G, int causal, int rb, int j, int table_pages) {
  return at_most(block_tiles(s, G, causal, rb, j), table_pages);
}

// What a tile of block j costs, by the waves of a workgroup that have rows of it: in the form of 384 rows (12 waves, three a SIMD) 4, or where there
// are rows for two a SIMD or one, 3 or 2 (the waves without rows leave the products out); 1 in the other forms.
constexpr int most_cost(int rb) { return rb == 384 ? 4 : 1; }
constexpr int block_cost(const Sequence& s, const Group& G, int rb, int j) {
  if (rb != 384) return 1;
  const int rows = s.n * G.n - j * rb;
  return rows > 256 ? 4 : rows > 128 ? 3 : 2;
}

// What a unit costs besides its tiles, in tiles: queries in and out, the first keys' way.  Units of 384 rows against 2 and 8 tiles take 10 us and 3.0 a
// tile, longer ones 7 and 2.4 to 2.9; shared out by their tiles alone, the last workgroup of such a call was done at 320 us and the first at 102.
constexpr int kUnitTiles = 4;
constexpr int64_t unit_length(int nt, int cost) { return (int64_t)(nt + kUnitTiles) * cost; }
// where tile t of a unit begins
constexpr int64_t tile_place(int t, int cost) { return t == 0 ? 0 : (int64_t)(t + kUnitTiles) * cost; }
// tiles that `left` of a run is worth from tile t of a unit on (boundaries lie at tiles: nothing is left over)
constexpr int64_t divided(int64_t x, int64_t by) { return (uint64_t)(x | by) >> 32 ? x / by : (int64_t)((uint32_t)x / (uint32_t)by); }
constexpr int tiles_left(int64_t left, int t, int nt, int cost) {
  const int64_t all = divided(left, cost) - (t == 0 ? kUnitTiles : 0);
  return all < nt - t ? (int)all : nt - t;
}

// The tiles of all units end to end, at their cost, in equal runs for `n` workgroups.  (The division is the 32-bit one where that does.)
constexpr int kMaxShares = 512;       // workgroups of a launch at most
constexpr int least_tiles(int rb) { return rb == 384 ? 1 : 2; }   // fewest tiles a workgroup is started for (units that are cut)
constexpr int kWholeTiles = 16;       // pages of a table under which no unit is cut
struct Shares {
  int64_t total;
  int n;
  bool whole;                         // no unit is cut
  constexpr int64_t begin(int i) const { return divided(total * i, n); }
  constexpr int64_t run() const { return divided(total, n); }
};
constexpr Shares shares_of(int64_t total, int most, int rb, bool whole) {
  const int64_t worth = total / (((whole ? 1 : least_tiles(rb)) + kUnitTiles) * (whole ? 1 : most_cost(rb)));
  return {total, (int)(worth < 1 ? 1 : worth < most ? worth : most), whole};
}
// The workgroup of a launch that takes run `rank`: a contiguous run of runs per XCD.  -1: none.
constexpr int rank_of(int block, const Shares& sh) {
  const int per_xcd = (sh.n + 7) / 8, rank = (block & 7) * per_xcd + (block >> 3);
  return (block >> 3) < per_xcd && rank < sh.n ? rank : -1;
}
// A run boundary that lies `in` behind the beginning of a unit of nt tiles at this cost goes to the tile there, or to an end that is so near that a part
// of its own costs more than it gives, or where no unit is cut to the nearer end.  The result may be nt: the next unit's beginning.  (Three tiles for
// near, and units of up to 16 tiles and a run uncut: five ragged prompts 83 us where they are 74 now, nine of up to 2,930 rows 83 and 75.)
constexpr int kNearTiles = 2;
constexpr int boundary_tile(const Shares& sh, int64_t in, int nt, int cost) {
  if (sh.whole) return 2 * in >= unit_length(nt, cost) ? nt : 0;
  const int t = (int)divided(in, cost) - kUnitTiles;
  return t > kNearTiles ? (t < nt - kNearTiles ? t : nt) : 2 * t < nt ? 0 : nt;
}
// A unit that several runs share: run i leaves its part in slot 2*i + 1 if its part begins the unit, else in slot 2*i.
constexpr int64_t part_slot(int run, bool begins) { return 2 * (int64_t)run + (begins ? 1 : 0); }
// Of boundary i, at tile t of the unit of nt tiles that begins at `begin`: if it cuts the unit and is the first that does, how many runs share the unit (the
// one in front of the boundary, the one behind it, ..).  0: not this boundary's business.
constexpr int parts_at(const Shares& sh, int i, int64_t begin, int t, int nt, int cost) {
  if (t <= 0 || t >= nt || sh.begin(i - 1) >= begin + tile_place(kNearTiles + 1, cost)) return 0;
  int parts = 2;
  while (i + parts - 1 < sh.n && sh.begin(i + parts - 1) < begin + tile_place(nt - kNearTiles, cost)) ++parts;
  return parts;
}

}  // namespace pkh3
