// How products on plain rows are shared out among workgroups, for the kernels and for host tests alike: plain C++, no HIP.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace pkh3 {

enum ProductMode { kPlain = 0, kGated = 1, kGrad = 2, kGatedGrad = 3 };

constexpr int kChunk = 64;        // contraction elements of a chunk

// How a product's tiles are shared out.  Every workgroup takes `rounds` whole tiles.  The contraction of each of the `rest` tiles behind them is cut into `cuts` parts of as
// many chunks (or one more); the parts are units of their own, those of the same part of all tiles beside each other: workgroups that run together then read the same part
// of the matrices they share.
struct ProductShare {
  int m_tiles, n_tiles, chunks, groups, rounds, rest, cuts, blocks;
};
constexpr int units_of(const ProductShare& s) { return s.rest * s.cuts; }
// first chunk of a part
constexpr int part_begin(const ProductShare& s, int part) { return (int)((int64_t)s.chunks * part / s.cuts); }

// What a workgroup does in its turn: unit `at` of the rounds' tiles or of the parts.  The workgroups come to the 8 XCDs round-robin; those of one XCD take units beside each other.
constexpr int unit_of(int turns, int turn, int group, int groups) { return ((group & 7) * turns + turn) * (groups >> 3) + (group >> 3); }
constexpr int part_turns(const ProductShare& s) { return (units_of(s) + s.groups - 1) / s.groups; }

// Where a tile lies: the tiles of B in `blocks` blocks as wide as each other, or one tile wider, each of which walks down the tiles of A.  The workgroups that run behind
// one L2 at a time take tiles that follow each other, and read from memory once what they share, so a block is about as wide as it is high in rows.
struct TilePlace {
  int m, n;
};
constexpr TilePlace tile_of(const ProductShare& s, int lin) {
  const int width = s.n_tiles / s.blocks, wider = s.n_tiles - width * s.blocks, in_wider = wider * (width + 1) * s.m_tiles;
  if (lin < in_wider) {
    const int block = lin / ((width + 1) * s.m_tiles), rem = lin - block * (width + 1) * s.m_tiles;
    return {rem / (width + 1), block * (width + 1) + rem % (width + 1)};
  }
  const int block = (lin - in_wider) / (width * s.m_tiles), rem = lin - in_wider - block * width * s.m_tiles;
  return {rem / width, wider * (width + 1) + block * width + rem % width};
}
// The blocks for `together` tiles behind an L2, of `height` rows of A to `wide` of B: width^2 * wide = together * height, no narrower than fills them.
constexpr int tile_blocks(int together, int height, int wide, int m_tiles, int n_tiles) {
  int width = 1;
  while (width < n_tiles && (width * width * wide < together * height || width * m_tiles < together)) ++width;
  return (2 * n_tiles + width) / (2 * width) < 1 ? 1 : (2 * n_tiles + width) / (2 * width);
}

// How a call is carried out, by its sizes alone.
struct ProductPlan {
  bool thin;                     // the form for few rows
  int tb, fb;                    // 16-row blocks of A and of B a wave: tiles of 32 * tb rows of A and 32 * fb of B
  ProductShare share;
  int sum_rows;                  // rows of partial column sums
  size_t part_off, sums_off, total;   // bytes of the workspace
};

constexpr bool product_offered(bool a_across, bool b_across, int mode) {
  if (a_across) return b_across && mode == kPlain;
  return b_across ? mode != kGated : mode <= kGated;
}

constexpr size_t whole_256(size_t n) { return (n + 255) / 256 * 256; }

// The form of pkh3_rows_thin.hip, for few rows of operands along: workgroups of up to 64 rows times 32 columns, or of 16 where 32 would leave CUs without one (and with gates).
constexpr int thin_rows(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : 64; }
constexpr bool thin_narrow(int M, int N) { return (int64_t)((N + 31) / 32) * ((M + thin_rows(M) - 1) / thin_rows(M)) < 192; }
// Its time as plan_time() has it: a workgroup's rows and weights at the 90 GB/s a CU that calls of one workgroup a CU reach, 60 where there are more.  That knows of no memory behind
// the CUs and of no results, as plan_time() does not.  Over 55 products of 1 to 6,000 rows, weights out of memory, both forms timed: up to 300 rows the choice takes up to 1.15 times the
// better form (64 rows, 8,192 to 2,048: 23.9 us, tiles 20.8), where the few rows' form is right up to half of it (128 rows, 2,048 to 2,048: 8.6 us, tiles 19.1).  Above, most choices are right too
// (424 rows, 912 to 200: 5.9 us, tiles 10.6; 3,255 rows, 224 to 120: 4.7, 7.7), but the form is also taken where tiles take less, by up to 35 %: 693 rows, 408 to 1,560 13.1 us, tiles
// 9.5; 2,373 rows, 80 to 768 10.4, 7.0; 6,001 rows, 264 to 248 14.7, 9.6.
constexpr int64_t thin_time(int M, int N, int K, int mode) {
  const int columns = mode == kGated || thin_narrow(M, N) ? 16 : 32, blocks = thin_rows(M) + (mode == kGated ? 32 : columns);
  const int64_t groups = (int64_t)((N + columns - 1) / columns) * ((M + thin_rows(M) - 1) / thin_rows(M)), bytes = (int64_t)blocks * K * 2;
  return groups <= 256 ? bytes / 900 : bytes * groups / 256 / 600;
}

// The time that a plan takes, in hundredths of a microsecond besides the launch, from what was measured with weights that come from memory: a chunk of a
// tile of 256 x 256, 128 x 256, 128 x 128, 96 x 128 and 64 x 128 rows 1.1, 0.8, 0.52, 0.46 and 0.36 us, what a tile takes besides 5, 3.5, 2.5, 2.2 and 2; parts go to memory and
// come back at 6 TB/s, and are joined by a launch of its own, 8 us.  (Over 42 products of 128 to 9,500 rows the choice takes 0.6 % longer than the best of the
// forms and cuts, at worst 15 %.)  What a smaller tile costs in copies for each product it gives back where there are few tiles: 1,085 x 2,048 x 2,048 takes 33.4 us in 72
// tiles of 128 x 256, 24.7 in 144 of 128 x 128 and 21.9 in 192 of 96 x 128; 1,044 x 1,600 with a contraction of 608 12.5 us in tiles of 128 x 128, 11.6 of 96 x 128 and
// 10.2 of 64 x 128; 4,000 x 2,048 x 2,048 35 us in 256 tiles of 128 x 256 and 43 of 128 x 128; 3,265 x 9,296 x 2,320 127 us of 256 x 256 and 159 of 128 x 256.
constexpr int64_t plan_time(const ProductShare& s, int tb, int fb, int M) {
  const int64_t chunk = tb > 4 ? 110 : fb > 4 ? 80 : tb > 3 ? 52 : tb > 2 ? 46 : 36, tile = tb > 4 ? 500 : fb > 4 ? 350 : tb > 3 ? 250 : tb > 2 ? 220 : 200;
  int64_t time = s.rounds * (s.chunks * chunk + tile);
  if (s.rest) time += part_turns(s) * ((int64_t)((s.chunks + s.cuts - 1) / s.cuts) * chunk + tile);
  if (s.cuts > 1) {
    const int64_t rows = (int64_t)s.m_tiles * 32 * tb, bytes = (int64_t)units_of(s) * 32 * tb * 32 * fb * 4 * M / rows * 2;
    time += 800 + bytes / 60000;
  }
  return time;
}

// Tiles that there are, in 16-row blocks a wave.  (Those of 96 rows not where A is stored across, whose rows come to LDS in units of 64.)
constexpr int kForms[5][2] = {{8, 8}, {4, 8}, {4, 4}, {3, 4}, {2, 4}};

constexpr ProductPlan plan_product(int M, int N, int K, bool along, int mode, bool sums, bool a_across = false) {
  ProductPlan plan{};
  int64_t best = 0;
  for (const auto& form : kForms) {
    const int tb = form[0], fb = form[1], columns = mode == kGated ? 16 * fb : 32 * fb;
    if (tb == 3 && a_across) continue;
    ProductShare s{};
    s.m_tiles = (M + 32 * tb - 1) / (32 * tb), s.n_tiles = (N + columns - 1) / columns;
    s.chunks = (K + kChunk - 1) / kChunk;
    s.groups = 256;                                  // one on every CU
    const int64_t tiles = (int64_t)s.m_tiles * s.n_tiles;
    s.rounds = (int)(tiles / s.groups);
    s.rest = (int)(tiles - (int64_t)s.rounds * s.groups);
    const int together = tiles < 256 ? (int)(tiles + 7) / 8 : 32;
    s.blocks = tile_blocks(together, 32 * tb, 32 * fb, s.m_tiles, s.n_tiles);
    const int most = s.rest == 0 || s.chunks < 4 ? 1 : s.chunks / 2 < 64 ? s.chunks / 2 : 64;
    for (int cuts = 1; cuts <= most && (cuts == 1 || s.rest * cuts <= 4 * s.groups); ++cuts) {
      s.cuts = cuts;
      const int64_t time = plan_time(s, tb, fb, M);
      if (plan.tb == 0 || time < best) plan.tb = tb, plan.fb = fb, plan.share = s, best = time;
    }
  }
  if (along && thin_time(M, N, K, mode) < best) {
    plan.thin = true;
    return plan;
  }
  const ProductShare& s = plan.share;
  plan.sum_rows = sums ? s.m_tiles * 2 : 0;
  plan.sums_off = s.cuts > 1 ? whole_256((size_t)units_of(s) * 32 * plan.tb * 32 * plan.fb * sizeof(float)) : 0;
  plan.total = plan.sums_off + whole_256((size_t)plan.sum_rows * (mode == kGatedGrad ? 2 : 1) * N * sizeof(float));
  return plan;
}

}  // namespace pkh3
