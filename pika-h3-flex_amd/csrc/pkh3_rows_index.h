// How products on plain rows are shared out among workgroups, for the kernels and for host tests alike: plain C++, no HIP.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace pkh3 {

enum ProductMode { kPlain = 0, kGated = 1, kGrad = 2, kGatedGrad = 3 };

constexpr int kTileB = 256;       // rows of B of a tile
constexpr int kChunk = 64;        // contraction elements of a chunk

// How a product's tiles are shared out.  Every workgroup takes `rounds` whole tiles; the chunks of the `rest` tiles behind them lie end to end and are cut into
// `runs` runs, one a workgroup (as many runs as tiles: whole tiles), the first `longer` of them of run_chunks + 1 chunks, the others of run_chunks.  A run covers parts of at
// most two tiles, since there are at least as many runs as tiles.
struct ProductShare {
  int m_tiles, n_tiles, chunks, groups, rounds, rest, runs, run_chunks, longer, unused;
};
// first chunk of a run
constexpr int run_begin(const ProductShare& s, int run) {
  const int r = run < s.runs ? run : s.runs;
  return r * s.run_chunks + (r < s.longer ? r : s.longer);
}
// the run that holds a chunk
constexpr int run_of(const ProductShare& s, int chunk) {
  const int behind = s.longer * (s.run_chunks + 1);
  return chunk < behind ? chunk / (s.run_chunks + 1) : s.longer + (chunk - behind) / s.run_chunks;
}
// where a run's part of the tile whose first chunk is tile_begin lies among the parts: the one that the run begins in comes first
constexpr int part_slot(const ProductShare& s, int run, int tile_begin) { return 2 * run + (run_begin(s, run) < tile_begin ? 1 : 0); }

// Where a tile lies: blocks of 8 tiles of B walk down the tiles of A, so that the workgroups that run behind one L2 at a time share 8 tiles of B and 4 of A.
struct TilePlace {
  int m, n;
};
constexpr TilePlace tile_of(const ProductShare& s, int lin) {
  constexpr int kBlockN = 8;
  const int full = s.n_tiles / kBlockN * kBlockN;
  if (lin < full * s.m_tiles) return {lin % (kBlockN * s.m_tiles) / kBlockN, lin / (kBlockN * s.m_tiles) * kBlockN + lin % kBlockN};
  const int over = lin - full * s.m_tiles, width = s.n_tiles - full;
  return {over / width, full + over % width};
}

// How a call is carried out, by its sizes alone.
struct ProductPlan {
  int tb;                        // 16-row blocks of A a wave: tiles of 32 * tb rows of A and 256 of B
  ProductShare share;
  int sum_rows;                  // rows of partial column sums
  size_t part_off, sums_off, total;   // bytes of the workspace
};

constexpr bool product_offered(bool a_across, bool b_across, int mode) {
  if (a_across) return b_across && mode == kPlain;
  return b_across ? mode != kGated : mode <= kGated;
}

constexpr size_t whole_256(size_t n) { return (n + 255) / 256 * 256; }

constexpr ProductPlan plan_product(int M, int N, int K, int mode, bool sums) {
  ProductPlan plan{};
  plan.tb = M > 1024 ? 8 : M > 256 ? 4 : 2;
  const int columns = mode == kGated ? kTileB / 2 : kTileB;
  ProductShare& s = plan.share;
  s.m_tiles = (M + 32 * plan.tb - 1) / (32 * plan.tb), s.n_tiles = (N + columns - 1) / columns;
  s.chunks = (K + kChunk - 1) / kChunk;
  const int tiles = s.m_tiles * s.n_tiles;
  s.groups = 256;                                    // one on every CU
  s.rounds = tiles / s.groups;
  s.rest = tiles - s.rounds * s.groups;
  // tiles behind the whole rounds: shared out where that saves more than it costs
  s.runs = s.rest;
  if (s.rest && s.rest * 3 < s.groups * 2) {
    const int64_t runs = (int64_t)s.rest * s.chunks / 4;
    s.runs = runs < s.rest ? s.rest : runs > s.groups ? s.groups : (int)runs;
  }
  if (s.rest) s.run_chunks = s.rest * s.chunks / s.runs, s.longer = s.rest * s.chunks % s.runs;
  plan.sum_rows = sums ? s.m_tiles * 2 : 0;
  plan.sums_off = s.runs > s.rest ? whole_256((size_t)2 * s.runs * 32 * plan.tb * kTileB * sizeof(float)) : 0;
  plan.total = plan.sums_off + whole_256((size_t)plan.sum_rows * (mode == kGatedGrad ? 2 : 1) * N * sizeof(float));
  return plan;
}

}  // namespace pkh3
