"""The paged K/V cache without a GPU: refusals of the C entries and of the Python front end, and the index arithmetic of the kernels in a
host build -- batches whose arrays hold anything, and every tile of every unit done once."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

import pika_h3_flex_amd as pk
from pika_h3_flex_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pika-h3-flex_amd", "csrc")


def test_struct_layout_matches_header():
    header = open(os.path.join(ROOT, "include", "pkh3_paged.h")).read()
    body = header[header.index("typedef struct pkh3_paged_args {"): header.index("} pkh3_paged_args;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = [re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1] for decl in body.split(";") if decl.strip() for part in decl.split(",")]
    assert names == [f[0] for f in _lib.PagedArgs._fields_]


def _args():
    a = _lib.PagedArgs()
    buf = 0x10000   # made-up, aligned addresses: refusals come before anything looks at them
    for n in ("pages", "starts", "lengths", "table", "q", "k", "v", "o", "workspace"):
        setattr(a, n, buf)
    for n in ("q", "k", "v", "o"):
        setattr(a, n + "_ss", 4 * 128)
        setattr(a, n + "_sh", 128)
    a.n_pages, a.table_stride, a.B, a.table_pages, a.rows, a.kv_heads, a.heads, a.D = 9, 4, 2, 4, 5, 2, 4, 128
    a.norm_eps = 1e-6
    a.workspace_bytes = 1 << 30
    return a


def test_sizes_on_the_host(lib):
    assert lib.pkh3_paged_record_bytes(0) == 32768 and lib.pkh3_paged_record_bytes(_lib.PAGED_FP8) == 16384 + 128
    assert lib.pkh3_paged_record_bytes(8) == 0
    a = _args()
    n = lib.pkh3_paged_workspace_bytes(C.byref(a))
    assert n > 0 and n % 256 == 0
    a.rows = 0
    assert lib.pkh3_paged_workspace_bytes(C.byref(a)) > 0
    a.heads = 3
    assert lib.pkh3_paged_workspace_bytes(C.byref(a)) == 0


def _set(**kw):
    return lambda a: [setattr(a, k, v) for k, v in kw.items()]


COMMON = [
    (_set(pages=0), _lib.PKH3_ENULL), (_set(pages=0x10010), _lib.PKH3_EALIGN), (_set(starts=0), _lib.PKH3_ENULL),
    (_set(lengths=0), _lib.PKH3_ENULL), (_set(table=0), _lib.PKH3_ENULL), (_set(starts=0x10002), _lib.PKH3_EALIGN),
    (_set(D=64), _lib.PKH3_EHEADDIM), (_set(flags=4), _lib.PKH3_EARG), (_set(B=0), _lib.PKH3_ESHAPE), (_set(B=1025), _lib.PKH3_ESHAPE),
    (_set(rows=-1), _lib.PKH3_ESHAPE), (_set(rows=(1 << 24) + 1), _lib.PKH3_ESHAPE), (_set(kv_heads=0), _lib.PKH3_ESHAPE),
    (_set(table_pages=0), _lib.PKH3_ESHAPE), (_set(table_pages=(1 << 24) + 1), _lib.PKH3_ESHAPE), (_set(table_stride=-4), _lib.PKH3_ESTRIDE),
    (_set(n_pages=0), _lib.PKH3_ESHAPE), (_set(n_pages=1 << 31), _lib.PKH3_ESHAPE), (_set(rows=1 << 24, heads=65534), _lib.PKH3_ESHAPE),
]
ROWS_IN = [(_set(rope_mode=3), _lib.PKH3_EARG), (_set(rope_mode=1), _lib.PKH3_ENULL), (_set(rope_mode=1, rope_cos=0x10008, rope_sin=0x10000), _lib.PKH3_EALIGN),
           (_set(norm_w=0x10004), _lib.PKH3_EALIGN), (_set(norm_w=0x10000, norm_eps=-1.0), _lib.PKH3_EARG),
           (_set(norm_w=0x10000, norm_eps=float("nan")), _lib.PKH3_EARG)]


def _refuses(lib, entry, mutate, code):
    a = _args()
    mutate(a)
    assert getattr(lib, entry)(C.byref(a), None) == code
    assert lib.pkh3_last_error() != b""


@pytest.mark.parametrize("mutate,code", COMMON + ROWS_IN + [
    (_set(q=0), _lib.PKH3_ENULL), (_set(o=0), _lib.PKH3_ENULL), (_set(q=0x10008), _lib.PKH3_EALIGN), (_set(q_ss=132), _lib.PKH3_ESTRIDE),
    (_set(q_sh=-128), _lib.PKH3_ESTRIDE), (_set(o_sh=0), _lib.PKH3_ESTRIDE), (_set(o_ss=0), _lib.PKH3_ESTRIDE), (_set(heads=3), _lib.PKH3_ESHAPE),
    (_set(heads=0), _lib.PKH3_ESHAPE), (_set(softmax_scale=float("nan")), _lib.PKH3_EARG), (_set(softmax_scale=float("inf")), _lib.PKH3_EARG),
    (_set(workspace=0), _lib.PKH3_EWORKSPACE), (_set(workspace=0x10010), _lib.PKH3_EWORKSPACE), (_set(workspace_bytes=1024), _lib.PKH3_EWORKSPACE)])
def test_attention_refuses(lib, mutate, code):
    _refuses(lib, "pkh3_paged_attn", mutate, code)


@pytest.mark.parametrize("mutate,code", [c for c in COMMON[:-1]] + ROWS_IN + [
    (_set(k=0), _lib.PKH3_ENULL), (_set(v=0x10008), _lib.PKH3_EALIGN), (_set(k_ss=100), _lib.PKH3_ESTRIDE), (_set(flags=2), _lib.PKH3_EARG)])
def test_write_refuses(lib, mutate, code):
    _refuses(lib, "pkh3_paged_write", mutate, code)


@pytest.mark.parametrize("mutate,code", [c for c in COMMON[:-1]] + [
    (_set(k=0), _lib.PKH3_ENULL), (_set(v=0), _lib.PKH3_ENULL), (_set(v_sh=64), _lib.PKH3_ESTRIDE), (_set(k_sh=0), _lib.PKH3_ESTRIDE), (_set(flags=2), _lib.PKH3_EARG)])
def test_read_refuses(lib, mutate, code):
    _refuses(lib, "pkh3_paged_read", mutate, code)


def test_outputs_that_overlap_themselves_are_refused(lib):
    """Strides that give two rows, or two heads of different rows, one address, whichever is the outer one; strides that interleave without overlapping are not."""
    import itertools

    for ss, sh, rows, heads in itertools.product((128, 136, 256, 384, 512, 640, 1024), (128, 136, 256, 384, 512, 640, 1024), (1, 2, 5), (1, 2, 4)):
        at = sorted(r * ss + h * sh for r in range(rows) for h in range(heads))
        overlap = any(b - a < 128 for a, b in zip(at, at[1:]))
        # where the strides pass, a refusal behind theirs: nothing is launched
        for entry, name, behind in (("pkh3_paged_attn", "o", dict(workspace=0)), ("pkh3_paged_read", "k", dict(v=0)), ("pkh3_paged_read", "v", None)):
            if behind is None and not overlap:
                continue
            a = _args()
            a.rows, a.heads, a.kv_heads = rows, heads, heads
            for n, x in dict(behind or {}, k_ss=heads * 128, v_ss=heads * 128).items():
                setattr(a, n, x)
            setattr(a, name + "_ss", ss)
            setattr(a, name + "_sh", sh)
            want = _lib.PKH3_ESTRIDE if overlap else _lib.PKH3_EWORKSPACE if name == "o" else _lib.PKH3_ENULL
            assert getattr(lib, entry)(C.byref(a), None) == want, (entry, name, ss, sh, rows, heads)


def test_reading_both_sides_into_one_place_is_refused(lib):
    a = _args()
    assert a.k == a.v and lib.pkh3_paged_read(C.byref(a), None) == _lib.PKH3_EARG
    assert b"k and v" in lib.pkh3_last_error()


def test_no_rows_is_no_launch(lib):
    a = _args()
    a.rows = 0
    for entry in ("pkh3_paged_write", "pkh3_paged_read", "pkh3_paged_attn"):
        assert getattr(lib, entry)(C.byref(a), None) == 0 and lib.pkh3_last_error() == b""
    assert lib.pkh3_paged_attn(None, None) == _lib.PKH3_ENULL


def test_batches_are_checked_where_they_are_built():
    build = lambda *a: pk.PagedBatch.build(*a, device="cpu")   # noqa: E731
    b = build([1, 0, 3], [70, 0, 3], [[4, 2], [], [0]])
    assert b.starts.tolist() == [0, 1, 1, 4] and b.lengths.tolist() == [70, 0, 3] and b.table.tolist() == [[4, 2], [-1, -1], [0, -1]] and b.rows == 4
    assert build([2], [0], [[]]).table.tolist() == [[-1]]
    for bad in (([], [], []), ([1], [1, 2], [[0]]), ([1], [65], [[0]]), ([-1], [1], [[0]]), ([1], [-1], [[0]]), ([1], [1], [[-2]]),
                ([1] * 1025, [1] * 1025, [[0]] * 1025)):
        with pytest.raises(ValueError):
            build(*bad)


def test_the_front_end_refuses_what_the_kernels_cannot_take():
    """Tensors of the host, wrong types, shapes and strides are errors before any call."""
    cache = pk.PagedKV(3, 2, device="cpu")
    batch = pk.PagedBatch.build([1], [1], [[0]], device="cpu")
    rows = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    for call in (lambda: pk.paged_write(cache, batch, rows, rows), lambda: pk.paged_attention(rows, cache, batch), lambda: pk.paged_read(cache, batch)):
        with pytest.raises(ValueError, match="device memory"):
            call()
    with pytest.raises(TypeError):
        pk.paged_attention(rows.float(), cache, batch)
    with pytest.raises(ValueError):
        pk.paged_attention(rows[..., :64], cache, batch)
    with pytest.raises(ValueError):
        pk.paged_write(cache, batch, rows[:, :1], rows)
    with pytest.raises(ValueError):
        pk.PagedKV(0, 2, device="cpu")
    with pytest.raises(ValueError):
        pk.PagedKV(3, 2, device="cpu", data=torch.zeros((3, 2, 5), dtype=torch.uint8))
    with pytest.raises(ValueError, match="say how many"):
        pk.paged_read(cache, pk.PagedBatch(batch.starts, batch.lengths, batch.table))


# ---- index arithmetic ----

def _run(tmp_path, body):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "host.cc", tmp_path / "host"
    src.write_text('#include "pkh3_paged_index.h"\n#include <stdio.h>\n#include <stdlib.h>\n#include <vector>\n#include <algorithm>\nusing namespace pkh3;\n'
                   '#define CHECK(x, ...) do { if (!(x)) { printf(#x ": " __VA_ARGS__); return 1; } } while (0)\n'
                   "[[maybe_unused]] static int any(int lo, int hi) { return lo + (int)(rand() % (hi - lo + 1)); }\n"
                   "int main() {\n  srand(1);\n" + body + "\n  return 0;\n}\n")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src), "-o", str(exe)],
                   check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_rows_and_pages_stay_in_range_whatever_the_arrays_hold(tmp_path):
    _run(tmp_path, """
  const int wild[] = {0, 1, 5, 63, 64, 65, 1000, -1, -7, 2147483647, -2147483647 - 1, 16777216, 1 << 30};
  const int n_wild = sizeof(wild) / sizeof(int);
  for (int a = 0; a < n_wild; ++a) for (int b = 0; b < n_wild; ++b) for (int c = 0; c < n_wild; ++c)
    for (int rows : {0, 1, 70, 16777216}) for (int pages : {1, 3, 16777216}) {
      const Sequence s = make_sequence(wild[a], wild[b], wild[c], rows, pages);
      CHECK(s.first >= 0 && s.n >= 0 && s.first + s.n <= rows && s.keys >= 0 && s.keys <= pages * 64, "%d %d %d", wild[a], wild[b], wild[c]);
      const int tiles = tiles_of_rows(s);
      CHECK((tiles > 0) == (s.n > 0) && tiles <= s.n / 64 + 2, "%d tiles of %d rows", tiles, s.n);
      for (int i : {0, 1, tiles / 2, tiles - 1}) {
        if (i < 0 || i >= tiles) continue;
        const TileRows t = tile_rows(s, i);
        CHECK(t.p0 >= 0 && t.p0 < t.p1 && t.p1 <= 64 && t.row0 + t.p0 >= s.first && t.row0 + t.p1 <= s.first + s.n, "tile %d", i);
      }
      for (int g : {1, 6}) for (int causal : {0, 1}) for (int rb : {16, 32, 128, 384}) {
        const Group G = make_group(g);
        if (s.n == 0 || (int64_t)rows * g > (1 << 30)) continue;
        const int blocks = blocks_of(s, G, rb);
        for (int j : {0, blocks / 2, blocks - 1}) {
          const int t = block_tiles(s, G, causal, rb, j);
          CHECK(t >= 1 && t <= (pages > 1 ? pages : 1), "%d tiles", t);
          for (int r = j * rb; r < std::min((j + 1) * rb, s.n * g); ++r) {
            const int k = row_keys(s, G, causal, r);
            CHECK(k >= 0 && k <= s.keys && k <= 64 * t, "row %d sees %d", r, k);
            CHECK(k == (causal ? std::max(0, std::min(s.keys, s.keys - s.n + r / g + 1)) : s.keys), "row %d sees %d", r, k);
            CHECK(k >= row_keys(s, G, causal, j * rb), "the first row of a block sees least");
          }
        }
      }
    }
  for (int g = 1; g <= 65535; g = g < 70 ? g + 1 : g + any(1, 999)) {
    const Group G = make_group(g);
    for (int k = 0; k < 300; ++k) {
      const int r = k < 40 ? k : k < 80 ? (1 << 30) - k + 39 : k < 200 ? any(0, (1 << 30) - 1) : std::min(any(0, (1 << 30) / g) * g + any(-1, 1) + (k == 200), (1 << 30) - 1);
      if (r >= 0) CHECK(G.token(r) == r / g, "%d / %d is %d", r, g, G.token(r));
    }
  }
  for (int id : {-1, 0, 4, 5, 2147483647}) CHECK(page_in_pool(id, 5) == (id >= 0 && id < 5 ? id : -1), "%d", id);""")


def test_every_row_lies_in_one_tile_of_the_launch(tmp_path):
    _run(tmp_path, """
  for (int go = 0; go < 3000; ++go) {
    const int B = any(1, 9);
    std::vector<int> starts(1, any(0, 2)), keys;
    for (int b = 0; b < B; ++b) {
      starts.push_back(starts.back() + (any(0, 3) ? any(0, 3) ? any(0, 5) : any(0, 300) : 0));
      keys.push_back(any(0, 3) ? any(0, 400) : any(0, 3));
    }
    const int rows = starts.back() + any(0, 2);
    std::vector<int> times(rows, 0);
    int64_t tiles = 0;
    for (int b = 0; b < B; ++b) {
      const Sequence s = make_sequence(starts[b], starts[b + 1], keys[b], rows, 10);
      tiles += tiles_of_rows(s);
      for (int i = 0; i < tiles_of_rows(s); ++i) {
        const TileRows t = tile_rows(s, i);
        for (int at = t.p0; at < t.p1; ++at) {
          ++times[t.row0 + at];
          CHECK(t.tile * 64 + at == s.position() + (t.row0 + at - s.first), "place");
        }
      }
    }
    CHECK(tiles <= most_tiles(rows, B), "%lld tiles, the launch has %lld", (long long)tiles, (long long)most_tiles(rows, B));
    for (int r = 0; r < rows; ++r) CHECK(times[r] == (r >= starts[0] && r < starts[B] ? 1 : 0), "row %d: %d times", r, times[r]);
  }""")


def test_runs_cover_every_tile_of_every_unit_once(tmp_path):
    """The walk of the attention kernels, all workgroups of a launch: every tile of every unit in one run, a unit's parts in slots of their own, and
    every cut unit joined at one boundary, in the order of the runs."""
    _run(tmp_path, """
  for (int go = 0; go < 6000; ++go) {
    const int B = any(1, 6), H = any(1, 4), causal = any(0, 1), rb = go % 5 <= 1 ? 384 : go % 5 == 2 ? 128 : go % 5 == 3 ? 32 : 16;
    const int grid = go % 3 == 0 ? 8 : go % 3 == 1 ? 24 : 512;
    const Group G = make_group(any(1, 4));
    struct Unit { int64_t begin; int nt, cost; };
    std::vector<Unit> units;
    int64_t total = 0;
    for (int b = 0; b < B; ++b) {
      const int n = any(0, 2) ? any(0, 40) : any(0, 900), keys = any(0, 3) ? any(0, 2000) : any(0, 64);
      const Sequence s = make_sequence(0, n, keys, 1000, 100);
      for (int h = 0; h < H; ++h)
        for (int j = 0; j < blocks_of(s, G, rb); ++j) {
          const int t = block_tiles(s, G, causal, rb, j), cost = block_cost(s, G, rb, j);
          CHECK(cost >= 1 && cost <= most_cost(rb), "cost %d", cost);
          units.push_back({total, t, cost});
          total += unit_length(t, cost);
        }
    }
    const bool whole = any(0, 4) == 0;
    const Shares sh = shares_of(total, grid, rb, whole);
    CHECK(sh.n >= 1 && sh.n <= grid && sh.begin(0) == 0 && sh.begin(sh.n) == total, "%d runs", sh.n);
    std::vector<int> who(sh.n, 0);
    for (int block = 0; block < grid; ++block) {
      const int r = rank_of(block, sh);
      CHECK(r >= -1 && r < sh.n, "rank %d", r);
      if (r >= 0) ++who[r];
    }
    for (int r = 0; r < sh.n; ++r) CHECK(who[r] == 1, "run %d of %d taken %d times", r, sh.n, who[r]);
    if (total == 0) continue;
    // where every run begins: unit and tile, and the same as a place in the space of all tiles; parts as its workgroup leaves them
    std::vector<int> unit_of(sh.n), tile_of(sh.n), parts(sh.n);
    std::vector<int64_t> pos(sh.n + 1, total);
    for (int r = 0, u = 0; r < sh.n; ++r) {
      while (sh.begin(r) >= units[u].begin + unit_length(units[u].nt, units[u].cost)) ++u;
      const int t = boundary_tile(sh, sh.begin(r) - units[u].begin, units[u].nt, units[u].cost);
      CHECK(t >= 0 && t <= units[u].nt && (!whole || t == 0 || t == units[u].nt), "tile %d", t);
      unit_of[r] = u, tile_of[r] = t, pos[r] = units[u].begin + tile_place(t, units[u].cost);
      parts[r] = r == 0 ? 0 : parts_at(sh, r, units[u].begin, t, units[u].nt, units[u].cost);
    }
    CHECK(pos[0] == 0, "the first run begins at %lld", (long long)pos[0]);
    for (int r = 0; r < sh.n; ++r) CHECK(pos[r] <= pos[r + 1], "run %d is negative", r);
    // the walk
    std::vector<std::vector<int>> done(units.size()), shared(units.size());
    std::vector<int> slot(2 * sh.n, -1);
    for (size_t u = 0; u < units.size(); ++u) done[u].assign(units[u].nt, 0);
    for (int r = 0; r < sh.n; ++r) {
      int64_t left = pos[r + 1] - pos[r];
      int u = unit_of[r], t = tile_of[r];
      if (left > 0 && t == units[u].nt) ++u, t = 0;
      while (left > 0) {
        const int take = tiles_left(left, t, units[u].nt, units[u].cost);
        CHECK(take >= 1, "run %d stands still", r);
        for (int i = 0; i < take; ++i) ++done[u][t + i];
        if (!(t == 0 && take == units[u].nt)) {
          const int64_t at = part_slot(r, t == 0);
          CHECK(at >= 0 && at < 2 * sh.n && slot[at] < 0, "slot %lld twice", (long long)at);
          slot[at] = u;
          shared[u].push_back(r);
        }
        left -= (int64_t)(take + (t == 0 ? kUnitTiles : 0)) * units[u].cost;
        ++u, t = 0;
      }
      CHECK(left == 0, "run %d ends inside a tile", r);
    }
    for (size_t u = 0; u < units.size(); ++u)
      for (int t = 0; t < units[u].nt; ++t) CHECK(done[u][t] == 1, "tile %d of unit %d done %d times", t, (int)u, done[u][t]);
    // the second launch
    std::vector<int> joined(units.size(), 0);
    for (int r = 1; r < sh.n; ++r) {
      if (!parts[r]) continue;
      const int u = unit_of[r];
      ++joined[u];
      CHECK(parts[r] == (int)shared[u].size(), "%d parts of %d", parts[r], (int)shared[u].size());
      for (int k = 0; k < parts[r]; ++k) CHECK(slot[part_slot(r - 1 + k, k == 0)] == u && shared[u][k] == r - 1 + k, "part %d", k);
    }
    for (size_t u = 0; u < units.size(); ++u) CHECK(joined[u] == (shared[u].empty() ? 0 : 1), "unit of %d parts joined %d times", (int)shared[u].size(), joined[u]);
  }
  CHECK(divided(7, 2) == 3 && divided(1ll << 40, 3) == (1ll << 40) / 3 && divided(5, 1ll << 33) == 0 && divided(4294967295ll, 7) == 4294967295ll / 7, "division");""")


def test_rows_are_written_in_their_own_place_or_not_at_all(tmp_path):
    """Whatever starts and lengths hold, a row that a write stores stands at length - end + row of the values as they are: no other key's place is taken."""
    _run(tmp_path, """
  const int wild[] = {0, 1, 5, 63, 64, 65, 129, 192, 193, 1000, -1, -7, 2147483647, -2147483647 - 1, 16777216, 1 << 30};
  const int n_wild = sizeof(wild) / sizeof(int);
  for (int a = 0; a < n_wild; ++a) for (int b = 0; b < n_wild; ++b) for (int c = 0; c < n_wild; ++c)
    for (int rows : {0, 1, 70, 200}) for (int pages : {1, 3, 16777216}) {
      const Sequence s = make_written(wild[a], wild[b], wild[c], rows, pages);
      CHECK(s.n >= 0 && s.first >= 0 && s.first + s.n <= rows && s.keys >= 0 && s.keys <= pages * 64, "%d %d %d", wild[a], wild[b], wild[c]);
      std::vector<int64_t> place(rows, -1);
      CHECK(tiles_of_rows(s) <= s.n / 64 + 2, "tiles");
      for (int i = 0; i < tiles_of_rows(s); ++i) {
        const TileRows t = tile_rows(s, i);
        for (int at = t.p0; at < t.p1; ++at) {
          CHECK(t.row0 + at >= 0 && t.row0 + at < rows && place[t.row0 + at] < 0, "row %d", t.row0 + at);
          place[t.row0 + at] = (int64_t)t.tile * 64 + at;
        }
      }
      for (int r = 0; r < rows; ++r) {
        const int64_t own = (int64_t)wild[c] - wild[b] + r;
        CHECK(place[r] == (r >= wild[a] && r < wild[b] && own >= 0 && own < (int64_t)pages * 64 ? own : -1), "row %d of %d %d %d at %lld", r, wild[a], wild[b], wild[c], (long long)place[r]);
      }
    }
  for (int go = 0; go < 3000; ++go) {   // values in range: the same rows as everywhere, those in front of the first key aside
    const int start = any(0, 50), n = any(0, 300), keys = any(0, 640), rows = start + n + any(0, 3);
    const Sequence s = make_sequence(start, start + n, keys, rows, 10), w = make_written(start, start + n, keys, rows, 10);
    CHECK(w.n == std::min(n, keys), "%d of %d rows", w.n, n);
    if (w.n) CHECK(w.first - w.position() == s.first - s.position() && w.keys == s.keys && tiles_of_rows(w) <= tiles_of_rows(s), "place");
  }""")


def test_rows_see_the_keys_up_to_their_own_place(tmp_path):
    """Whatever starts and lengths hold: under the causal limit a row sees what is stored up to length - end + row of the values as they are, otherwise all of it."""
    _run(tmp_path, """
  const int wild[] = {0, 1, 5, 63, 64, 65, 129, 192, 193, 1000, -1, -7, 2147483647, -2147483647 - 1, 16777216, 1 << 30};
  const int n_wild = sizeof(wild) / sizeof(int);
  for (int a = 0; a < n_wild; ++a) for (int b = 0; b < n_wild; ++b) for (int c = 0; c < n_wild; ++c)
    for (int rows : {0, 1, 70, 200}) for (int pages : {1, 3, 16777216}) for (int causal : {0, 1}) {
      const Sequence s = make_attended(wild[a], wild[b], wild[c], rows, pages, causal);
      CHECK(s.n >= 0 && s.first >= 0 && s.first + s.n <= rows, "%d %d %d", wild[a], wild[b], wild[c]);
      CHECK(s.n == std::max<int64_t>(0, (int64_t)std::min(wild[b], rows) - std::max(wild[a], 0)), "%d rows", s.n);
      const int64_t held = std::max<int64_t>(0, std::min<int64_t>(wild[c], (int64_t)pages * 64));
      for (int g : {1, 6}) for (int rb : {16, 32, 384}) {
        const Group G = make_group(g);
        for (int r = 0; r < s.n * g; ++r) {
          const int64_t own = (int64_t)wild[c] - wild[b] + s.first + r / g, sees = causal ? std::max<int64_t>(0, std::min(held, own + 1)) : held;
          const int t = block_tiles(s, G, causal, rb, r / rb, pages), k = row_keys(s, G, causal, r);
          CHECK(t >= 1 && t <= pages && sees <= 64ll * t, "%d tiles", t);
          CHECK(std::min<int64_t>(k, pages * 64ll) == sees, "row %d of %d %d %d sees %d", r, wild[a], wild[b], wild[c], k);
          CHECK(std::min<int64_t>(s.keys, pages * 64ll) >= sees && k >= row_keys(s, G, causal, r / rb * rb), "keys");
        }
      }
    }""")


def test_the_processor_refuses_what_does_not_go_with_pages():
    proc = pk.PikaH3AttnProcessor()
    cache = pk.PagedKV(2, 1, device="cpu")
    batch = pk.PagedBatch.build([3], [3], [[0]], device="cpu")
    x = torch.zeros((1, 3, 128), dtype=torch.bfloat16)

    class Attn:
        heads = 1

    with pytest.raises(ValueError, match="together"):
        proc(Attn(), x, paged_kv=cache)
    for bad in (dict(encoder_hidden_states=x), dict(attention_mask=torch.ones((1, 3), dtype=torch.bool)), dict(fp8_qk=True), dict(residual=x)):
        with pytest.raises(ValueError, match="do not go with it"):
            proc(Attn(), x, paged_kv=cache, paged_batch=batch, **bad)
    with pytest.raises(ValueError, match="packed"):
        proc(Attn(), x.expand(2, 3, 128), paged_kv=cache, paged_batch=batch)
    with pytest.raises(ValueError, match="packed"):
        proc.write_paged(Attn(), x[0], cache, batch)


@pytest.mark.parametrize("option", [dict(paged_causal=True), dict(paged_write=False)])
def test_the_processor_refuses_options_of_paged_calls_without_pages(option):
    """Who forgets the pool does not get attention without the causal limit, or over the call's own keys."""
    x = torch.zeros((1, 3, 128), dtype=torch.bfloat16)

    class Attn:
        heads = 1

    with pytest.raises(ValueError, match="paged_kv"):
        pk.PikaH3AttnProcessor()(Attn(), x, **option)


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_have_their_own_addresses(how):
    """What a pool and a batch keep of their tensors beside them is that of the copy's tensors."""
    import copy
    import pickle

    import pika_h3_flex_amd as pk

    record = pk.PagedKV(1, 1, device="cpu").record_bytes
    pool = pk.PagedKV(3, 2, data=torch.arange(3 * 2 * record, dtype=torch.int64).to(torch.uint8).view(3, 2, record))
    batch = pk.PagedBatch.build([1, 2], [5, 70], [[2], [0, 1]], device="cpu")
    again = copy.deepcopy((pool, batch)) if how == "deepcopy" else pickle.loads(pickle.dumps((pool, batch)))
    assert torch.equal(again[0].data, pool.data) and (again[0].pages, again[0].heads, again[0].fp8) == (3, 2, False)
    assert again[0]._head == (again[0].data.data_ptr(), 3) and again[0]._head != pool._head
    assert again[1].rows == 3 and torch.equal(again[1].table, batch.table)
    assert again[1]._arrays == (again[1].starts.data_ptr(), again[1].lengths.data_ptr(), again[1].table.data_ptr(), 2)
    assert again[1]._arrays[:3] != batch._arrays[:3]


def test_workspace_of_any_call_has_the_stated_bound(lib):
    """Sizes from a single row to the largest call, both kinds of pages: never nothing, never more than the header says."""
    for rows in (0, 1, 17, 40, 1000, 1 << 20):
        for B in (1, 7, 1024):
            for kv, heads in ((1, 1), (4, 32), (24, 24)):
                for pages in (1, 16, 17, 2000, 1 << 20):
                    for flags in (0, _lib.PAGED_FP8, _lib.PAGED_FP8 | _lib.PAGED_CAUSAL):
                        a = _lib.PagedArgs(n_pages=1, B=B, table_pages=pages, rows=rows, kv_heads=kv, heads=heads, D=128, flags=flags)
                        assert 0 < lib.pkh3_paged_workspace_bytes(C.byref(a)) <= 103_000_000


def test_tensors_that_moved_are_taken_where_they_are():
    """A batch's or a pool's tensor that was resized, set or given other data since the last call: its checks are made again, and the call gets the new address."""
    from pika_h3_flex_amd import paged

    cache = pk.PagedKV(3, 2, device="cpu")
    batch = pk.PagedBatch.build([1, 2], [5, 70], [[2], [0, 1]], device="cpu")
    look = lambda: paged._place(cache, batch)   # noqa: E731
    look()
    batch.lengths.data = torch.tensor([7, 71], dtype=torch.int32)
    look()
    assert batch._arrays[1] == batch.lengths.data_ptr()
    wide = torch.full((2, 9), -1, dtype=torch.int32)
    batch.table.set_(wide[:, :5])
    look()
    assert batch._arrays[2:] == (wide.data_ptr(), 9) and batch._sizes == (2, 5)
    cache.data.data = torch.zeros_like(cache.data)
    look()
    assert cache._head == (cache.data.data_ptr(), 3)
    for change, back in ((lambda: batch.lengths.resize_(1), lambda: batch.lengths.resize_(2)), (lambda: batch.starts.resize_(400), lambda: batch.starts.resize_(3)),
                         (lambda: batch.table.resize_(3, 5), lambda: batch.table.resize_(2, 5)), (lambda: cache.data.resize_(2, 2, 32768), lambda: cache.data.resize_(3, 2, 32768)),
                         (lambda: batch.lengths.set_(torch.zeros(4, dtype=torch.int32)[::2]), lambda: batch.lengths.set_(torch.zeros(2, dtype=torch.int32)))):
        change()
        for _ in range(2):
            with pytest.raises(ValueError):
                look()
        back()
        look()
    assert batch._arrays[:2] == (batch.starts.data_ptr(), batch.lengths.data_ptr()) and cache._head[0] == cache.data.data_ptr()
    batch.lengths.data = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="int32"):
        look()
