// Attention of new rows over a paged K/V cache: softmax(norm_rope(q) K^T * scale) V, every sequence over its own pages.
//
// The work.  The new rows of a sequence times the query heads that share one of the cache's heads are the query rows of a (sequence, kv
// head): row r is token r / G, head r % G of the group, so that the heads of a group read their keys once.  A block of RB of them
// is a unit; its tiles are the pages that its last row sees.  How many units there are and how long each of them is, the host does not
// know: it is in the batch's arrays.  So the tiles of all units are laid end to end and every workgroup takes an equal run of them,
// whatever the lengths: it adds the sequences up, finds where its run begins, and walks from there.  A unit that lies in one run is
// finished there; of one that is cut every workgroup leaves its part (un-normalised O, running maximum, row sum, all fp32) in a
// slot of its own, and a second launch adds the parts up in the order of the runs.  Nothing waits for anything, and the bits
// do not depend on who is first.  (At most two parts a workgroup: the unit its run begins in and the one it ends in.)
//
// The arithmetic is that of the dense calls (see pkh3_attn_fwd.hip): S^T = K Q'^T and O^T += V^T P^T on the 16x16x32 MFMA, P
// from one to the other in its lane, running maximum raised when exceeded by 2^8.  Queries without norm and rotation are taken as they are, and the softmax
// scale multiplies S^T (in fp32, in the subtraction of the maximum).  After norm or rotation Q' is rounded to bf16, as in the dense calls: to
// keep what that leaves would be half as many products of S^T again, and registers that the tile form does not have.  Blocks of 16 rows keep it.
// e4m3 keys times their power of two are exact in bf16; the scale of a value's key goes to P instead, exact there as well.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "pkh3_paged.h"
#include "pkh3_internal.h"
#include "pkh3_wave.h"

namespace pkh3 {

constexpr int kSplitWaves = 4;

// The lane's number, made where it is used
__device__ __forceinline__ int lane_here() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// ---- the tile space ----

__device__ __forceinline__ Sequence attended(const PagedParams& p, int b) {
  return make_attended(p.starts[b], p.starts[b + 1], p.lengths[b], p.rows, p.table_pages, p.causal);
}
__device__ __forceinline__ Sequence uniform_attended(const PagedParams& p, int b) {
  return make_attended(uniform_int(p.starts, b), uniform_int(p.starts, b + 1), uniform_int(p.lengths, b), p.rows, p.table_pages, p.causal);
}

__device__ __forceinline__ int blocks_of(const PagedParams& p, const Sequence& s, int rb) { return blocks_of(s, p.G, rb); }
__device__ __forceinline__ int block_tiles(const PagedParams& p, const Sequence& s, int rb, int j) { return block_tiles(s, p.G, p.causal, rb, j, p.table_pages); }
__device__ __forceinline__ int row_keys(const PagedParams& p, const Sequence& s, int r) { return row_keys(s, p.G, p.causal, r); }
__device__ __forceinline__ int block_cost(const PagedParams& p, const Sequence& s, int rb, int j) { return block_cost(s, p.G, rb, j); }
__device__ __forceinline__ int64_t unit_cost(const PagedParams& p, const Sequence& s, int rb, int j) {
  return unit_length(block_tiles(p, s, rb, j), block_cost(p, s, rb, j));
}

// Where a run begins: sequence, head, block and tile, and how far in the space of all tiles the unit and the tile begin.
struct Place {
  int b, h, j, t;
  int64_t unit, pos;
};

// The sums of the tiles of all sequences in `cum`, by the whole workgroup.  Blocks of a causal sequence differ in length: where
// there are more than a few, a wave adds them up together.
__device__ __forceinline__ void sum_tiles(const PagedParams& p, int64_t* cum, int rb) {
  constexpr int kAlone = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  for (int at = 64 * wave; at < p.B; at += 64 * waves) {
    const int b = at + lane;
    int64_t mine = 0;
    bool many = false;
    if (b < p.B) {
      const Sequence s = attended(p, b);
      const int blocks = blocks_of(p, s, rb);
      many = p.causal && blocks > kAlone;
      if (!p.causal) mine = blocks ? (blocks - 1) * unit_cost(p, s, rb, 0) + unit_cost(p, s, rb, blocks - 1) : 0;
      else if (!many)
        for (int j = 0; j < blocks; ++j) mine += unit_cost(p, s, rb, j);
    }
    for (unsigned long long left = __ballot(many); left; left &= left - 1) {
      const int l = __ffsll((unsigned long long)left) - 1;
      const Sequence s = uniform_attended(p, __builtin_amdgcn_readfirstlane(at + l));
      const int blocks = blocks_of(p, s, rb);
      int64_t sum = 0;
      for (int j = lane; j < blocks; j += 64) sum += unit_cost(p, s, rb, j);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      if (lane == l) mine = sum;
    }
    if (b < p.B) cum[b + 1] = mine * p.H;
  }
  prefix_sums(cum, p.B);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x), hi = __builtin_amdgcn_readfirstlane((unsigned)((uint64_t)x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The boundary at `pos`, brought to a tile (see boundary_tile); 0 <= pos < cum[B]
__device__ __forceinline__ Place find_place(const PagedParams& p, const int64_t* cum, int rb, const Shares& sh, int64_t pos) {
  Place at;
  at.b = find_sequence(cum, p.B, pos);
  const Sequence s = uniform_attended(p, at.b);
  const int blocks = blocks_of(p, s, rb);
  const int64_t per_head = divided(cum[at.b + 1] - cum[at.b], p.H);
  int64_t rest = pos - cum[at.b];
  at.h = __builtin_amdgcn_readfirstlane((int)divided(rest, per_head));
  rest -= at.h * per_head;
  if (blocks == 1) {
    at.j = 0;
  } else if (!p.causal) {
    at.j = __builtin_amdgcn_readfirstlane(min((int)divided(rest, unit_cost(p, s, rb, 0)), blocks - 1));
    rest -= at.j * unit_cost(p, s, rb, 0);
  } else {
    const int lane = threadIdx.x & 63;
    for (int first = 0;; first += 64) {
      int64_t x = first + lane < blocks ? unit_cost(p, s, rb, first + lane) : 0;
      const int64_t own = x;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
      const unsigned long long past = __ballot(x > rest);
      if (past || first + 64 >= blocks) {
        const int l = past ? __ffsll((unsigned long long)past) - 1 : blocks - 1 - first;
        at.j = __builtin_amdgcn_readfirstlane(first + l);
        rest -= __shfl(x - own, l);
        break;
      }
      rest -= __shfl(x, 63);
    }
  }
  const int nt = block_tiles(p, s, rb, at.j), cost = block_cost(p, s, rb, at.j);
  at.unit = uniform64(pos - rest);
  at.t = __builtin_amdgcn_readfirstlane(boundary_tile(sh, rest, nt, cost));
  at.pos = at.unit + tile_place(at.t, cost);
  return at;
}

// The run of this workgroup: which one, what it costs, the unit and tile it begins at, and how long runs are.  False: none.  The first wave finds its beginning, the
// second its end, `found` (LDS) tells the others.  Leaves what the second launch has to know of the run's beginning.
struct Run {
  int rank;
  int64_t left, length;
};
__device__ __forceinline__ bool find_run(const PagedParams& p, const int64_t* cum, int64_t* found, int rb, Run& run, Place& at) {
  const Shares sh = shares_of(cum[p.B], gridDim.x, rb, p.whole != 0);
  run.rank = rank_of(blockIdx.x, sh);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.cuts[0] = i32x4{sh.n, 0, 0, 0};
  if (run.rank < 0 || sh.total == 0) return false;
  if (threadIdx.x < 64) {
    const Place x = find_place(p, cum, rb, sh, sh.begin(run.rank));
    if (threadIdx.x == 0) {
      found[0] = (int64_t)(uint32_t)x.b << 32 | (uint32_t)x.h;
      found[1] = (int64_t)(uint32_t)x.j << 32 | (uint32_t)x.t;
      found[2] = x.pos;
      if (run.rank > 0) {
        const Sequence s = uniform_attended(p, x.b);
        const int nt = block_tiles(p, s, rb, x.j);
        p.cuts[run.rank] = i32x4{x.b, x.h, x.j, parts_at(sh, run.rank, x.unit, x.t, nt, block_cost(p, s, rb, x.j))};
      }
    }
  } else if (threadIdx.x < 128) {
    const int64_t end = run.rank + 1 < sh.n ? find_place(p, cum, rb, sh, sh.begin(run.rank + 1)).pos : sh.total;
    if (threadIdx.x == 64) found[3] = end;
  }
  run.length = uniform64(sh.run());
  __syncthreads();
  const int64_t bh = uniform64(found[0]), jt = uniform64(found[1]);
  at.b = (int)(bh >> 32), at.h = (int)bh, at.j = (int)(jt >> 32), at.t = (int)jt;
  run.left = uniform64(found[3] - found[2]);
  return run.left > 0;
}

// On to the next unit of a run with `left` to go.  False where there is none.
__device__ __forceinline__ bool next_unit(const PagedParams& p, Place& at, Sequence& s, int& blocks, int rb, int64_t left) {
  if (left <= 0) return false;
  if (++at.j < blocks) return true;
  at.j = 0;
  if (++at.h < p.H) return true;
  at.h = 0;
  do {
    if (++at.b >= p.B) return false;
    s = uniform_attended(p, at.b);
  } while (s.n == 0);
  blocks = blocks_of(p, s, rb);
  return true;
}

// 1 / l; rows without a key: 0.  (A sum that is not a number stays one.)
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }

// A part of a unit in the scratch: RB rows of 128 (in the tile form blocks of 16 rows, as the lanes hold them), then the rows' maxima, then their sums
constexpr int kCutFloats = 4 * kMaxShares;   // of the records in front of the parts
__host__ __device__ constexpr int part_floats(int rb) { return rb * (kD + 2); }

// ---- the split form: few query rows, the waves of a workgroup share the keys out ----
//
// A unit is one or two blocks of 16 query rows, and each of the four waves walks a quarter of the run's part of it in 32-key halves.  No two
// waves read the same images, so these go straight from memory into the registers of the MFMAs: no LDS and no barrier in the loop, the
// next keys asked for under the softmax, the values under S^T.  The waves' results meet in LDS.  Bound by the bytes of K and V: one token of 24 heads
// over 124,992 keys 261 us, 5.9 TB/s; eight over up to 48,360 in e4m3 214, 5.7 TB/s.  REST: what the rounding of Q' to bf16 leaves is kept, in
// bf16 as well, and its products with K are added to S^T; under the bytes of 16 rows that is free (the error of a result against 64 bits falls from 0.0029 of
// it to 0.0024, where the rounding of P and of the result is left), with 32 rows, whose keys come out of L2, calls took up to 1.8 times as long.

template <int QB>
struct SplitState {
  bf16x8 qf[QB][4];
  f32x4 o[8][QB];
  float m[QB], l[QB];
};

// The weights of one half tile, the running maximum and the row sums.  ve: exponents of the values' scales.
template <bool FP8, int QB>
__device__ __forceinline__ void split_softmax(SplitState<QB>& w, const f32x4 (&s)[2][QB], bf16x8 (&pf)[QB], const unsigned (&ve)[2], float c) {
  float alpha[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float mx = s[0][qb][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kb][qb][i]);
    mx = max_across_groups(mx) * c;
    const float m_new = mx > w.m[qb] + kRescaleSlack ? mx : w.m[qb];
    alpha[qb] = __builtin_amdgcn_exp2f(w.m[qb] - m_new);
    w.m[qb] = m_new;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[j >> 2][qb][j & 3], c, -m_new));
      sum += e;
      pf[qb][j] = (__bf16)(FP8 ? e * exponent_scale((ve[j >> 2] >> (8 * (j & 3))) & 0xffu) : e);
    }
    w.l[qb] = w.l[qb] * alpha[qb] + sum;
  }
  bool raised = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) raised |= alpha[qb] != 1.0f;
  if (__any(raised)) {
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[db][qb][i] *= alpha[qb];
  }
}

// Values of keys that do not exist are zero, whatever their places hold (a weight of zero alone does not do it): in the pieces as they were
// loaded, eight bf16 or two times eight e4m3 of the keys v_image_key(g, 0 .. 7).
template <bool FP8, int N>
__device__ __forceinline__ void clear_missing(i32x4 (&v)[N], int there, int g) {
  int keep[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (!FP8) {
      keep[i] = (v_image_key(g, 2 * i) < there ? 0xffff : 0) | (v_image_key(g, 2 * i + 1) < there ? 0xffff0000 : 0);
    } else {
      keep[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) keep[i] |= v_image_key(g, 4 * (i & 1) + j) < there ? 0xff << (8 * j) : 0;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] &= keep[i];
}

// The address of query row r of (sequence, kv head) in a [rows, heads, 128] tensor, and its token
__device__ __forceinline__ int64_t row_offset(const PagedParams& p, const Sequence& s, int h, int r, int64_t ss, int64_t sh, int& token) {
  token = p.G.token(r);
  return (int64_t)(s.first + token) * ss + (int64_t)(h * p.G.n + r - token * p.G.n) * sh;
}

// Sixteen query rows from r0 on (those past the last are the last one again), as they lie in memory ..
__device__ __forceinline__ void ask_queries(const PagedParams& p, const Sequence& s, int h, int r0, Rows16& q, int lane) {
  const int last = s.n * p.G.n - 1;
  int token;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q.v[i] = *(const i32x4*)(p.q + row_offset(p, s, h, min(r0 + 4 * i + (lane >> 4), last), p.q_ss, p.q_sh, token) + (lane & 15) * 16);
}
// .. and through norm and rotation, in the lane order of the B images, by way of 4 KiB of LDS of the wave's own
__device__ __forceinline__ void queries_moved(const PagedParams& p, const Sequence& s, int r0, const Rows16& q, const NormLanes& norm, char* turn, int lane,
                                              float factor, float (&x)[32]) {
  Rows16 cos, sin;
  RopeQuarter rope;
  if (p.rope_mode != 0) {
    const int last = s.n * p.G.n - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = p.G.token(min(r0 + 4 * i + (lane >> 4), last));
      const int64_t at = (int64_t)(s.first + token) * (kD / 2 * (int)sizeof(float)) + (lane & 15) * 16;
      cos.v[i] = *(const i32x4*)((const char*)p.cos_t + at);
      sin.v[i] = *(const i32x4*)((const char*)p.sin_t + at);
    }
  }
  bf16x8 raw[4];
  turn_elements(q, raw, turn, lane);
  if (p.rope_mode != 0) {
    turn_table(cos, rope.c, p.rope_mode, turn, lane);
    turn_table(sin, rope.s, p.rope_mode, turn, lane);
  }
  norm_row(x, raw, p.norm_w != nullptr, p.eps, norm, factor);
  rope_row(x, p.rope_mode, rope);
}

template <bool FP8, int QB, bool REST>
__global__ __launch_bounds__(64 * kSplitWaves, 2) void paged_split_kernel(PagedParams p) {
  constexpr int RB = 16 * QB, NW = kSplitWaves;
  constexpr int kSlot = QB * 8 * 64 * 16;                      // one wave's O^T in fp32
  constexpr int kRecord = FP8 ? kPageRecord8 : kPageRecord16;
  constexpr int kN = FP8 ? 4 : 8;                              // 16-byte pieces of a lane of a half tile's K, and of its V
  constexpr int kVOff = FP8 ? kK8TileBytes : kKTileBytes;
  constexpr int kScaleOff = kK8TileBytes + kVTileBytes / 2;
  __shared__ __attribute__((aligned(1024))) char part[NW * kSlot];
  static_assert(!REST || QB == 1, "see above");
  __shared__ __attribute__((aligned(1024))) char rows[(REST ? 2 : 1) * QB * 4096];   // Q' in bf16, and what that leaves
  __shared__ float part_m[NW][QB][16], part_l[NW][QB][16];
  static_assert((kMaxSequences + 1) * sizeof(int64_t) <= sizeof(part), "the sums lie where the waves' results meet afterwards");
  const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int64_t* cum = (int64_t*)part;
  sum_tiles(p, cum, RB);
  __shared__ int64_t found[4];
  Run run;
  Place at;
  if (!find_run(p, cum, found, RB, run, at)) return;
  int64_t left = run.left;
  Sequence s = uniform_attended(p, at.b);
  int blocks = blocks_of(p, s, RB);
  if (at.t == block_tiles(p, s, RB, at.j)) {
    at.t = 0;
    if (!next_unit(p, at, s, blocks, RB, left)) return;
  }

#pragma unroll 1
  while (left > 0) {
    const int nt = block_tiles(p, s, RB, at.j), take = tiles_left(left, at.t, nt, 1);
    __syncthreads();                                           // the sums, or the results of the unit before, are read
    SplitState<QB> w;
    int sees[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) sees[qb] = row_keys(p, s, at.j * RB + 16 * qb + c16);
    const int all_see = __builtin_amdgcn_readfirstlane(row_keys(p, s, at.j * RB));   // the first row sees least
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) w.o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) w.m[qb] = kNoMax, w.l[qb] = 0.f;

    const int first = 2 * at.t + wave * 2 * take / NW, end = 2 * at.t + (wave + 1) * 2 * take / NW;
    const char* head = p.pages + (int64_t)at.h * kRecord;
    auto record = [&](int id) { return head + (int64_t)max(id, 0) * p.page_stride; };
    i32x4 kf[kN];
    unsigned ke[2] = {0, 0};
    int id = -1;
    auto ask_k = [&](int page, int half) {
      const char* r = record(page);
#pragma unroll
      for (int j = 0; j < kN; ++j) kf[j] = *(const i32x4*)(r + half * (kN * 1024) + (j * 64 + lane) * 16);
      if constexpr (FP8) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) ke[kb] = ((const unsigned char*)r)[kScaleOff + 32 * half + 16 * kb + c16];
      }
    };
    Rows16 q;
    NormLanes norm;
    if (wave < QB) {                                           // (on their way before the page is known)
      ask_queries(p, s, at.h, at.j * RB + 16 * wave, q, lane);
      load_norm_lanes(norm, p.norm_w, lane);
    }
    if (first < end) {
      id = uniform_page(p, at.b, first >> 1);
      ask_k(id, first & 1);
    }
    if (wave < QB) {
      float x[32];
      queries_moved(p, s, at.j * RB + 16 * wave, q, norm, part + wave * 4096, lane, 1.0f, x);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        bf16x8 img, rest;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          img[j] = (__bf16)x[8 * ks + j];
          rest[j] = (__bf16)(x[8 * ks + j] - (float)img[j]);
        }
        char* to = rows + ((wave * 4 + ks) * 64 + lane) * 16;
        *(bf16x8*)to = img;
        if constexpr (REST) *(bf16x8*)(to + QB * 4096) = rest;
      }
    }
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) w.qf[qb][ks] = *(const bf16x8*)(rows + ((qb * 4 + ks) * 64 + lane) * 16);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    auto rest = [&](int qb, int ks) { return *(const bf16x8*)(rows + QB * 4096 + ((qb * 4 + ks) * 64 + lane) * 16); };
#pragma unroll 1
    for (int i = first; i < end; ++i) {
      const int next = min(i + 1, end - 1);
      const int id_next = uniform_page(p, at.b, next >> 1);
      const int half = i & 1;
      i32x4 vf[kN];
      unsigned ve[2] = {0, 0};
      const char* r = record(id);
#pragma unroll
      for (int j = 0; j < kN; ++j) vf[j] = *(const i32x4*)(r + kVOff + half * (kN * 1024) + (j * 64 + lane) * 16);
      if constexpr (FP8) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) ve[kb] = *(const unsigned*)(r + kScaleOff + 64 + 32 * half + 16 * kb + 4 * g4);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x4 sT[2][QB];
      if constexpr (!FP8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {                          // image (ks, kb) = (j / 2, j % 2)
          if constexpr (REST) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) sT[j & 1][qb] = PKH3_MFMA16(__builtin_bit_cast(bf16x8, kf[j]), rest(qb, j >> 1), j < 2 ? zero : sT[j & 1][qb]);
          }
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
            sT[j & 1][qb] = PKH3_MFMA16(__builtin_bit_cast(bf16x8, kf[j]), w.qf[qb][j >> 1], !REST && j < 2 ? zero : sT[j & 1][qb]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {                          // chunk (kb, c2) = (j / 2, j % 2): images ks = 2*c2, 2*c2 + 1
          const float scale = exponent_scale(ke[j >> 1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bf16x8 a = expand_fp8(kf[j][2 * e], kf[j][2 * e + 1], scale);
            const int ks = 2 * (j & 1) + e;
            if constexpr (REST) {
#pragma unroll
              for (int qb = 0; qb < QB; ++qb) sT[j >> 1][qb] = PKH3_MFMA16(a, rest(qb, ks), ks == 0 ? zero : sT[j >> 1][qb]);
            }
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) sT[j >> 1][qb] = PKH3_MFMA16(a, w.qf[qb][ks], !REST && ks == 0 ? zero : sT[j >> 1][qb]);
          }
        }
      }
      ask_k(id_next, next & 1);
      __builtin_amdgcn_sched_barrier(0);
      // of this half: keys that exist, and that every query sees
      const int there = id < 0 ? 0 : s.keys - 32 * i;
      if (min(there, all_see - 32 * i) < 32) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * kb + 4 * g4 + e >= min(there, sees[qb] - 32 * i)) sT[kb][qb][e] = -INFINITY;
        clear_missing<FP8>(vf, there, g4);
        if constexpr (FP8) {                                   // (nor may their scales be anything but numbers)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * kb + 4 * g4 + e >= there) ve[kb] &= ~(0xffu << (8 * e));
        }
      }
      bf16x8 pf[QB];
      split_softmax<FP8, QB>(w, sT, pf, ve, p.c);
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        bf16x8 v;
        if constexpr (!FP8) v = __builtin_bit_cast(bf16x8, vf[db]);
        else v = expand_fp8(vf[db >> 1][2 * (db & 1)], vf[db >> 1][2 * (db & 1) + 1], 1.0f);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) w.o[db][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[qb], w.o[db][qb], 0, 0, 0);
      }
      id = id_next;
    }
    // (the last products are written back before anything reads them, whatever the compiler places here)
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) asm volatile("s_nop 15" : "+v"(w.o[db][qb])::"memory");

    // the waves' results meet: `part` was the queries' turning place until the barrier above
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) *(f32x4*)(part + wave * kSlot + ((db * QB + qb) * 64 + lane) * 16) = w.o[db][qb];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float l = wave_sum_groups(w.l[qb]);
      if (g4 == 0) part_l[wave][qb][c16] = l, part_m[wave][qb][c16] = w.m[qb];
    }
    __syncthreads();
    const bool finished = at.t == 0 && take == nt;
    float* slot = p.partials + part_slot(run.rank, at.t == 0) * part_floats(RB);
    const int row = threadIdx.x >> 4, chunk = threadIdx.x & 15;   // 8 columns of one of 16 rows
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = at.j * RB + 16 * qb + row;
      if (r >= s.n * p.G.n) continue;
      float top = kNoMax, l = 0.f, a[NW];
#pragma unroll
      for (int j = 0; j < NW; ++j) top = fmaxf(top, part_m[j][qb][row]);
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        a[j] = __builtin_amdgcn_exp2f(part_m[j][qb][row] - top);
        l += a[j] * part_l[j][qb][row];
      }
      f32x4 sum[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[e] = zero;
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          // columns 8*chunk + 4*e .. +3: block db = chunk / 2, lane group 2*(chunk % 2) + e
          const f32x4 t = *(const f32x4*)(part + j * kSlot + (((chunk >> 1) * QB + qb) * 64 + 16 * (2 * (chunk & 1) + e) + row) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[e][i] += a[j] * t[i];
        }
      }
      if (finished) {
        const float inv = inverse_sum(l);
        bf16x8 out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = (__bf16)(sum[i >> 2][i & 3] * inv);
        int token;
        *(bf16x8*)(p.o + row_offset(p, s, at.h, r, p.o_ss, p.o_sh, token) + chunk * 16) = out;
      } else {
        *(f32x4*)(slot + (16 * qb + row) * kD + chunk * 8) = sum[0];
        *(f32x4*)(slot + (16 * qb + row) * kD + chunk * 8 + 4) = sum[1];
        if (chunk == 0) {
          slot[RB * kD + 16 * qb + row] = top;
          slot[RB * (kD + 1) + 16 * qb + row] = l;
        }
      }
    }
    left -= take + (at.t == 0 ? kUnitTiles : 0);
    at.t = 0;
    if (!next_unit(p, at, s, blocks, RB, left)) return;
  }
}

// ---- the tile form: many query rows, all waves of a workgroup share every key tile ----
// A unit is 384 query rows, 32 a wave; twelve waves are three a SIMD, one workgroup a CU.  The loop is that of the dense calls: K/V tiles in an LDS ring
// of three, two tiles ahead of the products, one barrier a tile.  The page of a tile is looked up a step before its copy.  (Units of 128 rows
// in four waves, three workgroups a CU, in halves of tiles, were behind on all but some calls of a few dozen rows, and there by 2 %: 1,560 rows over
// 48,360 keys 881 us here, 1,355 there; 120 rows over 20,000 keys 58 and 72; three requests against 77 to 512 keys 212 and 218.)
// Eight-bit pages come to LDS as they are, one step further ahead, and are expanded there to the bf16 images of the loop, a share of
// them by every wave, under the products of the step before: once for all waves, and the loop has no conversions.
//

// The kernel's arguments, read again where they are used: those of the queries and outputs, kept through the loop, take the scalar registers that its copies need.
__device__ __forceinline__ PagedParams arguments_here() {
  PagedParams args;
  auto* a = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  __builtin_memcpy(&args, (const char*)a, sizeof(args));
  return args;
}

constexpr int kTileWaves = 12, kTileRows = 32 * kTileWaves;
constexpr int kImageBytes = kKTileBytes + kVTileBytes;                    // of a tile's bf16 images
constexpr int kRawBytes = kPageRecord8;                                   // of a tile's e4m3 values and scales, as they come
constexpr int kTurnBytes12 = kTileWaves * 4096;                           // where queries and outputs are turned around
// bf16: a ring of three tiles, the turning place where the third goes and behind it.  e4m3: two tiles of images (the turning place), two as they come
template <bool FP8>
constexpr int tile_lds_bytes() {
  static_assert(2 * kImageBytes >= kTurnBytes12 && kTurnBytes12 > kImageBytes, "the places");
  return FP8 ? 2 * kImageBytes + 2 * kRawBytes : 2 * kImageBytes + kTurnBytes12;
}

// A query's running maximum in the log2 domain, negative.  FOLD: the softmax scale and log2 e ride in Q', which norm or rotation has rounded to bf16 anyway,
// and the sums of S^T begin with it (a quad, as the MFMA takes it), so that they are the exponents of the weights as they come out.  Otherwise Q' is the
// query as it is, and the scale multiplies in the subtraction.
template <bool FOLD>
struct Running {
  f32x4 neg[FOLD ? 2 : 1];
  float m[FOLD ? 1 : 2];
  __device__ __forceinline__ float negative(int qb) const {
    if constexpr (FOLD) return neg[qb][0];
    else return m[qb];
  }
  __device__ __forceinline__ f32x4 first(int qb) const {
    if constexpr (FOLD) return neg[qb];
    else return f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void set(int qb, float x) {
    if constexpr (FOLD) neg[qb] = f32x4{x, x, x, x};
    else m[qb] = x;
  }
};

// S^T of a tile (see qk_tile: images read AHEAD of their products)
template <int AHEAD, bool FOLD>
__device__ __forceinline__ void tile_qk(WaveState<false>& w, const Running<FOLD>& run, const char* kbuf, int lane) {
  bf16x8 kf[16];                                                          // (half, ks, kb2)
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) kf[i] = *(const bf16x8*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int ks = (i >> 1) & 3, kb = 2 * (i >> 3) + (i & 1);
#pragma unroll
    for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.s[kb][qb] = PKH3_MFMA16(kf[i], w.qf[qb][ks], ks == 0 ? run.first(qb) : w.s[kb][qb]);
    if (i + AHEAD < 16) kf[i + AHEAD] = *(const bf16x8*)(kbuf + ((i + AHEAD) * 64 + lane) * 16);
  }
  PKH3_SGB(kSgDsRead, AHEAD);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    PKH3_SGB(kSgMfma, 2);
    if (i + AHEAD < 16) PKH3_SGB(kSgDsRead, 1);
  }
}

// see tile_softmax: beside weights that began at 1 or more and go down by 2^-126 at most before they are gone themselves
constexpr float kSomeWeight = 0x1p-100f;

// The weights of a tile, as operands of P.V (see softmax_blocks of the dense calls).  MASKED: lim[qb] keys of it exist for the lane's query.
// The maximum of a query is that of its first tile with keys, and is raised when exceeded by 2^8.  Whether any is, the largest exponent tells as an integer (any
// positive float is a larger one than any negative, and NaN than all): no order among the negative ones is needed.  A lane that has no weight yet looks.
template <bool MASKED, bool FOLD>
__device__ __forceinline__ void tile_softmax(WaveState<false>& w, Running<FOLD>& run, bf16x8 (&pf)[2][2], float c, const int (&lim)[2], int lane) {
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int mine = lim[qb] - 4 * (lane >> 4);                           // (against constants from here on)
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = w.s[kb][qb][i];
        if constexpr (!FOLD) x = fmaf(x, c, run.negative(qb));
        if constexpr (MASKED) x = 16 * kb + i >= mine ? -INFINITY : x;
        w.s[kb][qb][i] = x;
      }
  }
  int most = __float_as_int(w.s[0][0][0]);
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = max(most, __float_as_int(w.s[kb][qb][i]));
  if (__any(most > __float_as_int(kRescaleSlack) || w.l[0] == 0.f || w.l[1] == 0.f)) {
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      float top = w.s[0][qb][0];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, w.s[kb][qb][i]);
      top = max_across_groups(top);
      const float before = wave_sum_groups(w.l[qb]);
      const bool none = before == 0.f;                                    // no maximum yet
      const float up = none ? (top > -INFINITY ? top : 0.f) : top > kRescaleSlack ? top : 0.f;
      const float alpha = none ? 0.f : __builtin_amdgcn_exp2f(-up);
      run.set(qb, run.negative(qb) - up);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.s[kb][qb][i] -= up;
      // a lane without a weight whose query has some in others need not look again: it gets one that is nothing beside those
      w.l[qb] = none ? 0.f : fmaxf(w.l[qb] * alpha, kSomeWeight);
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[db][qb][i] *= alpha;
    }
  }
  const bf16x2 one2 = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      bf16x8 pk;
#pragma unroll
      for (int j = 0; j < 8; ++j) pk[j] = (__bf16)__builtin_amdgcn_exp2f(w.s[2 * half + (j >> 2)][qb][j & 3]);
      // row sum over the rounded weights, the same numbers P.V takes
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const bf16x2 pr = {pk[j], pk[j + 1]};
        w.l[qb] = __builtin_amdgcn_fdot2_f32_bf16(pr, one2, w.l[qb], false);
      }
      pf[half][qb] = pk;
    }
}

// O^T += V^T P^T of a tile, V images read four ahead of their products
__device__ __forceinline__ void tile_pv(WaveState<false>& w, const bf16x8 (&pf)[2][2], const char* vbuf, int lane) {
  bf16x8 vg[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) vg[i] = *(const bf16x8*)(vbuf + (i * 64 + lane) * 16);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.o[i & 7][qb] = PKH3_MFMA16(vg[i], pf[i >> 3][qb], w.o[i & 7][qb]);
    if (i + 4 < 16) vg[i + 4] = *(const bf16x8*)(vbuf + ((i + 4) * 64 + lane) * 16);
  }
}

// A wave's share of a tile's e4m3 values to bf16 images.  1 KiB of them, 16 values a lane, are two images.  A key's values have one scale: of K that is
// one per lane, of V one per value of the eight, applied as the value is converted (the conversion takes a power of two along).
__device__ __forceinline__ void expand_tile(const char* raw, char* images, int wave, int lane) {
  const int g = lane >> 4, c = lane & 15;
  const char* scales = raw + kRawBytes - kPageScales;
#pragma unroll 1
  for (int piece = wave; piece < 16; piece += kTileWaves) {
    const i32x4 v = *(const i32x4*)(raw + (piece * 64 + lane) * 16);
    if (piece < 8) {                                                      // key block kb, images ks = 2*c2, 2*c2 + 1
      const int kb = piece >> 1, c2 = piece & 1;
      const float scale = exponent_scale((unsigned char)scales[16 * kb + c]);
      char* to = images + ((((kb >> 1) * 4 + 2 * c2) * 2 + (kb & 1)) * 64 + lane) * 16;
      *(bf16x8*)to = expand_fp8(v[0], v[1], scale);
      *(bf16x8*)(to + 2048) = expand_fp8(v[2], v[3], scale);
    } else {                                                              // (half, dbp), images db = 2*dbp, 2*dbp + 1
      const int half = (piece - 8) >> 2, dbp = piece & 3;
      unsigned e[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) e[kb] = *(const unsigned*)(scales + 64 + 32 * half + 16 * kb + 4 * g);
      char* to = images + kKTileBytes + ((half * 8 + 2 * dbp) * 64 + lane) * 16;
#pragma unroll
      for (int par = 0; par < 2; ++par) {
        *(bf16x8*)(to + par * 1024) = expand_fp8_keys(v[2 * par], v[2 * par + 1], e);
      }
    }
  }
}

// Values of keys that do not exist are zero (see clear_missing), in the V images of a tile in LDS
__device__ __forceinline__ void clear_missing_images(char* v, int there, int wave) {
#pragma unroll 1
  for (int n = wave; n < 16; n += kTileWaves) {                           // images: of a half 8
    const int lane = lane_here(), half = n >> 3;
    char* at = v + (n * 64 + lane) * 16;
    i32x4 piece[1] = {*(const i32x4*)at};
    clear_missing<false>(piece, there - 32 * half, lane >> 4);
    *(i32x4*)at = piece[0];
  }
}

template <bool FP8, bool FOLD>
__global__ __launch_bounds__(64 * kTileWaves, 1) void paged_tile_kernel(PagedParams p) {
  constexpr int RB = kTileRows, kRecord = FP8 ? kPageRecord8 : kPageRecord16;   // (a record is what a tile takes in the ring that pages are copied to)
  constexpr int kPieces = kRecord / 1024;                                 // whole KiB of it
  __shared__ __attribute__((aligned(1024))) char lds[tile_lds_bytes<FP8>()];
  __shared__ float norm_w[kD];                                            // from here a unit has them at once
  static_assert((kMaxSequences + 1) * sizeof(int64_t) <= sizeof(lds), "the sums");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int64_t* cum = (int64_t*)lds;
  sum_tiles(p, cum, RB);
  __shared__ int64_t found[4];
  Run run;
  Place at;
  if (!find_run(p, cum, found, RB, run, at)) return;
  int64_t left = run.left;
  Sequence s = uniform_attended(p, at.b);
  int blocks = blocks_of(p, s, RB);
  if (at.t == block_tiles(p, s, RB, at.j)) {
    at.t = 0;
    if (!next_unit(p, at, s, blocks, RB, left)) return;
  }
  char* copies = lds + (FP8 ? 2 * kImageBytes : 0);                       // the ring that pages are copied to
  // 4 KiB of the wave's own, for queries on their way in and outputs on their way out, that no copy ahead of the loop goes to
  char* turn = lds + (FP8 ? 0 : 2 * kImageBytes) + wave * 4096;

  // Pages of the tiles [64*n, 64*n + 64) of the sequence, one a lane.  (A scalar load in every step would have every wait for an LDS read behind it wait for
  // all of them: the two come back in no order.)
  int ids, ids_of = -1, ids_from = -1;
  auto page = [&](int tile) {
    if ((tile & ~63) != ids_from) {
      ids_of = at.b, ids_from = tile & ~63;
      const int t = ids_from + lane_here();
      ids = t < p.table_pages ? page_in_pool(p.table[(int64_t)at.b * p.table_stride + t], p.n_pages) : -1;
    }
    return __builtin_amdgcn_readlane(ids, tile & 63);
  };
  auto copy = [&](int id, int slot) {
    const char* record = p.pages + (int64_t)max(id, 0) * p.page_stride + (int64_t)at.h * kRecord;
    const unsigned lane_off = lane_here() * 16;
    char* d = copies + slot * kRecord;
#pragma unroll
    for (int n = 0; n < (kPieces + kTileWaves - 1) / kTileWaves; ++n) {
      const int piece = n * kTileWaves + wave;
      if ((n + 1) * kTileWaves <= kPieces || piece < kPieces) lds_dma16(record + piece * 1024, lane_off, d + piece * 1024);
    }
    if constexpr (FP8) {
      if (wave == kTileWaves - 1 && lane_off < kPageScales) lds_dma16(record + kPieces * 1024, lane_off, d + kPieces * 1024);
    }
  };
  // Workgroups that walk the same keys at the same time find them in their L2.  So they start where their neighbours are: with R tiles a run, every run inside a
  // unit begins at the multiple of R in it and goes on from its own first tile when it is through; a run over the end of one unit does the beginning of
  // the next first.  At any time all of a head are then at one of a few places, R apart, whatever block of rows they have.
  struct {
    int b, h, j, t;
    int64_t left;
  } later = {-1, 0, 0, 0, 0};                                             // the end of a unit that is done after the beginning of the next
  if (at.t > 0) {
    const int nt = block_tiles(p, s, RB, at.j), cost = block_cost(p, s, RB, at.j);
    const int64_t behind = left - (int64_t)(nt - at.t) * cost;
    Place next = at;
    Sequence next_s = s;
    int next_blocks = blocks;
    next.t = 0;
    if (next_unit(p, next, next_s, next_blocks, RB, behind)) {
      const int next_nt = block_tiles(p, next_s, RB, next.j);
      if (tiles_left(behind, 0, next_nt, block_cost(p, next_s, RB, next.j)) < next_nt) {
        later = {at.b, at.h, at.j, at.t, left - behind};
        at = next, s = next_s, blocks = next_blocks, left = behind;
      }
    }
  }
  auto advance = [&]() {
    if (next_unit(p, at, s, blocks, RB, left)) return true;
    if (later.b < 0) return false;
    at.b = later.b, at.h = later.h, at.j = later.j, at.t = later.t, left = later.left;
    s = uniform_attended(p, at.b);
    blocks = blocks_of(p, s, RB);
    later.b = -1;
    return true;
  };

  int id[3];                                                              // pages of this tile, the next and the one after it
  int nt, take, first, start;                                             // of the unit: its tiles, those of this run, its first one and where it starts
  auto tile_at = [&](int n) {                                             // the run's n-th tile
    const int i = start + n;
    return i < first + take ? i : i - take;
  };
  Rows16 ahead[2];
  auto begin_unit = [&]() {                                               // asks for everything the unit's loop begins with
    nt = block_tiles(p, s, RB, at.j);
    const int cost = block_cost(p, s, RB, at.j);
    take = tiles_left(left, at.t, nt, cost);
    left -= (int64_t)(take + (at.t == 0 ? kUnitTiles : 0)) * cost;
    first = start = at.t;
    if (first > 0 && first + take < nt) {
      const int apart = max((int)divided(run.length, cost), 1);
      const int place = (first + apart - 1) / apart * apart;
      start = __builtin_amdgcn_readfirstlane(place < first + take ? place : first);
    }
    if (at.b != ids_of) ids_from = -1;                                    // (mostly those of the unit before)
#pragma unroll
    for (int i = 0; i < 3; ++i) id[i] = page(tile_at(i));                 // (past the end: a page, or none, that is not used)
    copy(id[0], 0);
    copy(id[take > 1 ? 1 : 0], 1);                                        // (of a single tile: once more)
  };
  auto ask = [&](int qb) { ask_queries(arguments_here(), s, at.h, at.j * RB + 32 * wave + 16 * qb, ahead[qb], lane_here()); };
  if (threadIdx.x < kD) norm_w[threadIdx.x] = p.norm_w ? p.norm_w[threadIdx.x] : 1.0f;
  __syncthreads();                                                        // the sums are read
  begin_unit();
  ask(0), ask(1);
#pragma unroll 1
  for (;;) {
    // what is made of the lane's number is made where it is used: kept from unit to unit, or from the queries to the output, it does not fit the registers
    const int r0 = at.j * RB + 32 * wave, last = s.n * p.G.n - 1;
    const bool idle = r0 > last;                                          // a wave without rows: copies and barriers alone
    WaveState<false> w;
    if (!idle) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int l = lane_here();
        NormLanes norm;
        load_norm_lanes(norm, norm_w, l);
        float x[32];
        queries_moved(arguments_here(), s, r0 + 16 * qb, ahead[qb], norm, turn, l, FOLD ? p.c : 1.0f, x);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) w.qf[qb][ks][j] = (__bf16)x[8 * ks + j];
      }
    }
    const int all_see = __builtin_amdgcn_readfirstlane(row_keys(p, s, r0));   // keys that every row of the wave sees
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) w.o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) w.l[qb] = 0.f;
    Running<FOLD> run_max;
    run_max.set(0, 0.f), run_max.set(1, 0.f);

    int slot = 0, slot_prev = 2;
    if constexpr (FP8) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      expand_tile(copies, lds, wave, lane_here());
    }
    // One tile.  MASKED: some rows of the wave do not see all of its keys, or its page is not there.
    auto step = [&](int n, int i, auto masked, auto works) {
      constexpr bool MASKED = decltype(masked)::value, WORKS = decltype(works)::value;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      char* images = lds + slot * kImageBytes;
      int there = 0;
      if constexpr (MASKED) {
        there = id[0] < 0 ? 0 : s.keys - kTileKeys * i;
        if (there < kTileKeys) {
          clear_missing_images(images + kKTileBytes, there, wave);
          __syncthreads();
        }
      }
      if constexpr (WORKS) {
        tile_qk<MASKED || FOLD ? 3 : 4, FOLD>(w, run_max, images, lane_here());
      }
      if constexpr (!FP8) {
        if (n + 2 < take) copy(id[2], slot_prev);
        slot_prev = slot;
        slot = slot == 2 ? 0 : slot + 1;
      } else {
        if (n + 2 < take) copy(id[2], slot);
        if (n + 1 < take) expand_tile(copies + (slot ^ 1) * kRecord, lds + (slot ^ 1) * kImageBytes, wave, lane_here());
        slot ^= 1;
      }
      id[0] = id[1], id[1] = id[2], id[2] = page(tile_at(n + 3));
      if constexpr (WORKS) {
        int lim[2] = {};                                                  // (made here: kept from step to step, it does not fit the registers)
        if constexpr (MASKED) {
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) lim[qb] = min(there, row_keys(p, s, r0 + 16 * qb + (lane_here() & 15)) - kTileKeys * i);
        }
        bf16x8 pf[2][2];
        tile_softmax<MASKED, FOLD>(w, run_max, pf, p.c, lim, lane_here());
        tile_pv(w, pf, images + kKTileBytes, lane_here());
      }
    };
    // Whether a tile is masked differs from wave to wave, how many barriers it has does not: a tile with keys that do not exist, or a page that does not,
    // is masked for all.
    const int whole = all_see / kTileKeys;                               // tiles in front of this one are seen whole by all rows
    int n = 0, i = start;
    if (idle) {
#pragma unroll 1
      for (; n < take; i = tile_at(++n)) step(n, i, std::true_type{}, std::false_type{});
    }
    bool plain = i < whole && id[0] >= 0;
#pragma unroll 1
    while (n < take) {
#pragma unroll 1
      while (plain) {
        step(n, i, std::false_type{}, std::true_type{});
        i = tile_at(++n);
        plain = n < take && i < whole && id[0] >= 0;
      }
#pragma unroll 1
      while (n < take && !plain) {
        step(n, i, std::true_type{}, std::true_type{});
        i = tile_at(++n);
        plain = n < take && i < whole && id[0] >= 0;
      }
    }
    PKH3_MFMA_DRAIN(w);

    __syncthreads();                                                      // every wave is done reading: the ring is free
    // the next unit's first steps and queries are on their way while this one's rows go out
    const Sequence out_s = s;
    const int out_h = at.h;
    const bool finished = at.t == 0 && take == nt, begins = at.t == 0;
    at.t = 0;
    const bool more = advance();
    if (more) begin_unit();
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      ask(qb);                                                            // (without a next unit: rows of this one, which nobody takes)
      asm volatile("" ::: "memory");                                      // (one block after the other: both at once do not fit the registers)
      if (!idle) {
        const int out_lane = lane_here(), c16 = out_lane & 15, g4 = out_lane >> 4;
        const PagedParams args = arguments_here();
        const float l = wave_sum_groups(w.l[qb]);
        if (finished) {
          const float inv = inverse_sum(l);
#pragma unroll
          for (int db = 0; db < 8; ++db) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (__bf16)(w.o[db][qb][e] * inv);
            *(bf16x4*)(turn + c16 * 256 + (((2 * db + (g4 >> 1)) ^ c16) * 16) + 8 * (g4 & 1)) = v;
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int row = 4 * n + g4, r = r0 + 16 * qb + row;
            const bf16x8 v = *(const bf16x8*)(turn + row * 256 + ((c16 ^ row) * 16));
            int token;
            const int64_t to = row_offset(args, out_s, out_h, min(r, last), args.o_ss, args.o_sh, token);
            if (r <= last) *(bf16x8*)(args.o + to + c16 * 16) = v;
          }
        } else {
          // as the lanes hold it, whole KiB a store: by rows, 64 bytes of 16 of them a store, a workgroup's part took 12 us
          float* part = args.partials + part_slot(run.rank, begins) * part_floats(RB);
          float* to = part + (2 * wave + qb) * (16 * kD) + out_lane * 4;
          if (r0 + 16 * qb + c16 <= last) {
#pragma unroll
            for (int db = 0; db < 8; ++db) *(f32x4*)(to + db * 256) = w.o[db][qb];
            const int row = 32 * wave + 16 * qb + c16;
            if (g4 == 0) part[RB * kD + row] = l == 0.f ? kNoMax : -run_max.negative(qb), part[RB * (kD + 1) + row] = l;
          }
        }
      }
    }
    if (!more) return;
  }
}

// ---- the parts of units that more than one workgroup worked on ----
//
// Workgroup i of the launch in front, if its run begins inside a unit and is the first that does, has left in cut[i] which unit that is and how many
// runs share it: its parts are slot 1 of run i - 1 and slot 0 of i, i + 1, .., in that order.  This launch takes as long as what hangs together in it: eight
// parts are asked for at once.  (Found by every workgroup for itself, from the sums of the whole batch, the units were most of it:
// 41 to 52 us of 256 x 48 workgroups.)
constexpr int kPartsAtOnce = 8;

// `n` of eight parts (all of them in registers) to what is there of those in front
__device__ __forceinline__ void add_parts(float& top, float& l, f32x4& sum, const float (&m)[kPartsAtOnce], const float (&w)[kPartsAtOnce],
                                          const f32x4 (&o)[kPartsAtOnce], int n) {
  float most = top;
#pragma unroll
  for (int i = 0; i < kPartsAtOnce; ++i) most = i < n ? fmaxf(most, m[i]) : most;
  const float a0 = __builtin_amdgcn_exp2f(top - most);
  top = most;
  l *= a0;
#pragma unroll
  for (int k = 0; k < 4; ++k) sum[k] *= a0;
#pragma unroll
  for (int i = 0; i < kPartsAtOnce; ++i) {
    if (i < n) {
      const float a = __builtin_amdgcn_exp2f(m[i] - top);
      l += a * w[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += a * o[i][k];
    }
  }
}

// An eighth of a unit's rows a workgroup (blockIdx.y), 32 threads a row and part, four columns each: a row's parts are dealt out to four such groups (of
// units of 16 rows) or two, a single row's to eight.  (Eight rows a workgroup, a group each, their parts one after the other: 768 rows over 16,384 keys
// 60 us where it is 58 now, single tokens of 32 query heads over 8,192 keys 31.5 and 29.5.)
template <int RB>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p) {
  constexpr int kRows = RB / 8;
  __shared__ f32x4 part_sum[256];
  __shared__ float part_m[8], part_l[8];
  const int run = (int)blockIdx.x + 1;
  const i32x4 cut = p.cuts[run];
  if (run >= p.cuts[0][0] || cut[3] == 0) return;
  const Sequence s = uniform_attended(p, cut[0]);
  const int rows = min(RB, s.n * p.G.n - cut[2] * RB), row0 = (int)blockIdx.y * kRows;
  if (row0 >= rows) return;
  const int here = min(kRows, rows - row0), groups = here > 2 ? 2 : 8 / here;   // groups of 32 threads a row
  const int mine = threadIdx.x >> 5, col = (threadIdx.x & 31) * 4;
  const int row = min(row0 + mine / groups, rows - 1), sub = mine % groups;   // (those past the last: as the last, not stored)
  float top = kNoMax, l = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int i0 = sub; i0 < cut[3]; i0 += kPartsAtOnce * groups) {
    float m[kPartsAtOnce], w[kPartsAtOnce];
    f32x4 o[kPartsAtOnce];
#pragma unroll
    for (int i = 0; i < kPartsAtOnce; ++i) {
      const int part = min(i0 + i * groups, cut[3] - 1);
      const float* t = p.partials + part_slot(run - 1 + part, part == 0) * part_floats(RB);
      m[i] = t[RB * kD + row];
      w[i] = t[RB * (kD + 1) + row];
      o[i] = *(const f32x4*)(t + row * kD + col);
    }
    add_parts(top, l, sum, m, w, o, (cut[3] - i0 + groups - 1) / groups);
  }
  part_sum[threadIdx.x] = sum;
  if ((threadIdx.x & 31) == 0) part_m[mine] = top, part_l[mine] = l;
  __syncthreads();
  if (sub != 0 || mine / groups >= here) return;
  const float own = top;
  for (int g = 1; g < groups; ++g) top = fmaxf(top, part_m[mine + g]);
  const float a0 = __builtin_amdgcn_exp2f(own - top);
  l *= a0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum[e] *= a0;
  for (int g = 1; g < groups; ++g) {
    const float a = __builtin_amdgcn_exp2f(part_m[mine + g] - top);
    l += a * part_l[mine + g];
    const f32x4 o = part_sum[threadIdx.x + 32 * g];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += a * o[e];
  }
  const float inv = inverse_sum(l);
  bf16x4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (__bf16)(sum[e] * inv);
  int token;
  *(bf16x4*)(p.o + row_offset(p, s, cut[1], cut[2] * RB + row, p.o_ss, p.o_sh, token) + col * 2) = out;
}

// The same for the tile form, whose parts lie as its lanes hold them: blockIdx.y / 2 is a block of 16 rows, and wave w has the columns 16*db .. +15 of it for
// db = 4 * (blockIdx.y % 2) + w, four of row c a lane (16*g + c).  The rows go out by way of LDS.
__global__ __launch_bounds__(256) void paged_merge_tile_kernel(PagedParams p) {
  constexpr int RB = kTileRows;
  __shared__ __attribute__((aligned(16))) char turn[2048];
  const int run = (int)blockIdx.x + 1;
  const i32x4 cut = p.cuts[run];
  if (run >= p.cuts[0][0] || cut[3] == 0) return;
  const Sequence s = uniform_attended(p, cut[0]);
  const int rows = min(RB, s.n * p.G.n - cut[2] * RB), row0 = (int)(blockIdx.y >> 1) * 16, half = blockIdx.y & 1;
  if (row0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int at = min(row0 + c, rows - 1);                        // (rows that are not there: another's, and nothing is stored)
  const int col = row0 * kD + (4 * half + wave) * 256 + (16 * g + at - row0) * 4;
  float top = kNoMax, l = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int i0 = 0; i0 < cut[3]; i0 += kPartsAtOnce) {
    float m[kPartsAtOnce], w[kPartsAtOnce];
    f32x4 o[kPartsAtOnce];
#pragma unroll
    for (int i = 0; i < kPartsAtOnce; ++i) {
      const int part = min(i0 + i, cut[3] - 1);
      const float* t = p.partials + part_slot(run - 1 + part, part == 0) * part_floats(RB);
      m[i] = t[RB * kD + at];
      w[i] = t[RB * (kD + 1) + at];
      o[i] = *(const f32x4*)(t + col);
    }
    add_parts(top, l, sum, m, w, o, cut[3] - i0);
  }
  const float inv = inverse_sum(l);
  bf16x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = (__bf16)(sum[k] * inv);
  *(bf16x4*)(turn + c * 128 + (((2 * wave + (g >> 1)) ^ (c & 7)) * 16) + 8 * (g & 1)) = v;
  __syncthreads();
  const int out = threadIdx.x >> 3, chunk = threadIdx.x & 7;
  if (out >= 16 || row0 + out >= rows) return;
  int token;
  *(bf16x8*)(p.o + row_offset(p, s, cut[1], cut[2] * RB + row0 + out, p.o_ss, p.o_sh, token) + half * 128 + chunk * 16) =
      *(const bf16x8*)(turn + out * 128 + ((chunk ^ (out & 7)) * 16));
}

// ---- host ----

// The form of a call, from what the host knows of it; the table's width stands for the lengths.  Where the query rows of a (sequence, kv head) are 32 or fewer on
// the average, the split form.  Where they are more, it is still ahead while there is little to do: its blocks of 32 rows are twelve times as many, so that
// all CUs have some, and a tile of one takes 0.4 us against 2.6.  The tile form takes about as long as one of its units of up to 16 tiles (longer ones are
// cut), the split form as its tiles and kUnitTiles more a block: it goes as far as 900 blocks of 16 tiles.  (us, split / tile, bf16: 768 blocks over 128, 256,
// 512 and 1,024 keys 19 / 22, 21 / 26, 26 / 34, 36 / 50; 1,152 blocks over 256 keys 30 / 26; 8 heads over 4,096 keys, 384 rows 29 / 44, 768 rows 38 / 48, three
// such batches 55 / 55.)  It reads a key once for 32 rows: out of L2 that is well, but where a head's keys do not fit the 4 MB of one, or all
// of them the 32 MB of all, it falls behind sooner (8 heads over 16,384 keys: 96 rows 38 / 40, 192 rows 63 / 46; 64 heads over 4,096: 96 rows 69 / 41).
// The mean stands for every sequence: a chunk of 1,000 rows over 15,000 keys of 24 heads that is alone among 64 takes blocks of 16 rows, 903 us, and
// the tile form with one sequence in the batch, 179.
enum PagedForm { kSplit16, kSplit32, kTile };
static PagedForm form_of(int rows, int B, int H, int G, int table_pages, bool fp8) {
  const int64_t all = (int64_t)rows * G, used = std::max(1, std::min(rows, B));
  if (all <= 16 * used) return kSplit16;
  if (all <= 32 * used) return kSplit32;
  const int64_t tiles = (all / 32 + used) * H * (table_pages + kUnitTiles);
  const int64_t keys = (int64_t)table_pages * (fp8 ? 1 : 2) * 16384;      // bytes of a head's
  const bool cached = keys <= 4 << 20 && keys * H * used <= 32 << 20;
  return tiles <= (cached ? 900 * (std::min(table_pages, kWholeTiles) + kUnitTiles) : 8192) ? kSplit32 : kTile;
}
static int rows_of(PagedForm f) { return f == kSplit16 ? 16 : f == kSplit32 ? 32 : kTileRows; }
static int most_workgroups(PagedForm f) { return f == kTile ? kMaxShares / 2 : kMaxShares; }
// As many workgroups as there are places for, but no more than the units that there can be (two a unit, where these differ in length), or where they are cut
// the runs that they are worth (see shares_of): what finds itself without work has added the batch up first, beside those that have some (768
// rows over 1,024 keys of 3 heads, 72 units: 20 us among 512 workgroups, 16 among these).
static int workgroups_of(PagedForm f, const PagedParams& p, int cus) {
  const int rb = rows_of(f), places = (f == kTile ? 1 : 2) * cus;
  const int64_t units = ((int64_t)p.rows * p.G.n / rb + std::min(p.rows, p.B)) * p.H;
  const int64_t runs = p.whole ? units * (p.causal || p.B > 1 ? 2 : 1) : units * (p.table_pages + kUnitTiles) / (least_tiles(rb) + kUnitTiles) + 1;
  return std::min(most_workgroups(f), std::max(8, (int)std::min<int64_t>(places / 8 * 8, (runs + 7) / 8 * 8)));
}

size_t paged_attn_scratch(int rows, int B, int H, int G, int table_pages, bool fp8) {
  const PagedForm f = form_of(rows, B, H, G, table_pages, fp8);
  return (size_t)2 * most_workgroups(f) * part_floats(rows_of(f)) + kCutFloats;
}

// Tables of so few pages that whole units are no longer than cutting them and putting them together again: one launch.
static bool short_table(int table_pages) { return table_pages <= kWholeTiles; }

template <class Kernel, class Merge>
static hipError_t launch_form(Kernel kernel, int threads, Merge merge, int blocks, int grid, const PagedParams& p, hipStream_t st) {
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.whole) return e;
  hipLaunchKernelGGL(merge, dim3(grid - 1, blocks), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedParams& given, bool fp8, hipStream_t st) {
  PagedParams p = given;
  p.whole = short_table(p.table_pages);
  int cus = 0;
  const hipError_t e = device_cu_count(&cus);
  if (e != hipSuccess) return e;
  const PagedForm f = form_of(p.rows, p.B, p.H, p.G.n, p.table_pages, fp8);
  const int grid = workgroups_of(f, p, cus);
  const bool moved = p.norm_w != nullptr || p.rope_mode != 0;
  switch (f) {
    case kSplit16:
      return launch_form(fp8 ? (moved ? paged_split_kernel<true, 1, true> : paged_split_kernel<true, 1, false>)
                             : (moved ? paged_split_kernel<false, 1, true> : paged_split_kernel<false, 1, false>), 64 * kSplitWaves, paged_merge_kernel<16>, 8, grid, p, st);
    case kSplit32:
      return launch_form(fp8 ? paged_split_kernel<true, 2, false> : paged_split_kernel<false, 2, false>, 64 * kSplitWaves, paged_merge_kernel<32>, 8, grid, p, st);
    default:
      return launch_form(fp8 ? (moved ? paged_tile_kernel<true, true> : paged_tile_kernel<true, false>)
                             : (moved ? paged_tile_kernel<false, true> : paged_tile_kernel<false, false>),
                         64 * kTileWaves, paged_merge_tile_kernel, kTileRows / 8, grid, p, st);
  }
}

}  // namespace pkh3
