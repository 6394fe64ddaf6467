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
// from one to the other in its lane, running maximum raised when exceeded by 2^8.  Q' is rounded to bf16 after norm and rotation and not
// before: the softmax scale multiplies S^T (in fp32, in the subtraction of the maximum), so that queries without norm and rotation are exact.
// e4m3 keys times their power of two are exact in bf16; the scale of a value's key goes to P instead, exact there as well.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "pkh3_paged.h"
#include "pkh3_internal.h"

namespace pkh3 {

constexpr float kNoMax = -FLT_MAX;       // the running max before the first key: finite, so that rows without a key add up to nothing
constexpr float kRescaleSlack = 8.0f;    // the running max is raised only when exceeded by 2^8
constexpr int kSplitWaves = 4;

// ---- the tile space ----

__device__ __forceinline__ int blocks_of(const PagedParams& p, const Sequence& s, int rb) { return blocks_of(s, p.G, rb); }
__device__ __forceinline__ int block_tiles(const PagedParams& p, const Sequence& s, int rb, int j) { return block_tiles(s, p.G, p.causal, rb, j); }
__device__ __forceinline__ int row_keys(const PagedParams& p, const Sequence& s, int r) { return row_keys(s, p.G, p.causal, r); }

// Where a run begins: sequence, head, block and tile.
struct Place {
  int b, h, j, t;
};

// The sums of the tiles of all sequences in `cum`, by the whole workgroup.  Blocks of a causal sequence differ in length: where
// there are more than a few, a wave adds them up together.
__device__ __forceinline__ void sum_tiles(const PagedParams& p, int64_t* cum, int rb) {
  constexpr int kAlone = 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  for (int at = 64 * wave; at < p.B; at += 64 * waves) {
    const int b = at + lane;
    int64_t mine = 0;
    bool many = false;
    if (b < p.B) {
      const Sequence s = sequence(p, b);
      const int blocks = blocks_of(p, s, rb);
      many = p.causal && blocks > kAlone;
      if (!p.causal) mine = blocks ? (int64_t)blocks * block_tiles(p, s, rb, 0) : 0;
      else if (!many)
        for (int j = 0; j < blocks; ++j) mine += block_tiles(p, s, rb, j);
    }
    for (unsigned long long left = __ballot(many); left; left &= left - 1) {
      const int l = __ffsll((unsigned long long)left) - 1;
      const Sequence s = uniform_sequence(p, __builtin_amdgcn_readfirstlane(at + l));
      const int blocks = blocks_of(p, s, rb);
      int64_t sum = 0;
      for (int j = lane; j < blocks; j += 64) sum += block_tiles(p, s, rb, j);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      if (lane == l) mine = sum;
    }
    if (b < p.B) cum[b + 1] = mine * p.H;
  }
  prefix_sums(cum, p.B);
}

__device__ __forceinline__ Place find_place(const PagedParams& p, const int64_t* cum, int rb, int64_t pos) {
  Place at;
  at.b = find_sequence(cum, p.B, pos);
  const Sequence s = uniform_sequence(p, at.b);
  const int64_t per_head = (cum[at.b + 1] - cum[at.b]) / p.H;
  const int64_t in = pos - cum[at.b];
  at.h = __builtin_amdgcn_readfirstlane((int)(in / per_head));
  int64_t rest = in - at.h * per_head;
  if (!p.causal) {
    const int nt = block_tiles(p, s, rb, 0);
    at.j = __builtin_amdgcn_readfirstlane((int)(rest / nt));
    at.t = __builtin_amdgcn_readfirstlane((int)(rest - (int64_t)at.j * nt));
    return at;
  }
  const int lane = threadIdx.x & 63, blocks = blocks_of(p, s, rb);
  for (int first = 0;; first += 64) {
    int64_t x = first + lane < blocks ? block_tiles(p, s, rb, first + lane) : 0;
    const int64_t own = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    const unsigned long long past = __ballot(x > rest);
    if (past || first + 64 >= blocks) {
      const int l = past ? __ffsll((unsigned long long)past) - 1 : 63;
      at.j = __builtin_amdgcn_readfirstlane(first + l);
      at.t = __builtin_amdgcn_readfirstlane((int)(rest - __shfl(x - own, l)));
      return at;
    }
    rest -= __shfl(x, 63);
  }
}

// A part of a unit in the scratch: RB rows of 128, then their maxima, then their sums
__host__ __device__ constexpr int part_floats(int rb) { return rb * (kD + 2); }

// ---- the split form: few query rows, the waves of a workgroup share the keys out ----
//
// A unit is one or two blocks of 16 query rows, and each of the four waves walks a quarter of the run's part of it in 32-key halves.  No two
// waves read the same images, so these go straight from memory into the registers of the MFMAs: no LDS and no barrier in the loop, the
// next keys asked for under the softmax, the values under S^T.  The waves' results meet in LDS.  Bound by the bytes of K and V.

template <bool FP8, int QB>
struct SplitState {
  bf16x8 qf[QB][4];
  f32x4 o[8][QB];
  float m[QB], l[QB];
};

// The weights of one half tile, the running maximum and the row sums.  ve: exponents of the values' scales.
template <bool FP8, int QB>
__device__ __forceinline__ void split_softmax(SplitState<FP8, QB>& w, const f32x4 (&s)[2][QB], bf16x8 (&pf)[QB], const unsigned (&ve)[2], float c) {
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
  token = (int)((unsigned)r / (unsigned)p.G);
  return (int64_t)(s.first + token) * ss + (int64_t)(h * p.G + r - token * p.G) * sh;
}

// Sixteen query rows from r on (those past the last are the last one again) through norm and rotation, in the lane order of the B images.
__device__ __forceinline__ void query_rows(const PagedParams& p, const Sequence& s, int h, int r0, char* turn, int lane, bf16x8 (&out)[4]) {
  const int last = s.n * p.G - 1;
  Rows16 q, cos, sin;
  int token[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = row_offset(p, s, h, min(r0 + 4 * i + (lane >> 4), last), p.q_ss, p.q_sh, token[i]);
    q.v[i] = *(const i32x4*)(p.q + at + (lane & 15) * 16);
  }
  NormLanes norm;
  load_norm_lanes(norm, p.norm_w, lane);
  RopeQuarter rope;
  if (p.rope_mode != 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = (int64_t)(s.first + token[i]) * (kD / 2 * (int)sizeof(float)) + (lane & 15) * 16;
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
  float x[32];
  norm_row(x, raw, p.norm_w != nullptr, p.eps, norm, 1.0f);
  rope_row(x, p.rope_mode, rope);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks)
#pragma unroll
    for (int j = 0; j < 8; ++j) out[ks][j] = (__bf16)x[8 * ks + j];
}

template <bool FP8, int QB>
__global__ __launch_bounds__(64 * kSplitWaves, 2) void paged_split_kernel(PagedParams p) {
  constexpr int RB = 16 * QB, NW = kSplitWaves;
  constexpr int kSlot = QB * 8 * 64 * 16;                      // one wave's O^T in fp32
  constexpr int kRecord = FP8 ? kPageRecord8 : kPageRecord16;
  constexpr int kN = FP8 ? 4 : 8;                              // 16-byte pieces of a lane of a half tile's K, and of its V
  constexpr int kVOff = FP8 ? kK8TileBytes : kKTileBytes;
  constexpr int kScaleOff = kK8TileBytes + kVTileBytes / 2;
  __shared__ __attribute__((aligned(1024))) char part[NW * kSlot];
  __shared__ __attribute__((aligned(1024))) char rows[QB * 4096];
  __shared__ float part_m[NW][QB][16], part_l[NW][QB][16];
  static_assert((kMaxSequences + 1) * sizeof(int64_t) <= sizeof(part), "the sums lie where the waves' results meet afterwards");
  const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  int64_t* cum = (int64_t*)part;
  sum_tiles(p, cum, RB);
  const Shares sh = shares_of(cum[p.B], gridDim.x);
  const int rank = rank_of(blockIdx.x, sh);
  if (rank < 0 || sh.total == 0) return;
  const int64_t begin = sh.begin(rank);
  int64_t left = sh.begin(rank + 1) - begin;
  Place at = find_place(p, cum, RB, begin);
  Sequence s = uniform_sequence(p, at.b);
  int blocks = blocks_of(p, s, RB);

#pragma unroll 1
  while (left > 0) {
    const int nt = block_tiles(p, s, RB, at.j), take = (int)min((int64_t)(nt - at.t), left);
    __syncthreads();                                           // the sums, or the results of the unit before, are read
    SplitState<FP8, QB> w;
    if (wave < QB) {
      bf16x8 img[4];
      query_rows(p, s, at.h, at.j * RB + 16 * wave, part + wave * 4096, lane, img);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) *(bf16x8*)(rows + ((wave * 4 + ks) * 64 + lane) * 16) = img[ks];
    }
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
    if (first < end) {
      id = uniform_page(p, at.b, first >> 1);
      ask_k(id, first & 1);
    }
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) w.qf[qb][ks] = *(const bf16x8*)(rows + ((qb * 4 + ks) * 64 + lane) * 16);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
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
        for (int j = 0; j < 8; ++j)                            // image (ks, kb) = (j / 2, j % 2)
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
            sT[j & 1][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[j]), w.qf[qb][j >> 1], j < 2 ? zero : sT[j & 1][qb], 0, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {                          // chunk (kb, c2) = (j / 2, j % 2): images ks = 2*c2, 2*c2 + 1
          const float scale = exponent_scale(ke[j >> 1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bf16x8 a = expand_fp8(kf[j][2 * e], kf[j][2 * e + 1], scale);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
              sT[j >> 1][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, w.qf[qb][2 * (j & 1) + e], (j & 1) + e == 0 ? zero : sT[j >> 1][qb], 0, 0, 0);
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
    float* slot = p.partials + part_slot(rank, at.t == 0) * part_floats(RB);
    const int row = threadIdx.x >> 4, chunk = threadIdx.x & 15;   // 8 columns of one of 16 rows
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = at.j * RB + 16 * qb + row;
      if (r >= s.n * p.G) continue;
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
        const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;     // (a sum that is not a number stays one)
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
    left -= take;
    at.t = 0;
    if (++at.j == blocks) {
      at.j = 0;
      if (++at.h == p.H) {
        at.h = 0;
        do {                                                   // (a run that goes on does so in a sequence with rows)
          if (++at.b >= p.B) return;
          s = uniform_sequence(p, at.b);
        } while (s.n == 0);
        blocks = blocks_of(p, s, RB);
      }
    }
  }
}

// ---- the parts of units that more than one workgroup worked on ----
//
// Boundary i between the runs of workgroups i - 1 and i, where it is the first inside its unit, does the unit: its parts are slot 1 of
// workgroup i - 1 and slot 0 of i, i + 1, .., in that order.  blockIdx.y: 8 of its rows.
template <int RB>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p, int grid) {
  __shared__ int64_t cum[kMaxSequences + 1];
  sum_tiles(p, cum, RB);
  const Shares sh = shares_of(cum[p.B], grid);
  const int first = (int)blockIdx.x;                             // the workgroup in front of the boundary
  if (first + 1 >= sh.n) return;
  const int64_t pos = sh.begin(first + 1);
  const Place at = find_place(p, cum, RB, pos);
  const Sequence s = uniform_sequence(p, at.b);
  const int parts = parts_behind(sh, first, pos - at.t, pos - at.t + block_tiles(p, s, RB, at.j));
  if (parts == 0) return;
  const int row = (int)blockIdx.y * 8 + (threadIdx.x >> 5), col = (threadIdx.x & 31) * 4;
  const int r = at.j * RB + row;
  if (r >= s.n * p.G) return;
  auto slot = [&](int i) { return p.partials + part_slot(first + i, i == 0) * part_floats(RB); };
  float top = kNoMax;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, slot(i)[RB * kD + row]);
  float l = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* t = slot(i);
    const float a = __builtin_amdgcn_exp2f(t[RB * kD + row] - top);
    l += a * t[RB * (kD + 1) + row];
    const f32x4 o = *(const f32x4*)(t + row * kD + col);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += a * o[e];
  }
  const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
  bf16x4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (__bf16)(sum[e] * inv);
  int token;
  *(bf16x4*)(p.o + row_offset(p, s, at.h, r, p.o_ss, p.o_sh, token) + col * 2) = out;
}

// ---- host ----

static int split_blocks(int rows, int B, int G) {   // 16-row blocks of a unit
  return (int64_t)rows * G > 16 * (int64_t)std::min(rows, B) ? 2 : 1;
}

size_t paged_attn_scratch(int rows, int B, int H, int G, int table_pages) {
  return (size_t)2 * kMaxShares * part_floats(16 * split_blocks(rows, B, G));
}

template <bool FP8, int QB>
static hipError_t launch_split(const PagedParams& p, int grid, hipStream_t st) {
  hipLaunchKernelGGL((paged_split_kernel<FP8, QB>), dim3(grid), dim3(64 * kSplitWaves), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_merge_kernel<16 * QB>), dim3(grid, 2 * QB), dim3(256), 0, st, p, grid);
  return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedParams& p, bool fp8, hipStream_t st) {
  int cus = 0;
  const hipError_t e = device_cu_count(&cus);
  if (e != hipSuccess) return e;
  const int grid = std::min(kMaxShares, std::max(8, 2 * cus / 8 * 8));
  if (split_blocks(p.rows, p.B, p.G) == 1) return fp8 ? launch_split<true, 1>(p, grid, st) : launch_split<false, 1>(p, grid, st);
  return fp8 ? launch_split<true, 2>(p, grid, st) : launch_split<false, 2>(p, grid, st);
}

}  // namespace pkh3
