// Matrix products on plain row-major matrices that finish their own results (include/pkh3_rows.h): out[m, n] = finish(sum over k of A(m, k) B(n, k)).
//
// Operands.  MFMA 16x16x32: lane (c = l % 16, g = l / 16) supplies elements 8*g .. +7 of row c of an operand, so a block of 16 rows x 32 contraction elements is 16
// bytes a lane ("image"), of A and of B alike.  B goes down the result's registers: a lane then holds four consecutive columns of out for one row.  Chunks of 64 contraction
// elements are copied memory -> LDS as they lie in memory, 128 bytes of a row at a time (what an L2 line holds), without passing through registers, and cut
// into images on the way from LDS:
//   along  (rows of K): 128 bytes a row; the 16-byte piece q of row r lies at place q ^ (r % 8), so that eight lanes that read piece q of eight rows meet no bank twice
//   across (K rows): units of 64 contraction elements x 64 rows, 128 bytes an element; the 32-byte piece b of element k lies at place b ^ (k % 4); a 16-lane
//          transposing read takes four elements of 16 rows and gives each lane those of one row (ds_read_b64_tr_b16), two of them an image
// A copy's LDS target is linear in the lane, so the places are chosen through the lanes' source addresses.
//
// Work split.  Workgroup = 4 waves, one per SIMD = 256 rows of B x 32*TB rows of A; wave (fh, th) = 128 rows of B x 16*TB of A.  Two chunks in LDS: while the products of a
// chunk's second half run, its place is filled with the chunk after the next, and the first half of the next chunk is read into registers.
#include <type_traits>

#include "pkh3_rows.h"

namespace pkh3 {

constexpr int kTileB = 256;       // rows of B of a workgroup
constexpr int kChunk = 64;        // contraction elements of a chunk

// The two halves of a direct-to-LDS copy: wave-uniform target and base address, per-lane byte offset.  `lanes`: all or none.
__device__ __forceinline__ void copy_to(unsigned lds_addr) { asm volatile("s_mov_b32 m0, %0" ::"s"(lds_addr) : "m0"); }
__device__ __forceinline__ void copy_from(const char* g, unsigned lane_off, unsigned long long lanes) {
  asm volatile("s_mov_b64 exec, %2\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1"
               :
               : "v"(lane_off), "s"(g), "s"(lanes)
               : "memory");
}

// c += a b, as an instruction: the compiler, left to place 256 accumulator registers itself, moves them between the halves of the register file inside the loop.
// AGPR: they lie in the accumulator half.
template <bool AGPR>
__device__ __forceinline__ void mfma_acc(f32x4& c, const bf16x8& a, const bf16x8& b) {
  if constexpr (AGPR) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}

typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(8))) short i16x8;
__device__ __forceinline__ bf16x8 read_across(const char* at) {
  using P = __attribute__((address_space(3))) i16x4*;
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at);
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 4 * 128));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// How one operand's tile of ROWS rows comes to LDS (COPIES 1 KiB copies of this wave) and from there to registers.
template <bool ACROSS, int ROWS, bool PAIRS>
struct Operand {
  static constexpr int kCopies = ROWS / 8 / 4;
  const char* next;              // of the chunk to copy next
  const char* next_pair;         // ... of the gates' rows (PAIRS)
  unsigned off[kCopies];
  int64_t advance;               // bytes from chunk to chunk

  // first: the tile's first row (column of out).  rows: of the matrix; pair: rows from values to gates.  left: contraction elements of the chunk.
  __device__ __forceinline__ void init(const char* src, int64_t stride, int first, int rows, int64_t pair, int lane, int wave, int64_t k0) {
    if constexpr (ACROSS) next = src + k0 * stride, advance = kChunk * stride;
    else next = src + first * stride + k0 * 2, next_pair = next + pair * stride, advance = kChunk * 2;
  }
  __device__ __forceinline__ void offsets(int64_t stride, int first, int rows, int lane, int wave, int left) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int piece = wave * kCopies + i;
      if constexpr (ACROSS) {
        const int k = 8 * (piece & 7) + (lane >> 3), place = lane & 7;
        const int col = (piece >> 3) * 64 + (((place >> 1) ^ (k & 3)) * 2 + (place & 1)) * 8;
        off[i] = (unsigned)(min(k, left - 1) * (unsigned)stride) + (unsigned)min(first + col, rows - 8) * 2u;
      } else {
        const int r = 8 * piece + (lane >> 3), q = (lane & 7) ^ (r & 7);
        const int row = PAIRS ? (r >> 5) * 16 + (r & 15) : r;   // (the gates' rows: from their own base)
        off[i] = (unsigned)min(row, rows - 1 - first) * (unsigned)stride + (unsigned)(q * 8 < left ? q * 16 : 0);
      }
    }
  }
  template <int I>
  __device__ __forceinline__ const char* base() const {
    // a wave's copies are 8 rows each, two of values and two of gates in turn
    if constexpr (PAIRS) return I & 2 ? next_pair : next;
    else return next;
  }
  __device__ __forceinline__ void step() {
    next += advance;
    if constexpr (PAIRS) next_pair += advance;
  }
};

// Where this lane finds image (block of 16 rows rb, half ks of a chunk) of a tile in LDS: a base per ... and constant offsets.
template <bool ACROSS>
struct Images {
  const char* at[ACROSS ? 4 : 2];
  __device__ __forceinline__ void init(const char* lds, int lane, int first_block) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (ACROSS) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        at[b] = lds + (8 * g + (c >> 2)) * 128 + (((b + first_block) & 3) ^ (c >> 2)) * 32 + (c & 3) * 8 + (first_block >> 2) * 8192;
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) at[ks] = lds + (first_block * 16 + c) * 128 + (((4 * ks + g) ^ (c & 7)) * 16);
    }
  }
  // RB: block behind the first one (whose number is a multiple of 4, or the blocks do not leave its unit)
  template <int RB>
  __device__ __forceinline__ bf16x8 read(int ks, int slot_bytes) const {
    if constexpr (ACROSS) return read_across(at[RB & 3] + (RB >> 2) * 8192 + ks * 4096 + slot_bytes);
    else return *(const bf16x8*)(at[ks] + RB * 2048 + slot_bytes);
  }
};

template <bool A_ACROSS, bool B_ACROSS, bool PAIRS, int TB>
__device__ __forceinline__ void product_loop(const ProductParams& p, int m0, int n0, int chunk0, int chunks, char* lds_raw, f32x4 (&acc)[TB][8]) {
  constexpr int kTileA = 32 * TB, kBytesB = kTileB * 128, kSlot = kBytesB + kTileA * 128;
  constexpr bool kAgpr = TB > 4;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fh = wave & 1, th = wave >> 1;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds_raw;
  const int64_t k0 = (int64_t)chunk0 * kChunk;
  const int left = (int)(p.K - k0) - (chunks - 1) * kChunk < kChunk ? (int)(p.K - k0) - (chunks - 1) * kChunk : kChunk;   // of the last chunk
  Operand<B_ACROSS, kTileB, PAIRS> ob;
  Operand<A_ACROSS, kTileA, false> oa;
  constexpr int CB = decltype(ob)::kCopies, CA = decltype(oa)::kCopies, PP = CA + CB;
  ob.init(p.b, p.b_stride, n0, p.N, p.N, lane, wave, k0);
  oa.init(p.a, p.a_stride, m0, p.M, 0, lane, wave, k0);
  auto offsets = [&](int k_left) {
    ob.offsets(p.b_stride, n0, p.N, lane, wave, k_left);
    oa.offsets(p.a_stride, m0, p.M, lane, wave, k_left);
  };
  offsets(chunks == 1 ? left : kChunk);
  unsigned long long lanes = ~0ull;                  // all lanes while chunks are left, then none
  int to_copy = chunks;
  auto piece_to = [&](auto ic, int slot) {
    constexpr int i = decltype(ic)::value;
    copy_to(lds0 + slot * kSlot + (i < CB ? (wave * CB + i) * 1024 : kBytesB + (wave * CA + i - CB) * 1024));
  };
  auto piece_from = [&](auto ic) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < CB) copy_from(ob.template base<i>(), ob.off[i], lanes);
    else copy_from(oa.template base<i - CB>(), oa.off[i - CB], lanes);
    if constexpr (i == PP - 1) {
      ob.step();
      oa.step();
      --to_copy;
      asm volatile("s_cmp_gt_i32 %1, 0\n\ts_cselect_b64 %0, -1, 0" : "=s"(lanes) : "s"(to_copy) : "scc");
      if (to_copy == 1 && left < kChunk) offsets(left);
    }
  };
  auto copy_chunk = [&](int slot) {
    static_for<PP>([&](auto ic) {
      piece_to(ic, slot);
      asm volatile("s_nop 0");
      piece_from(ic);
    });
  };
  Images<B_ACROSS> ib;
  Images<A_ACROSS> ia;
  ib.init(lds_raw, lane, fh * 8);
  ia.init(lds_raw + kBytesB, lane, th * TB);
  constexpr int kReads = 8 + TB;
  auto read_image = [&](auto ic, int ks, int slot_bytes, bf16x8 (&w)[8], bf16x8 (&x)[TB]) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < TB) x[i] = ia.template read<i>(ks, slot_bytes);
    else w[i - TB] = ib.template read<i - TB>(ks, slot_bytes);
  };
  // what lies behind the contraction's end is taken for zeros (both operands: it may be anything)
  auto clear_rest = [&](int from, bf16x8 (&w)[8], bf16x8 (&x)[TB]) {
    i32x4 keep;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int k = from + 8 * (lane >> 4) + 2 * d;
      keep[d] = (k < left ? 0xffff : 0) | (k + 1 < left ? (int)0xffff0000 : 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(i32x4, w[i]) & keep);
#pragma unroll
    for (int i = 0; i < TB; ++i) x[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(i32x4, x[i]) & keep);
    asm volatile("s_nop 1" ::: "memory");            // (an MFMA may not take a register right behind the instruction that wrote it)
  };

  static_for<TB>([&](auto tc) {
    static_for<8>([&](auto fc) { acc[decltype(tc)::value][decltype(fc)::value] = f32x4{0.f, 0.f, 0.f, 0.f}; });
  });
  bf16x8 wa[8], wb[8], xa[TB], xb[TB];               // images of a chunk's first and second half
  copy_chunk(0);
  copy_chunk(1);
  __builtin_amdgcn_s_waitcnt((PP & 15) | ((PP >> 4) << 14) | (7 << 4) | (15 << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  static_for<kReads>([&](auto ic) { read_image(ic, 0, 0, wa, xa); });
#pragma unroll 1
  for (int kc = 0; kc < chunks; ++kc) {
    const int slot = kc & 1, here = slot * kSlot, there = kSlot - here;
    const bool rest = kc == chunks - 1 && left < kChunk;
    if (rest) clear_rest(0, wa, xa);
    // first half; the second half's images meanwhile.  (Blocks of A back and forth: from one MFMA to the next only one operand changes.)
    static_for<8 * TB>([&](auto kk) {
      constexpr int k = decltype(kk)::value, fb = k / TB, t = fb & 1 ? TB - 1 - k % TB : k % TB;
      mfma_acc<kAgpr>(acc[t][fb], wa[fb], xa[t]);
      if constexpr (k % 2 == 0 && k / 2 < kReads) read_image(std::integral_constant<int, k / 2>{}, 1, here, wb, xb);
      if constexpr (TB == 2 && k % 2 == 1 && k / 2 + 8 < kReads) read_image(std::integral_constant<int, k / 2 + 8>{}, 1, here, wb, xb);
    });
    if (rest) clear_rest(32, wb, xb);
    // every wave holds the chunk in registers, and the next one is in LDS
    __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (0 << 8));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_for<8 * TB>([&](auto kk) {
      constexpr int k = decltype(kk)::value, fb = k / TB, t = fb & 1 ? TB - 1 - k % TB : k % TB;
      mfma_acc<kAgpr>(acc[t][fb], wb[fb], xb[t]);
      constexpr int kEvery = 8 * TB / PP;
      if constexpr (TB > 2) {
        if constexpr (k % 2 == 0 && k / 2 < kReads) read_image(std::integral_constant<int, k / 2>{}, 0, there, wa, xa);
        if constexpr (kEvery >= 4) {
          if constexpr (k % 4 == 1 && k / 4 < PP) piece_to(std::integral_constant<int, k / 4>{}, slot);
          if constexpr (k % 4 == 3 && k / 4 < PP) piece_from(std::integral_constant<int, k / 4>{});
        } else {
          if constexpr (k % 2 == 1 && k / 2 < PP) {
            piece_to(std::integral_constant<int, k / 2>{}, slot);
            asm volatile("s_nop 0");
            piece_from(std::integral_constant<int, k / 2>{});
          }
        }
      } else {
        if constexpr (k < kReads) read_image(std::integral_constant<int, k>{}, 0, there, wa, xa);
        if constexpr (k < PP) {
          piece_to(std::integral_constant<int, k>{}, slot);
          asm volatile("s_nop 0");
          piece_from(std::integral_constant<int, k>{});
        }
      }
    });
  }
  // the compiler does not know the instructions above for MFMAs: let the last one retire before anything reads the accumulators
  static_for<TB>([&](auto tc) {
    f32x4(&a)[8] = acc[decltype(tc)::value];
    if constexpr (kAgpr)
      asm volatile("s_nop 15\n\ts_nop 15" : "+a"(a[0]), "+a"(a[1]), "+a"(a[2]), "+a"(a[3]), "+a"(a[4]), "+a"(a[5]), "+a"(a[6]), "+a"(a[7])::"memory");
    else
      asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7])::"memory");
  });
}

constexpr int kStagePitch = 128 + 4;                 // floats between rows of staged results
constexpr int kStageBytes = 16 * kStagePitch * 4;    // of a wave

// A wave's results: 16 rows at a time through LDS (its own part), so that a row's columns leave in 16-byte pieces beside each other, 256 bytes a row.
// What else the results need is asked for a block of rows ahead.  CUT: the sums of a part of the contraction, as they are.
template <int MODE, bool CUT, int TB>
__device__ __forceinline__ void product_epilogue(const ProductParams& p, int cut, int m0, int n0, int sum_row, float* lds, const f32x4 (&acc)[TB][8]) {
  constexpr bool kPairs = MODE == kGated;
  constexpr int kPieces = kPairs ? 8 : 16;            // pieces of a row of the wave
  constexpr int kRows = 64 / kPieces, kPasses = 16 / kRows;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int piece = lane % kPieces, n = n0 + piece * 8, n_at = min(n, p.N - 8);
  const bool live = n < p.N;
  const float* from = lds + (lane / kPieces) * kStagePitch + (kPairs ? (piece >> 1) * 32 + (piece & 1) * 8 : piece * 8);
  Bias bias{};
  Extra<MODE> next[kPasses];
  auto ask = [&](int t) {
    if constexpr (!CUT) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) fetch<MODE>(p, min(m0 + 16 * t + i * kRows + lane / kPieces, p.M - 1), n_at, next[i]);
    }
  };
  if constexpr (!CUT) bias = load_bias<MODE>(p, n_at);
  ask(0);
  Piece sum_a{}, sum_b{};
#pragma unroll 1
  for (int t = 0; t < TB; ++t) {
    if (m0 + 16 * t >= p.M) break;
    __builtin_amdgcn_wave_barrier();
    static_for<TB>([&](auto tc) {
      if (t == decltype(tc)::value) {
#pragma unroll
        for (int f = 0; f < 8; ++f) *(f32x4*)(lds + c * kStagePitch + 16 * f + 4 * g) = acc[decltype(tc)::value][f];
      }
    });
    __builtin_amdgcn_wave_barrier();
    Extra<MODE> now[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) now[i] = next[i];
    if (t + 1 < TB) ask(t + 1);
    auto each = [&](auto&& use) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int m = m0 + 16 * t + i * kRows + lane / kPieces;
        Piece a = load_piece_f32((const char*)(from + i * kRows * kStagePitch)), b{};
        if constexpr (kPairs) b = load_piece_f32((const char*)(from + i * kRows * kStagePitch + 16));
        if (live && m < p.M) use(m, a, b, now[i]);
      }
    };
    if constexpr (CUT) {
      const int columns = kPairs ? 2 * p.N : p.N;
      each([&](int m, Piece& a, Piece& b, const Extra<MODE>&) {
        float* to = p.part + ((int64_t)cut * p.M + m) * columns + n;
        store_piece_f32((char*)to, a);
        if constexpr (kPairs) store_piece_f32((char*)(to + p.N), b);
      });
    } else {
      with_activation(p.act, [&](auto act) {
        each([&](int m, Piece& a, Piece& b, const Extra<MODE>& extra) {
          finish<MODE, decltype(act)::value>(p, m, n, a, b, bias, extra);
          if constexpr (MODE >= kGrad) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              sum_a.v[j] += a.v[j];
              if constexpr (MODE == kGatedGrad) sum_b.v[j] += b.v[j];
            }
          }
        });
      });
    }
  }
  if constexpr (MODE >= kGrad && !CUT) {
    if (p.sums) {
      const int columns = MODE == kGatedGrad ? 2 * p.N : p.N;
      float* at = p.sums + (int64_t)sum_row * columns + n;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int over = kPieces; over < 64; over *= 2) {
          sum_a.v[j] += __shfl_xor(sum_a.v[j], over, 64);
          if constexpr (MODE == kGatedGrad) sum_b.v[j] += __shfl_xor(sum_b.v[j], over, 64);
        }
      }
      if (live && lane < kPieces) {
        store_piece_f32((char*)at, sum_a);
        if constexpr (MODE == kGatedGrad) store_piece_f32((char*)(at + p.N), sum_b);
      }
    }
  }
}

template <bool A_ACROSS, bool B_ACROSS, int MODE, int TB>
__global__ __launch_bounds__(256, TB > 2 ? 1 : 2) void product_kernel(ProductParams p, int m_tiles, int n_tiles) {
  constexpr bool kPairs = MODE == kGated;
  constexpr int kSlot = (kTileB + 32 * TB) * 128;
  static_assert(2 * kSlot >= 4 * kStageBytes, "the results go through the chunks' places");
  __shared__ __attribute__((aligned(1024))) char lds_raw[2 * kSlot];
  // Workgroups go to the 8 XCDs round-robin; each takes one contiguous run of the tile order, in which blocks of 8 tiles of B walk down the tiles of A: the
  // workgroups that run behind one L2 at a time share 8 tiles of B and 4 of A.
  constexpr int kBlockN = 8;
  const int tiles = m_tiles * n_tiles, total = tiles * p.cuts, per_xcd = (total + 7) / 8;
  int lin = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || lin >= total) return;
  const int cut = lin / tiles;
  lin -= cut * tiles;
  const int full = n_tiles / kBlockN * kBlockN;
  int m_tile, n_tile;
  if (lin < full * m_tiles) {
    const int nb = lin / (kBlockN * m_tiles), rem = lin % (kBlockN * m_tiles);
    m_tile = rem / kBlockN;
    n_tile = nb * kBlockN + rem % kBlockN;
  } else {
    const int rest = lin - full * m_tiles, width = n_tiles - full;
    m_tile = rest / width;
    n_tile = full + rest % width;
  }
  const int chunks = (p.K + kChunk - 1) / kChunk;
  const int first = (int)((int64_t)chunks * cut / p.cuts), end = (int)((int64_t)chunks * (cut + 1) / p.cuts);
  const int m0 = m_tile * 32 * TB, n0 = n_tile * (kPairs ? kTileB / 2 : kTileB);
  f32x4 acc[TB][8];
  // (only the last part holds the contraction's end: the others end with whole chunks)
  product_loop<A_ACROSS, B_ACROSS, kPairs, TB>(p, m0, n0, first, end - first, lds_raw, acc);
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = m0 + (wave >> 1) * 16 * TB, wn = n0 + (wave & 1) * (kPairs ? 64 : 128);
  float* staged = (float*)(lds_raw + wave * kStageBytes);
  if (p.part) product_epilogue<MODE, true, TB>(p, cut, wm, wn, 0, staged, acc);
  else product_epilogue<MODE, false, TB>(p, 0, wm, wn, m_tile * 2 + (wave >> 1), staged, acc);
}

// The parts of a contraction that was cut, added up in their order, and finished: a workgroup is 8 rows x 32 pieces of 8 columns.
constexpr int kJoinRows = 8;

template <int MODE>
__global__ __launch_bounds__(256) void product_join_kernel(ProductParams p) {
  __shared__ Piece staged[MODE >= kGrad ? 2 * 256 : 1];
  const int n = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8, m = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
  const bool live = n < p.N && m < p.M;
  const int columns = MODE == kGated ? 2 * p.N : p.N;
  Piece a{}, b{};
  if (live) {
    Extra<MODE> extra;
    fetch<MODE>(p, m, n, extra);
    const char* from = (const char*)(p.part + (int64_t)m * columns + n);
    const int64_t next = (int64_t)p.M * columns * 4;
    for (int i = 0; i < p.cuts; ++i, from += next) {
      const Piece va = load_piece_f32(from);
#pragma unroll
      for (int j = 0; j < 8; ++j) a.v[j] += va.v[j];
      if constexpr (MODE == kGated) {
        const Piece vb = load_piece_f32(from + (int64_t)p.N * 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) b.v[j] += vb.v[j];
      }
    }
    const Bias bias = load_bias<MODE>(p, n);
    with_activation(p.act, [&](auto act) { finish<MODE, decltype(act)::value>(p, m, n, a, b, bias, extra); });
  }
  if constexpr (MODE >= kGrad) {
    if (!p.sums) return;
    staged[threadIdx.x] = a;
    staged[256 + threadIdx.x] = b;
    __syncthreads();
    if (threadIdx.x < 64) {
      const Piece* at = staged + (threadIdx.x >> 5) * 256 + (threadIdx.x & 31);
      Piece sum = at[0];
      for (int r = 1; r < kJoinRows; ++r) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum.v[j] += at[r * 32].v[j];
      }
      const bool second = threadIdx.x >= 32;
      if (n < p.N && (MODE == kGatedGrad || !second))
        store_piece_f32((char*)(p.sums + (int64_t)blockIdx.y * (MODE == kGatedGrad ? 2 * p.N : p.N) + (second ? p.N : 0) + n), sum);
    }
  }
}

// out[c] = sum over the rows of part[row][c], 32 columns a workgroup of 256: 8 lanes of 4 columns, 32 rows at a time
__global__ __launch_bounds__(256) void column_sums_kernel(const float* part, int rows, int columns, __bf16* out) {
  __shared__ f32x4 staged[256];
  const int col = blockIdx.x * 32 + (threadIdx.x & 7) * 4;
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  if (col < columns)
    for (int r = threadIdx.x >> 3; r < rows; r += 32) sum += *(const f32x4*)(part + (int64_t)r * columns + col);
  staged[threadIdx.x] = sum;
  for (int over = 128; over >= 8; over /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < over) staged[threadIdx.x] += staged[threadIdx.x + over];
  }
  if (threadIdx.x < 8 && col < columns) {
    const f32x4 v = staged[threadIdx.x];
    bf16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (__bf16)v[j];
    *(bf16x4*)(out + col) = o;
  }
}

static size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

bool product_offered(bool a_across, bool b_across, int mode) {
  if (a_across) return b_across && mode == kPlain;
  return b_across ? mode != kGated : mode <= kGated;
}

ProductPlan plan_product(int M, int N, int K, int mode, bool sums) {
  ProductPlan plan{};
  plan.tb = 8;
  plan.cuts = 1;
  const int tiles = (M + 32 * plan.tb - 1) / (32 * plan.tb);
  plan.sum_rows = !sums ? 0 : plan.cuts > 1 ? (M + kJoinRows - 1) / kJoinRows : tiles * 2;
  plan.part_off = 0;
  plan.sums_off = plan.cuts > 1 ? round_up((size_t)plan.cuts * M * (mode == kGated ? 2 : 1) * N * sizeof(float)) : 0;
  plan.total = plan.sums_off + round_up((size_t)plan.sum_rows * (mode == kGatedGrad ? 2 : 1) * N * sizeof(float));
  return plan;
}

template <bool A_ACROSS, bool B_ACROSS, int MODE>
static hipError_t launch_tiles(const ProductParams& p, const ProductPlan& plan, hipStream_t s) {
  const int columns = MODE == kGated ? kTileB / 2 : kTileB;
  const int m_tiles = (p.M + 32 * plan.tb - 1) / (32 * plan.tb), n_tiles = (p.N + columns - 1) / columns;
  const int total = m_tiles * n_tiles * plan.cuts;
  const dim3 grid((total + 7) / 8 * 8);
  product_kernel<A_ACROSS, B_ACROSS, MODE, 8><<<grid, 256, 0, s>>>(p, m_tiles, n_tiles);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.cuts == 1) return e;
  product_join_kernel<MODE><<<dim3((p.N + 255) / 256, (p.M + kJoinRows - 1) / kJoinRows), 256, 0, s>>>(p);
  return hipGetLastError();
}

static hipError_t launch_column_sums(const float* part, int rows, int columns, void* out, hipStream_t s) {
  column_sums_kernel<<<(columns + 31) / 32, 256, 0, s>>>(part, rows, columns, (__bf16*)out);
  return hipGetLastError();
}

hipError_t launch_product(ProductParams p, const ProductPlan& plan, bool a_across, bool b_across, int mode, void* sums, char* workspace, hipStream_t s) {
  p.sums = sums ? (float*)(workspace + plan.sums_off) : nullptr;
  p.part = plan.cuts > 1 ? (float*)(workspace + plan.part_off) : nullptr;
  p.cuts = plan.cuts;
  hipError_t e;
  if (a_across) e = launch_tiles<true, true, kPlain>(p, plan, s);
  else if (!b_across) e = mode == kGated ? launch_tiles<false, false, kGated>(p, plan, s) : launch_tiles<false, false, kPlain>(p, plan, s);
  else if (mode == kPlain) e = launch_tiles<false, true, kPlain>(p, plan, s);
  else if (mode == kGrad) e = launch_tiles<false, true, kGrad>(p, plan, s);
  else e = launch_tiles<false, true, kGatedGrad>(p, plan, s);
  if (e != hipSuccess || !sums) return e;
  return launch_column_sums(p.sums, plan.sum_rows, mode == kGatedGrad ? 2 * p.N : p.N, sums, s);
}

// ---- the gradient of an activation, and the sums of its columns ----

constexpr int kGradRows = 64;     // rows of a workgroup: 8 at a time, 32 pieces of 8 columns

template <int ACT>
__global__ __launch_bounds__(256) void activation_grad_kernel(ProductParams p) {
  __shared__ Piece staged[256];
  const int n = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8;
  Piece sum{};
  if (n < p.N)
    for (int i = threadIdx.x >> 5; i < kGradRows; i += 8) {
      const int m = blockIdx.y * kGradRows + i;
      if (m >= p.M) break;
      Piece a = load_piece(p.a + m * p.a_stride + (int64_t)n * 2), b{};
      if (p.out) {
        Extra<kGrad> extra;
        fetch(p, m, n, extra);
        finish<kGrad, ACT>(p, m, n, a, b, Bias{}, extra);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum.v[j] += a.v[j];
    }
  if (!p.sums) return;
  staged[threadIdx.x] = sum;
  for (int over = 128; over >= 32; over /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < over) {
#pragma unroll
      for (int j = 0; j < 8; ++j) staged[threadIdx.x].v[j] += staged[threadIdx.x + over].v[j];
    }
  }
  if (threadIdx.x < 32 && n < p.N) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p.sums[(int64_t)blockIdx.y * p.N + n + j] = staged[threadIdx.x].v[j];
  }
}

int activation_grad_rows(int M) { return (M + kGradRows - 1) / kGradRows; }

hipError_t launch_activation_grad(ProductParams p, void* sums, char* workspace, hipStream_t s) {
  p.sums = sums ? (float*)workspace : nullptr;
  const dim3 grid((p.N + 255) / 256, activation_grad_rows(p.M));
  if (p.act == 1) activation_grad_kernel<1><<<grid, 256, 0, s>>>(p);
  else if (p.act == 2) activation_grad_kernel<2><<<grid, 256, 0, s>>>(p);
  else if (p.act == 3) activation_grad_kernel<3><<<grid, 256, 0, s>>>(p);
  else activation_grad_kernel<0><<<grid, 256, 0, s>>>(p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !sums) return e;
  return launch_column_sums(p.sums, activation_grad_rows(p.M), p.N, sums, s);
}

}  // namespace pkh3
