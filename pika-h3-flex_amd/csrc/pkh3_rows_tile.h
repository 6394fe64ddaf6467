// Matrix products on plain row-major matrices that finish their own results (include/pkh3_rows.h): out[m, n] = finish(sum over k of A(m, k) B(n, k)).
//
// Operands.  MFMA 16x16x32: lane (c = l % 16, g = l / 16) supplies elements 8*g .. +7 of row c of an operand, so a block of 16 rows x 32 contraction elements is 16
// bytes a lane ("image"), of A and of B alike.  B goes down the result's registers: a lane then holds four consecutive columns of out for one row.  Chunks of 64 contraction
// elements are copied memory -> LDS as they lie in memory, 128 bytes of a row at a time (what an L2 line holds), without passing through registers, and cut
// into images on the way from LDS:
//   along  (rows of K): 128 bytes a row; the 16-byte piece q of row r lies at place q ^ (r % 8), so that eight lanes that read piece q of eight rows meet no bank twice
//   across (K rows): units of 64 contraction elements x 64 rows, 128 bytes an element; the 32-byte piece b of element k lies at place b ^ s(k), s of the bits 1 and 3 of k,
//          so that the eight elements that half a wave reads meet no bank twice; a 16-lane transposing read takes four elements of 16 rows and gives each lane those of one row (ds_read_b64_tr_b16), two of them an image
// A copy's LDS target is linear in the lane, so the places are chosen through the lanes' source addresses.
//
// Work split.  Workgroup = 4 waves, one per SIMD = 32*TB rows of A x 32*FB rows of B; wave (fh, th) = 16*TB x 16*FB of them.  256 workgroups, one a CU, take the tiles
// in turn (pkh3_rows_index.h), and the next tile's first chunks come while one's results leave.  Both operands have rings of two to four chunks in LDS.
//
// What bounds it.  256 x 256: the matrix units (2,048 of a chunk's 2,300 cycles), whose clock the board's power holds at 1.7 GHz: 15,342 x 2,048 with a contraction of 5,504
// takes 242 us, 1.43 PFLOP/s.  Smaller tiles: what a CU takes in of lines that its L2 does not have, about 40 GB/s, and waits that a single wave a SIMD leaves uncovered.  No unit is busy: of
// 1,085 x 2,048 x 2,048 in tiles of 96 x 128 (23 us) the matrix units work 27 % of the time, LDS delivers images 16 % of it, without a conflict, and the waves
// wait for 45 %; of 4,000 x 2,048 x 2,048 in 128 x 256 (37 us) 48, 18 and 31 %; of 2,003 x 5,160 x 1,400 in 256 x 256 (47 us) 51, 13 and 26 %.  The results of a tile
// are not covered by the next one's products: 15,342 x 5,504 gradients of gated halves, which read 675 MB and write 338, take 448 us where the product alone takes 240.
#pragma once
#include <type_traits>

#include "pkh3_rows.h"

namespace pkh3 {

// The second half of a copy by all lanes or none: it counts in the waits either way.  (Longer to issue: where it may not be due.)
__device__ __forceinline__ void copy_from_if(const char* g, unsigned lane_off, unsigned long long lanes) {
  asm volatile("s_mov_b64 exec, %2\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1" : : "v"(lane_off), "s"(g), "s"(lanes) : "memory");
}
enum Copying { kNoCopies, kCopies, kCopiesIf };
// c += a b, as an instruction: the compiler, left to place 256 accumulator registers itself, moves them between the halves of the register file inside the loop.
// AGPR: they lie in the accumulator half.
// FIRST: onto zeros.
template <bool AGPR>
__device__ __forceinline__ void mfma_first(f32x4& c, const bf16x8& a, const bf16x8& b) {
  if constexpr (AGPR) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
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

__device__ __forceinline__ int across_swizzle(int k) { return ((k >> 1) & 1) | ((k >> 2) & 2); }

// The lane, in a way that keeps what is worked out from it where it is used: along the tiles' loop there are no registers for it.
__device__ __forceinline__ int lane_here() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// How one operand's tile of ROWS rows comes to LDS, chunk after chunk into SLOTS places: kPieces copies of 1 KiB a chunk and wave.
template <bool ACROSS, int ROWS, bool PAIRS, int SLOTS>
struct Operand {
  static constexpr int kPieces = ROWS / 8 / 4, kSlot = ROWS * 128;
  const char* next;              // of the chunk to copy next
  const char* next_pair;         // ... of the gates' rows (PAIRS)
  unsigned off[kPieces];
  int64_t advance;               // bytes from chunk to chunk
  unsigned fill, ring;           // where this wave's part of that chunk goes, and where it goes in the first place
  int to_copy;                   // chunks left to copy

  // first: the tile's first row (column of out).  pair: rows from values to gates.
  __device__ __forceinline__ void init(const char* src, int64_t stride, int first, int64_t pair, int64_t k0, int count) {
    if constexpr (ACROSS) next = src + k0 * stride, advance = kChunk * stride;
    else next = src + first * stride + k0 * 2, next_pair = next + pair * stride, advance = kChunk * 2;
    fill = ring, to_copy = count;
  }
  // rows: of the matrix; left: contraction elements of the chunk.
  __device__ __forceinline__ void offsets(int64_t stride, int first, int rows, int wave, int left) {
    const int lane = lane_here();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = wave * kPieces + i;
      if constexpr (ACROSS) {
        const int k = 8 * (piece & 7) + (lane >> 3), place = lane & 7;
        const int col = (piece >> 3) * 64 + (((place >> 1) ^ across_swizzle(k)) * 2 + (place & 1)) * 8;
        off[i] = (unsigned)(min(k, left - 1) * (unsigned)stride) + (unsigned)min(first + col, rows - 8) * 2u;
      } else {
        const int r = 8 * piece + (lane >> 3), q = (lane & 7) ^ (r & 7);
        const int row = PAIRS ? (r >> 5) * 16 + (r & 15) : r;   // (the gates' rows: from their own base)
        off[i] = (unsigned)min(row, rows - 1 - first) * (unsigned)stride + (unsigned)(q * 8 < left ? q * 16 : 0);
      }
    }
  }
  // The two halves of copy I; the last one of a chunk moves on.
  template <int I>
  __device__ __forceinline__ void to() const {
    copy_to<I * 1024>(fill);
  }
  template <int I, Copying C>
  __device__ __forceinline__ void from(unsigned long long lanes) {
    // (with pairs a wave's copies are 8 rows each, two of values and two of gates in turn)
    const char* at = PAIRS && (I & 2) ? next_pair : next;
    if constexpr (C == kCopiesIf) copy_from_if(at, off[I], lanes);
    else copy_from(at, off[I]);
    if constexpr (I == kPieces - 1) {
      next += advance;
      if constexpr (PAIRS) next_pair += advance;
      --to_copy;
      fill = fill == ring + (SLOTS - 1) * kSlot ? ring : fill + kSlot;
    }
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
        at[b] = lds + (8 * g + (c >> 2)) * 128 + (((b + first_block) & 3) ^ across_swizzle(8 * g + (c >> 2))) * 32 + (c & 3) * 8 + (first_block >> 2) * 8192;
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

struct ProductCall {
  ProductParams p;
  ProductShare s;
};
// Memory behind a pointer that comes out of memory: device memory.  (Taken for anywhere, its accesses would wait for each other.)
template <class T>
__device__ __forceinline__ T* in_memory(T* p) {
  return (T*)(__attribute__((address_space(1))) T*)(uintptr_t)p;
}
// The kernel's argument, read anew where it is used: along the loop there are no scalar registers for it.
__device__ __forceinline__ ProductCall call_again() {
  typedef __attribute__((may_alias)) uint64_t Word;
  auto at = (const __attribute__((address_space(4))) uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  ProductCall call;
  static_assert(sizeof(call) % 8 == 0, "copied by words");
#pragma unroll
  for (int i = 0; i < (int)sizeof(call) / 8; ++i) ((Word*)&call)[i] = at[i];
  ProductParams& p = call.p;
  p.bias = in_memory(p.bias), p.gate = in_memory(p.gate), p.gate_index = in_memory(p.gate_index), p.residual = in_memory(p.residual);
  p.pre = in_memory(p.pre), p.out = in_memory(p.out), p.sums = in_memory(p.sums), p.part = in_memory(p.part);
  return call;
}

// A workgroup's way through its tiles.  start() sets out for chunks first .. first + count - 1 of a tile and copies the first few; run() forms the sums.
//
// Copies.  All of a workgroup's copies together take the CU's 64 bytes a clock for half as long as the 256 x 256 products of a chunk take (for longer than
// those of 64 rows), and have to be on their way for about a microsecond.  So the copies of a chunk are issued over the whole of a chunk's time, each half
// in the half chunk behind whose barrier the places they go to are free: `late` ones follow the barrier in the middle of a chunk, `soon` ones the half chunk after.
// Which copies these are and how many places an operand has follows from what fits LDS; the operands' places are counted apart.
template <bool A_ACROSS, bool B_ACROSS, bool PAIRS, int TB, int FB>
struct Walk {
  static constexpr int kTileA = 32 * TB, kTileB = 32 * FB;
  static constexpr int kAhead = FB < 8 ? 0 : TB > 4 ? 2 : 1;   // which of the three ways of copying ahead
  static constexpr int kSlotsB = kAhead ? 3 : 4, kSlotsA = kAhead == 2 ? 2 : 4;
  static constexpr bool kAgpr = TB * FB > 16;
  static_assert(!A_ACROSS || TB % 2 == 0, "units of 64 rows");
  using OB = Operand<B_ACROSS, kTileB, PAIRS, kSlotsB>;
  using OA = Operand<A_ACROSS, kTileA, false, kSlotsA>;
  static constexpr int CB = OB::kPieces, CA = OA::kPieces, PP = CA + CB;
  static constexpr int kBytesB = kSlotsB * OB::kSlot, kLds = kBytesB + kSlotsA * OA::kSlot;
  static constexpr int kReads = FB + TB;
  // copies: 0 .. CB - 1 of B, then of A.  256 x 256: A's behind the barrier, B's after; 128 x 256: the other way round; smaller tiles: half of them all
  static constexpr int kLateFrom = kAhead == 2 ? CB : 0, kLate = kAhead == 2 ? CA : kAhead ? CB : PP / 2;
  static constexpr int kSoonFrom = kAhead == 2 ? 0 : kLate, kSoon = PP - kLate;
  // copies on their way at the middle of a chunk when the next chunk has landed, and the chunks that start() brings on their way whole
  static constexpr int kOnTheirWay = kAhead == 2 ? kSoon : kAhead ? 2 * kSoon + kLate : 2 * PP;
  static constexpr int kStarted = kAhead == 2 ? 2 : 3;
  static constexpr int kLateAhead = kAhead == 2 ? 2 : kAhead ? 3 : 4;   // chunks from the one whose middle they follow to that of the late copies (the soon ones': kStarted)
  int lane, wave, m0, n0, chunks, left;
  OB ob;
  OA oa;
  Images<B_ACROSS> ib;
  Images<A_ACROSS> ia;

  __device__ __forceinline__ explicit Walk(char* lds_raw) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds_raw;
    ob.ring = lds0 + wave * CB * 1024;
    oa.ring = lds0 + kBytesB + wave * CA * 1024;
    ib.init(lds_raw, lane, (wave & 1) * FB);
    ia.init(lds_raw + kBytesB, lane, (wave >> 1) * TB);
  }
  __device__ __forceinline__ void offsets_b(int k_left) {
    const ProductParams p = call_again().p;
    ob.offsets(p.b_stride, n0, p.N, wave, k_left);
  }
  __device__ __forceinline__ void offsets_a(int k_left) {
    const ProductParams p = call_again().p;
    oa.offsets(p.a_stride, m0, p.M, wave, k_left);
  }
  template <int I>
  __device__ __forceinline__ void piece_to() const {
    if constexpr (I < CB) ob.template to<I>();
    else oa.template to<I - CB>();
  }
  template <int I, Copying C>
  __device__ __forceinline__ void piece_from(unsigned long long lanes) {
    if constexpr (I < CB) {
      ob.template from<I, C>(lanes);
      if constexpr (I == CB - 1) {
        if (ob.to_copy == 1 && left < kChunk) offsets_b(left);
      }
    } else {
      oa.template from<I - CB, C>(lanes);
      if constexpr (I == PP - 1) {
        if (oa.to_copy == 1 && left < kChunk) offsets_a(left);
      }
    }
  }
  template <int I, Copying C = kCopies>
  __device__ __forceinline__ void copy_piece(unsigned long long lanes = 0) {
    piece_to<I>();
    asm volatile("s_nop 0");
    piece_from<I, C>(lanes);
  }
  __device__ __forceinline__ void start(int m_first, int n_first, int first, int count) {
    const ProductParams p = call_again().p;
    m0 = m_first, n0 = n_first, chunks = count;
    const int64_t k0 = (int64_t)first * kChunk;
    const int64_t k_left = p.K - k0 - (int64_t)(count - 1) * kChunk;
    left = k_left < kChunk ? (int)k_left : kChunk;   // contraction elements of the last chunk
    ob.init(p.b, p.b_stride, n0, p.N, k0, count);
    oa.init(p.a, p.a_stride, m0, 0, k0, count);
    offsets_b(count == 1 ? left : kChunk);
    offsets_a(count == 1 ? left : kChunk);
    // what the halves of the chunks before the first would have copied
#pragma unroll 1
    for (int i = 0; i < min(kStarted, count); ++i) static_for<PP>([&](auto ic) { copy_piece<decltype(ic)::value>(); });
    if constexpr (kLateAhead > kStarted) {
      if (count > kStarted) static_for<kLate>([&](auto ic) { copy_piece<kLateFrom + decltype(ic)::value>(); });
    }
  }
  // the first chunk that start() copied has landed (of this wave's copies)
  __device__ __forceinline__ void wait_for_first() const {
    constexpr int kBehind = (kStarted - 1) * PP + (kLateAhead > kStarted ? kLate : 0);
    if (chunks > kStarted) __builtin_amdgcn_s_waitcnt(wait_for(kBehind, 15));
    else __builtin_amdgcn_s_waitcnt(wait_for(0, 15));
  }

  template <int I>
  __device__ __forceinline__ void read_image(int ks, int b_bytes, int a_bytes, bf16x8 (&w)[FB], bf16x8 (&x)[TB]) const {
    if constexpr (I < TB) x[I] = ia.template read<I>(ks, a_bytes);
    else w[I - TB] = ib.template read<I - TB>(ks, b_bytes);
  }
  // what lies behind the contraction's end is taken for zeros (both operands: it may be anything)
  __device__ __forceinline__ void clear_rest(int from, bf16x8 (&w)[FB], bf16x8 (&x)[TB]) const {
    i32x4 keep;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int k = from + 8 * (lane >> 4) + 2 * d;
      keep[d] = (k < left ? 0xffff : 0) | (k + 1 < left ? (int)0xffff0000 : 0);
    }
#pragma unroll
    for (int i = 0; i < FB; ++i) w[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(i32x4, w[i]) & keep);
#pragma unroll
    for (int i = 0; i < TB; ++i) x[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(i32x4, x[i]) & keep);
    asm volatile("s_nop 1" ::: "memory");            // (an MFMA may not take a register right behind the instruction that wrote it)
  }
  // Half a chunk (due: whether copies are, positive if so): the products of w and x with, between them, the reads of the next half's images and the copies FROM .. FROM + COUNT - 1.  At most one such thing follows an
  // MFMA where there are enough of them: a wave is alone on its SIMD, and the pipe idles whenever the rest takes longer to issue than the MFMA leaves free.
  // (Blocks of A back and forth: from one MFMA to the next only one operand changes.)
  template <bool FIRST, Copying C, int FROM, int COUNT>
  __device__ __forceinline__ void half(f32x4 (&acc)[TB][FB], bf16x8 (&w)[FB], bf16x8 (&x)[TB], int ks, int b_bytes, int a_bytes, bf16x8 (&w2)[FB], bf16x8 (&x2)[TB],
                                       int due) {
    unsigned long long lanes = 0;
    if constexpr (C == kCopiesIf) asm volatile("s_cmp_gt_i32 %1, 0\n\ts_cselect_b64 %0, -1, 0" : "=s"(lanes) : "s"(due) : "scc");
    if constexpr (FIRST) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_nop 1" ::: "memory");          // (registers that only now become sums)
      __builtin_amdgcn_sched_barrier(0);
    }
    constexpr bool kRoomy = FB * TB >= 2 * kReads && FB * TB / (kSoon > kLate ? kSoon : kLate) >= 4;
    static_for<FB * TB>([&](auto kk) {
      constexpr int k = decltype(kk)::value, fb = k / TB, t = fb & 1 ? TB - 1 - k % TB : k % TB;
      if constexpr (FIRST) mfma_first<kAgpr>(acc[t][fb], w[fb], x[t]);
      else mfma_acc<kAgpr>(acc[t][fb], w[fb], x[t]);
      constexpr int kEvery = FB * TB / COUNT;        // MFMAs from copy to copy
      if constexpr (kRoomy) {                        // a copy's halves follow different MFMAs
        if constexpr (k % 2 == 0 && k / 2 < kReads) read_image<k / 2>(ks, b_bytes, a_bytes, w2, x2);
        if constexpr (C != kNoCopies && k % kEvery == 1 && k / kEvery < COUNT) piece_to<FROM + k / kEvery>();
        if constexpr (C != kNoCopies && k % kEvery == 3 && k / kEvery < COUNT) piece_from<FROM + k / kEvery, C>(lanes);
      } else {
        if constexpr (k < kReads) read_image<k>(ks, b_bytes, a_bytes, w2, x2);
        if constexpr (C != kNoCopies && k % kEvery == 1 && k / kEvery < COUNT) copy_piece<FROM + k / kEvery, C>(lanes);
      }
    });
  }
  // The sums of the tile that start() set out for, whose first chunk has landed for every wave; `landed`: all that start() copied has.
  __device__ __forceinline__ void run(f32x4 (&acc)[TB][FB], bool landed) {
    bf16x8 wa[FB], wb[FB], xa[TB], xb[TB];             // images of a chunk's first and second half
    static_for<kReads>([&](auto ic) { read_image<decltype(ic)::value>(0, 0, 0, wa, xa); });
    int b_here = 0, a_here = 0, kc = 0;              // the chunk's places in LDS, and the chunk
    auto chunk = [&](auto first, auto copying, auto&& wait) __attribute__((always_inline)) {
      constexpr Copying C = decltype(copying)::value;
      const int b_there = b_here == (kSlotsB - 1) * OB::kSlot ? 0 : b_here + OB::kSlot;
      const int a_there = a_here == (kSlotsA - 1) * OA::kSlot ? 0 : a_here + OA::kSlot;
      const bool rest = kc == chunks - 1 && left < kChunk;
      if (rest) clear_rest(0, wa, xa);
      half<decltype(first)::value, C, kSoonFrom, kSoon>(acc, wa, xa, 1, b_here, a_here, wb, xb, chunks - kc - kStarted);
      if (rest) clear_rest(32, wb, xb);
      // every wave holds the chunk in registers, and the next one is in LDS
      wait();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      half<false, C, kLateFrom, kLate>(acc, wb, xb, 0, b_there, a_there, wa, xa, chunks - kc - kLateAhead);
      b_here = b_there, a_here = a_there;
    };
    using No = std::integral_constant<Copying, kNoCopies>;
    using Yes = std::integral_constant<Copying, kCopies>;
    using If = std::integral_constant<Copying, kCopiesIf>;
    chunk(std::true_type{}, If{}, [&]() {
      if (landed) __builtin_amdgcn_s_waitcnt(wait_for(63, 0));
      else if (chunks > kStarted) __builtin_amdgcn_s_waitcnt(wait_for(kOnTheirWay, 0));
      else __builtin_amdgcn_s_waitcnt(wait_for(0, 0));
    });
#pragma unroll 1
    for (kc = 1; kc + kLateAhead < chunks; ++kc)
      chunk(std::false_type{}, Yes{}, [&]() {
        if (kStarted > 2 && landed && kc < kStarted - 1) __builtin_amdgcn_s_waitcnt(wait_for(63, 0));
        else __builtin_amdgcn_s_waitcnt(wait_for(kOnTheirWay, 0));
      });
    // (where the soon copies go less far than the late ones, one of these chunks still has some)
#pragma unroll 1
    for (; kc < chunks; ++kc)
      chunk(std::false_type{}, std::conditional_t<(kLateAhead > kStarted), If, No>{}, [&]() { __builtin_amdgcn_s_waitcnt(wait_for(0, 0)); });
    // the compiler does not know the instructions above for MFMAs: let the last one retire before anything reads the accumulators
    static_for<TB>([&](auto tc) {
      f32x4(&a)[FB] = acc[decltype(tc)::value];
      if constexpr (FB == 4)
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3])::"memory");
      else if constexpr (kAgpr)
        asm volatile("s_nop 15\n\ts_nop 15" : "+a"(a[0]), "+a"(a[1]), "+a"(a[2]), "+a"(a[3]), "+a"(a[4]), "+a"(a[5]), "+a"(a[6]), "+a"(a[7])::"memory");
      else
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7])::"memory");
    });
  }
};

// A wave's results: 16 rows at a time, a lane 16 bytes of a row FB / 2 times (half as often with gates).  What else the results need is asked for a block of rows ahead.
// The accumulators of block t, which is known when the kernel runs: a branch, not an index.
template <int TB, int FB>
__device__ __forceinline__ void block_of(int t, const f32x4 (&acc)[TB][FB], f32x4 (&block)[FB]) {
  static_for<TB>([&](auto tc) {
    if (t == decltype(tc)::value) {
#pragma unroll
      for (int f = 0; f < FB; ++f) block[f] = acc[decltype(tc)::value][f];
    }
  });
}
template <bool PAIRS, int F, int FB>
__device__ __forceinline__ void pieces_of(const f32x4 (&block)[FB], Piece& a, Piece& b) {
  if constexpr (PAIRS) {
    a = eight_columns(block[4 * F], block[4 * F + 2]);
    b = eight_columns(block[4 * F + 1], block[4 * F + 3]);
  } else {
    a = eight_columns(block[2 * F], block[2 * F + 1]);
  }
}

template <int MODE, int ACT, int BESIDES, int TB, int FB>
__device__ __forceinline__ void finish_tile(const ProductParams& p, int m0, int n0, int sum_row, const Bias (&bias)[MODE == kGated ? FB / 4 : FB / 2], const f32x4 (&acc)[TB][FB]) {
  constexpr bool kPairs = MODE == kGated;
  constexpr int kPieces = kPairs ? FB / 4 : FB / 2;   // pieces of a row that a lane holds
  const Results<MODE> res(p, m0);
  const int lane = lane_here(), g = lane >> 4, c = lane & 15, n = n0 + eight_of(g);
  constexpr int kAsked = MODE == kGatedGrad ? 2 : kPieces;   // pieces whose extras are on their way (what the registers allow)
  typename Results<MODE>::Extra extra[kAsked];
  // The rows' places in the gate are asked for before any result leaves: a load waits for the stores before it, and these would wait for two of them in turn at every block
  // (30,543 x 5,144 with a contraction of 344, gate and residual: 410 us so, 317 now).
  constexpr bool kGate = MODE == kPlain && (BESIDES & kWithGate);
  int gate_of[kGate ? TB + 1 : 2] = {};
  if constexpr (kGate) {
#pragma unroll
    for (int t = 0; t < TB; ++t) gate_of[t] = res.gate_row(16 * t + c);
  }
#pragma unroll
  for (int i = 0; i < kAsked; ++i) res.template fetch<ACT, BESIDES>(c, n + 32 * i, gate_of[0], extra[i]);
  Piece sum_a[MODE >= kGrad ? kPieces : 1], sum_b[MODE == kGatedGrad ? kPieces : 1];
  if constexpr (MODE >= kGrad) {
#pragma unroll
    for (int f = 0; f < kPieces; ++f) {
      sum_a[f] = Piece{};
      if constexpr (MODE == kGatedGrad) sum_b[f] = Piece{};
    }
  }
  auto rows_of = [&](int t) __attribute__((always_inline)) {
    f32x4 block[FB];
    block_of<TB, FB>(t, acc, block);
    const int row = 16 * t + c;
    static_for<kPieces>([&](auto fc) {
      constexpr int f = decltype(fc)::value;
      Piece a, b{};
      pieces_of<kPairs, f, FB>(block, a, b);
      res.template finish<ACT, BESIDES>(row, n + 32 * f, a, b, bias[f], extra[f % kAsked]);
      if constexpr (MODE >= kGrad) {
        const bool there = row < res.rows;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum_a[f].v[j] += there ? a.v[j] : 0.f;
          if constexpr (MODE == kGatedGrad) sum_b[f].v[j] += there ? b.v[j] : 0.f;
        }
      }
      constexpr int ahead = f + kAsked;               // (past the last block: rows that nobody uses)
      res.template fetch<ACT, BESIDES>(16 * (t + ahead / kPieces) + c, n + ahead % kPieces * 32, gate_of[ahead / kPieces], extra[f % kAsked]);
      if constexpr (MODE == kGatedGrad) __builtin_amdgcn_sched_barrier(0);   // (one after the other: all at once they would not fit the registers)
    });
    if constexpr (kGate) {
#pragma unroll
      for (int i = 0; i < TB; ++i) gate_of[i] = gate_of[i + 1];
    }
  };
  // The first block by itself: where it met the others in the loop, the compiler would wait for as few accesses on their way as in the first turn, where no result has left yet,
  // and so, in every turn, for stores just issued (1,085 x 2,048 x 2,048, gate and residual: 23.4 us so, 22.8 now).  (Gradients take as long either way.)
  constexpr bool kPeel = BESIDES != 0;
  if constexpr (kPeel) rows_of(0);
#pragma unroll 1
  for (int t = kPeel; t < TB; ++t) rows_of(t);
  if constexpr (MODE >= kGrad) {
    if (p.sums) {
      // over the 16 rows that the lanes of a group hold
      const int columns = MODE == kGatedGrad ? 2 * p.N : p.N;
      float* to = p.sums + (int64_t)sum_row * columns;
      auto put = [&](Piece& v, int at) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float x = v.v[j];
          x = sum_with<0xB1>(x);
          x = sum_with<0x4E>(x);
          x = sum_with<0x141>(x);
          v.v[j] = sum_with<0x140>(x);
        }
        if (c == 0) store_piece_f32((char*)(to + at), v);
      };
#pragma unroll
      for (int f = 0; f < kPieces; ++f) {
        if (n + 32 * f >= p.N) continue;
        put(sum_a[f], n + 32 * f);
        if constexpr (MODE == kGatedGrad) put(sum_b[f], p.N + n + 32 * f);
      }
    }
  }
}

// The sums of a part of a contraction, as they are: rows as wide as the tile (values and gates: half of it each).
template <bool PAIRS, int TB, int FB>
__device__ __forceinline__ void leave_part(float* part, int rows, const f32x4 (&acc)[TB][FB]) {
  const int lane = lane_here(), g = lane >> 4, c = lane & 15;
#pragma unroll 1
  for (int t = 0; t < TB; ++t) {
    if (16 * t >= rows) break;
    f32x4 block[FB];
    block_of<TB, FB>(t, acc, block);
    // (values and gates: blocks of them in turn)
#pragma unroll
    for (int f = 0; f < FB; ++f)
      *(f32x4*)(part + (16 * t + c) * 32 * FB + 4 * g + (PAIRS ? (f >> 1) * 16 + (f & 1) * 16 * FB : f * 16)) = block[f];
  }
}

template <bool A_ACROSS, bool B_ACROSS, int MODE, int TB, int FB>
__global__ __launch_bounds__(256, 1) void product_kernel(ProductCall) {
  constexpr bool kPairs = MODE == kGated;
  constexpr int kColumns = kPairs ? 16 * FB : 32 * FB;   // of out, a tile
  using W = Walk<A_ACROSS, B_ACROSS, kPairs, TB, FB>;
  __shared__ __attribute__((aligned(1024))) char lds_raw[W::kLds];
  int turn = 0, m_tile = 0, n_tile = 0, first = 0, count = 0, slot = 0;
  // The next tile or part of one; false: none.  (Values chosen, not branches taken: the compiler keeps what either branch writes in memory.)
  auto advance = [&]() __attribute__((always_inline)) {
    const ProductShare s = call_again().s;
    const bool whole = turn < s.rounds;
    const int turns = whole ? s.rounds : part_turns(s), unit = unit_of(turns, whole ? turn : turn - s.rounds, blockIdx.x, s.groups);
    const bool more = whole || (turn - s.rounds < turns && unit < units_of(s));
    const int part = whole || !more ? 0 : unit / s.rest;
    const TilePlace place = tile_of(s, whole ? unit : s.rounds * s.groups + unit - part * s.rest);
    const int from = part_begin(s, part), to = whole ? s.chunks : part_begin(s, part + 1);
    ++turn;
    // (uniform, which the compiler loses sight of on the way)
    m_tile = __builtin_amdgcn_readfirstlane(place.m), n_tile = __builtin_amdgcn_readfirstlane(place.n);
    first = __builtin_amdgcn_readfirstlane(from), count = __builtin_amdgcn_readfirstlane(to - from);
    slot = __builtin_amdgcn_readfirstlane(whole || s.cuts == 1 ? -1 : unit);
    return __builtin_amdgcn_readfirstlane(more);
  };
  if (!advance()) return;
  W walk(lds_raw);
  auto set_out = [&]() __attribute__((always_inline)) { walk.start(m_tile * 32 * TB, n_tile * kColumns, first, count); };
  set_out();
  walk.wait_for_first();
  bool landed = false;
#pragma unroll 1
  for (;;) {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f32x4 acc[TB][FB];
    const int wave = walk.wave, wm = (wave >> 1) * 16 * TB, wn = (wave & 1) * (kColumns / 2);
    const int m0 = m_tile * 32 * TB + wm, n0 = n_tile * kColumns + wn, sum_row = m_tile * 2 + (wave >> 1);
    constexpr int kPieces = kPairs ? FB / 4 : FB / 2;
    Bias bias[kPieces];                                // (asked for here, it is there when the sums are)
    {
      const ProductParams p = call_again().p;
      const int n = n0 + eight_of(lane_here() >> 4);
#pragma unroll
      for (int f = 0; f < kPieces; ++f) bias[f] = B_ACROSS ? Bias{} : load_bias<MODE>(p, min(n + 32 * f, p.N - 8));
    }
    walk.run(acc, landed);
    const ProductParams p = call_again().p;
    float* part = slot < 0 ? nullptr : p.part + ((int64_t)slot * 32 * TB + wm) * 32 * FB + wn;
    const bool filled = p.M > m0;                      // the wave has rows: then at least so many of its stores were issued as results have pieces
    __builtin_amdgcn_s_waitcnt(wait_for(63, 0));
    __builtin_amdgcn_s_barrier();                      // (no wave reads chunks any more)
    asm volatile("" ::: "memory");
    const bool more = advance();
    if (more) set_out();                               // (the next tile's first chunks are on their way while this one's results leave)
    const bool whole = !part;
    if (part) {
      leave_part<kPairs, TB, FB>(part, p.M - m0, acc);
    } else if (p.M > m0 || MODE >= kGrad) {
      const ProductParams q = call_again().p;
      with_form<MODE, MODE == kPlain && B_ACROSS>(q, [&](auto act, auto besides) {
        finish_tile<MODE, decltype(act)::value, decltype(besides)::value, TB, FB>(q, m0, n0, sum_row, bias, acc);
      });
    }
    if (!more) break;
    // The copies are older than the epilogue's stores, of which there were at least so many, and both complete in their order.
    constexpr int kStores = TB * kPieces;
    if (whole && filled) __builtin_amdgcn_s_waitcnt(wait_for(kStores, 15));
    else __builtin_amdgcn_s_waitcnt(wait_for(0, 15));
    landed = true;
  }
}

template <int TB, int FB>
hipError_t launch_tiles_of(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s) {
  const dim3 grid(plan.share.groups);
  if (a_across) {
    if constexpr (TB % 2 == 0) product_kernel<true, true, kPlain, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  } else if (!b_across && mode == kPlain) product_kernel<false, false, kPlain, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  else if (!b_across) product_kernel<false, false, kGated, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  else if (mode == kPlain) product_kernel<false, true, kPlain, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  else if (mode == kGrad) product_kernel<false, true, kGrad, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  else product_kernel<false, true, kGatedGrad, TB, FB><<<grid, 256, 0, s>>>({p, plan.share});
  return hipGetLastError();
}

}  // namespace pkh3
