// Products of few rows (include/pkh3_rows.h, both operands along): what counts is how soon the weights are there.
//
// A workgroup is 16 or 32 columns (with gates 16 columns and their gates) times up to 64 rows, so that also a narrow layer has a workgroup for half of the CUs, and its
// waves share the contraction out.  No two of them read the same pieces, so every wave has a ring of chunks in LDS of its own and waits for its own copies alone, without a
// barrier; the waves' sums meet in LDS and are added up in the order of the contraction.  The way through LDS is for the copies: 128 bytes of a row by
// lanes beside each other take the CU's vector-memory path a quarter of the time that images straight into the registers take, where such lanes lie in
// different rows (16 rows, 4,096 x 12,288: 34 us that way).
//
// Bound by the weights: one row, 2,048 to 8,192, weights out of memory 8.6 us (3.9 TB/s, 2 us of them the launch) and 4.9 out of L2; 128 rows, 2,048 to 2,048 8.5, where tiles take 19;
// 200 rows, 8,192 to 2,048 25, tiles 24.  Where there are some more than 256 workgroups, a few CUs have two (10 rows, 4,368 to 8,960, 280 of them: 28.6 us, tiles 25.6).
#include "pkh3_rows.h"

namespace pkh3 {

constexpr int kThinWaves = 4;

template <int MODE, int TM, int FB, int DEPTH>
__global__ __launch_bounds__(64 * kThinWaves) void thin_product_kernel(ProductParams p) {
  constexpr bool kPairs = MODE == kGated;
  static_assert(!kPairs || FB == 2, "values and gates");
  constexpr int kCols = kPairs || FB == 1 ? 16 : 32, kBlocks = FB + TM, kSlot = kBlocks * 2048;
  static_assert(TM * FB * 1024 <= DEPTH * kSlot, "the sums go through the chunks' places");
  __shared__ __attribute__((aligned(1024))) char lds_raw[kThinWaves * DEPTH * kSlot];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * kCols, m0 = blockIdx.y * 16 * TM;
  const int chunks = (p.K + kChunk - 1) / kChunk, first = chunks * wave / kThinWaves, count = chunks * (wave + 1) / kThinWaves - first;
  const int left = p.K - (chunks - 1) * kChunk;        // contraction elements of the last chunk
  f32x4 acc[TM][FB];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int f = 0; f < FB; ++f) acc[t][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (count > 0) {
    // blocks of 16 rows: the columns' weights, then the rows; two copies of 8 rows a chunk each.  The piece q of row r lies at place q ^ (r % 8).
    const char* base[kBlocks];
    unsigned off[kBlocks][2], off_rest[kBlocks][2];
    const int q = (lane & 7) ^ (lane >> 3), q_rest = q * 8 < left ? q : 0;
    static_for<kBlocks>([&](auto bc) {
      constexpr int b = decltype(bc)::value;
      const int at = b < FB ? (kPairs ? n0 : n0 + 16 * b) : m0 + 16 * (b - FB), rows = b < FB ? p.N : p.M;
      const int64_t stride = b < FB ? p.b_stride : p.a_stride;
      const int from = min(at, rows - 1) + (kPairs && b == 1 ? p.N : 0);
      base[b] = (b < FB ? p.b : p.a) + from * stride + (int64_t)first * kChunk * 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned row = (unsigned)min(8 * h + (lane >> 3), rows - 1 - min(at, rows - 1)) * (unsigned)stride;
        off[b][h] = row + q * 16;
        off_rest[b][h] = row + q_rest * 16;
      }
    });
    const unsigned ring = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds_raw + wave * DEPTH * kSlot;
    const char* mine = lds_raw + wave * DEPTH * kSlot;
    // chunk i of the wave's into place `to` (past the last one: that one again, which nobody reads)
    auto copy = [&](int i, unsigned to) {
      const int at = min(i, count - 1);
      const bool rest = first + at == chunks - 1;
      static_for<kBlocks>([&](auto bc) {
        constexpr int b = decltype(bc)::value;
        const char* from = base[b] + (int64_t)at * (kChunk * 2);
        copy_to<b * 2048>(to);
        asm volatile("s_nop 0");
        copy_from(from, rest ? off_rest[b][0] : off[b][0]);
        copy_to<b * 2048 + 1024>(to);
        asm volatile("s_nop 0");
        copy_from(from, rest ? off_rest[b][1] : off[b][1]);
      });
    };
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) copy(i, ring + i * kSlot);
    int here = 0, before = (DEPTH - 1) * kSlot;          // the chunk's place, and that of the one before it
    const int image = c * 128, k0 = ((g ^ (c & 7)) * 16);
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      __builtin_amdgcn_s_waitcnt(wait_for(63, 0));       // the chunk before is in registers, its place free
      asm volatile("" ::: "memory");
      copy(i + DEPTH - 1, ring + before);
      __builtin_amdgcn_s_waitcnt(wait_for((DEPTH - 1) * kBlocks * 2, 15));
      asm volatile("" ::: "memory");
      bf16x8 im[2][kBlocks];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) im[ks][b] = *(const bf16x8*)(mine + here + b * 2048 + image + (k0 ^ (ks * 64)));
      if (first + i == chunks - 1 && left < kChunk) {    // zeros behind the contraction's end, in both operands
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const int keep = 32 * ks + 8 * g < left ? -1 : 0;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) im[ks][b] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(i32x4, im[ks][b]) & i32x4{keep, keep, keep, keep});
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
          for (int t = 0; t < TM; ++t) acc[t][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(im[ks][f], im[ks][FB + t], acc[t][f], 0, 0, 0);
      before = here;
      here = here == (DEPTH - 1) * kSlot ? 0 : here + kSlot;
    }
    __builtin_amdgcn_s_waitcnt(wait_for(0, 0));          // (the copies that nobody reads)
  }
  __syncthreads();                                       // every wave is through with its ring, where the sums go now
  f32x4* staged = (f32x4*)lds_raw;
  auto at = [&](int w, int block) { return staged + (w * TM * FB + block) * 64 + lane; };
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int f = 0; f < FB; ++f) *at(wave, t * FB + f) = acc[t][f];
  __syncthreads();
  if (wave >= TM) return;
  // wave t finishes block t of 16 rows
  f32x4 sum[FB];
#pragma unroll
  for (int f = 0; f < FB; ++f) {
    sum[f] = *at(0, wave * FB + f);
    for (int i = 1; i < kThinWaves; ++i) sum[f] += *at(i, wave * FB + f);
  }
  const Results<MODE> res(p, m0 + 16 * wave);
  // eight columns beside each other: out of two blocks, or of one, then in every other group of lanes
  const bool both = FB == 2 && !kPairs;
  Piece a = eight_columns(sum[0], sum[both ? 1 : 0]), b{};
  if constexpr (kPairs) b = eight_columns(sum[1], sum[1]);
  const int n = n0 + (both ? eight_of(g) : (g >> 1) * 8), row = both || !(g & 1) ? c : res.rows;
  const Bias bias = load_bias<MODE>(p, min(n, p.N - 8));
  if (res.rows <= 0) return;
  with_form<MODE, false>(p, [&](auto act, auto besides) {
    typename Results<MODE>::Extra extra;
    res.template fetch<decltype(act)::value, decltype(besides)::value>(row, n, decltype(besides)::value & kWithGate ? res.gate_row(row) : 0, extra);
    res.template finish<decltype(act)::value, decltype(besides)::value>(row, n, a, b, bias, extra);
  });
}

// Chunks of a wave in LDS: 64 to 144 KiB a workgroup.  Of narrow ones there may be more than CUs, and with up to 80 KiB two of them share one (one row, 2,048 to 6,000, weights out
// of memory: 10.6 us with eight waves and 128 KiB a workgroup, now 8.0; 24 rows, 2,048 to 5,120 12.7 with 144 KiB, now 10; 48 rows 14.8 with 120, now 12.8).
template <int MODE, int FB>
static void launch_rows(const ProductParams& p, hipStream_t s) {
  constexpr int kCols = MODE == kGated || FB == 1 ? 16 : 32;
  const int columns = (p.N + kCols - 1) / kCols;
  auto launch = [&](auto tm, auto depth) {
    constexpr int TM = decltype(tm)::value;
    thin_product_kernel<MODE, TM, FB, decltype(depth)::value><<<dim3(columns, (p.M + 16 * TM - 1) / (16 * TM)), 64 * kThinWaves, 0, s>>>(p);
  };
  using std::integral_constant;
  if (p.M <= 16) launch(integral_constant<int, 1>{}, integral_constant<int, FB == 1 ? 4 : 3>{});
  else if (p.M <= 32) launch(integral_constant<int, 2>{}, integral_constant<int, 3>{});
  else launch(integral_constant<int, 4>{}, integral_constant<int, FB == 1 ? 2 : 3>{});
}

hipError_t launch_thin(const ProductParams& p, int mode, hipStream_t s) {
  if (mode == kGated) launch_rows<kGated, 2>(p, s);
  else if (thin_narrow(p.M, p.N)) launch_rows<kPlain, 1>(p, s);
  else launch_rows<kPlain, 2>(p, s);
  return hipGetLastError();
}

}  // namespace pkh3
