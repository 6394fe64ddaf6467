// How products are carried out (include/pkh3_rows.h): the choice of tiles, the joining of contractions that were cut, sums of columns; and the gradient of an activation.
#include "pkh3_rows.h"

namespace pkh3 {

// The parts of the tiles whose contraction was cut, added up in their order, and finished: a workgroup is 8 pieces of 8 columns times 32 rows; with
// sums of columns it takes as many rows as a wave of product_kernel has, whose place in the sums it fills.
template <int MODE>
__global__ __launch_bounds__(256) void product_join_kernel(ProductParams p, ProductShare s, int tb, int fb) {
  constexpr bool kPairs = MODE == kGated;
  const int wide = 32 * fb, columns = kPairs ? wide / 2 : wide;
  __shared__ __attribute__((aligned(16))) Piece staged[MODE >= kGrad ? 2 * 256 : 1];
  const int rows = MODE >= kGrad ? 16 * tb : 32;
  const auto [m_tile, n_tile] = tile_of(s, s.rounds * s.groups + blockIdx.x);
  const Results<MODE> res(p, m_tile * 32 * tb + blockIdx.y * rows);
  const int col = (blockIdx.z * 8 + (threadIdx.x & 7)) * 8, n = n_tile * columns + col;
  Piece sum_a{}, sum_b{};
  with_form<MODE, false>(p, [&](auto act, auto besides) {
    for (int r = threadIdx.x >> 3; r < rows; r += 32) {
      if (n >= p.N || r >= res.rows) break;
      typename Results<MODE>::Extra extra;
      res.template fetch<decltype(act)::value, decltype(besides)::value>(r, n, decltype(besides)::value & kWithGate ? res.gate_row(r) : 0, extra);
      const Bias bias = load_bias<MODE>(p, n);
      Piece a{}, b{};
      for (int part = 0; part < s.cuts; ++part) {
        const int64_t slot = (int64_t)part * s.rest + blockIdx.x;
        const char* from = (const char*)(p.part + (slot * 32 * tb + blockIdx.y * rows + r) * wide + col);
        const Piece va = load_piece_f32(from);
#pragma unroll
        for (int j = 0; j < 8; ++j) a.v[j] += va.v[j];
        if constexpr (kPairs) {
          const Piece vb = load_piece_f32(from + columns * 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) b.v[j] += vb.v[j];
        }
      }
      res.template finish<decltype(act)::value, decltype(besides)::value>(r, n, a, b, bias, extra);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum_a.v[j] += a.v[j], sum_b.v[j] += b.v[j];
    }
  });
  if constexpr (MODE >= kGrad) {
    if (!p.sums) return;
    staged[threadIdx.x] = sum_a;
    staged[256 + threadIdx.x] = sum_b;
    for (int over = 128; over >= 8; over /= 2) {
      __syncthreads();
      const int i = threadIdx.x & 127, half = threadIdx.x >> 7;
      if (i < over) {
#pragma unroll
        for (int j = 0; j < 8; ++j) staged[half * 256 + i].v[j] += staged[half * 256 + i + over].v[j];
      }
    }
    const int half = threadIdx.x >> 7;
    if ((threadIdx.x & 127) < 8 && n < p.N && (MODE == kGatedGrad || !half)) {
      float* to = p.sums + (int64_t)(m_tile * 2 + blockIdx.y) * (MODE == kGatedGrad ? 2 * p.N : p.N) + half * p.N + n;
      store_piece_f32((char*)to, staged[half * 256 + (threadIdx.x & 7)]);
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

static hipError_t launch_column_sums(const float* part, int rows, int columns, void* out, hipStream_t s) {
  column_sums_kernel<<<(columns + 31) / 32, 256, 0, s>>>(part, rows, columns, (__bf16*)out);
  return hipGetLastError();
}

hipError_t launch_product(ProductParams p, const ProductPlan& plan, bool a_across, bool b_across, int mode, void* sums, char* workspace, hipStream_t s) {
  p.sums = sums ? (float*)(workspace + plan.sums_off) : nullptr;
  const bool cut = plan.share.cuts > 1;
  p.part = cut ? (float*)(workspace + plan.part_off) : nullptr;
  if (plan.thin) return launch_thin(p, mode, s);
  hipError_t e;
  if (plan.tb == 8) e = launch_tiles_8(p, plan, a_across, b_across, mode, s);
  else if (plan.fb == 8) e = launch_tiles_4(p, plan, a_across, b_across, mode, s);
  else if (plan.tb == 4) e = launch_tiles_4x4(p, plan, a_across, b_across, mode, s);
  else if (plan.tb == 3) e = launch_tiles_3x4(p, plan, a_across, b_across, mode, s);
  else e = launch_tiles_2x4(p, plan, a_across, b_across, mode, s);
  if (e != hipSuccess) return e;
  if (cut) {
    const dim3 grid(plan.share.rest, mode >= kGrad ? 2 : plan.tb, plan.fb / (mode == kGated ? 4 : 2));
    if (mode == kPlain) product_join_kernel<kPlain><<<grid, 256, 0, s>>>(p, plan.share, plan.tb, plan.fb);
    else if (mode == kGated) product_join_kernel<kGated><<<grid, 256, 0, s>>>(p, plan.share, plan.tb, plan.fb);
    else if (mode == kGrad) product_join_kernel<kGrad><<<grid, 256, 0, s>>>(p, plan.share, plan.tb, plan.fb);
    else product_join_kernel<kGatedGrad><<<grid, 256, 0, s>>>(p, plan.share, plan.tb, plan.fb);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (!sums) return e;
  return launch_column_sums(p.sums, plan.sum_rows, mode == kGatedGrad ? 2 * p.N : p.N, sums, s);
}

// ---- the gradient of an activation, and the sums of its columns ----

constexpr int kGradRows = 64;     // rows of a workgroup: 8 at a time, 32 pieces of 8 columns

template <int ACT>
__global__ __launch_bounds__(256) void activation_grad_kernel(ProductParams p) {
  __shared__ Piece staged[256];
  const int n = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8, first = blockIdx.y * kGradRows;
  const Results<kGrad> res(p, first);
  Piece sum{};
  if (n < p.N)
    for (int i = threadIdx.x >> 5; i < kGradRows && i < res.rows; i += 8) {
      Piece a = load_piece(p.a + (first + i) * p.a_stride + (int64_t)n * 2), b{};
      if (p.out) {
        Results<kGrad>::Extra extra;
        res.fetch<ACT, 0>(i, n, 0, extra);
        res.finish<ACT, 0>(i, n, a, b, Bias{}, extra);
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
