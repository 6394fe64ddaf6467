// Matrix products on plain row-major matrices that finish their own results (include/pkh3_rows.h): out[m, n] = finish(sum over k of A(m, k) B(n, k)).
#include "pkh3_rows.h"

namespace pkh3 {

constexpr int kTile = 128;        // rows of A and rows of B of a workgroup's tile
constexpr int kStep = 32;         // contraction elements of a round
constexpr int kPitch = kStep + 8; // elements between rows of a staged tile
constexpr int kStagePitch = 64 + 4;   // floats between rows of staged results

// Rows first .. first + 127 (of `rows`), contraction elements k .. k + 31 (of K) of a matrix into LDS, zeros where there are none.
// row_of: the matrix's row behind a row of the tile, or -1.
template <bool ACROSS, class F>
__device__ __forceinline__ void stage(const char* src, int64_t stride, int k, int K, F&& row_of, __bf16* lds) {
  if constexpr (!ACROSS) {
    for (int i = threadIdx.x; i < kTile * 4; i += 256) {
      const int r = i >> 2, kk = (i & 3) * 8, row = row_of(r);
      bf16x8 v{};
      if (row >= 0 && k + kk < K) v = *(const bf16x8*)(src + row * stride + (int64_t)(k + kk) * 2);
      *(bf16x8*)(lds + r * kPitch + kk) = v;
    }
  } else {
    for (int i = threadIdx.x; i < kStep * (kTile / 8); i += 256) {
      const int kk = i / (kTile / 8), r = i % (kTile / 8) * 8, row = row_of(r);
      bf16x8 v{};
      if (row >= 0 && k + kk < K) v = *(const bf16x8*)(src + (k + kk) * stride + (int64_t)row * 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) lds[(r + j) * kPitch + kk] = v[j];
    }
  }
}

template <bool A_ACROSS, bool B_ACROSS, int MODE>
__global__ __launch_bounds__(256) void product_kernel(ProductParams p) {
  constexpr bool kPairs = MODE == kGated;
  constexpr int kCols = kPairs ? kTile / 2 : kTile;   // columns of out of a tile
  __shared__ __attribute__((aligned(16))) __bf16 ta[kTile * kPitch], tb[kTile * kPitch];
  __shared__ __attribute__((aligned(16))) float staged[4][16 * kStagePitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.x * kCols, m0 = blockIdx.y * kTile;
  auto a_row = [&](int r) { return m0 + r < p.M ? m0 + r : -1; };
  // 16 rows of values, then 16 rows of their gates, in turn
  auto b_row = [&](int r) {
    const int n = kPairs ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
    return n >= p.N ? -1 : kPairs && (r & 16) ? n + p.N : n;
  };
  const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
  f32x4 acc[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[t][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < p.K; k += kStep) {
    __syncthreads();
    stage<A_ACROSS>(p.a, p.a_stride, k, p.K, a_row, ta);
    stage<B_ACROSS>(p.b, p.b_stride, k, p.K, b_row, tb);
    __syncthreads();
    bf16x8 x[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = *(const bf16x8*)(ta + (wm + 16 * i + c) * kPitch + 8 * g);
      w[i] = *(const bf16x8*)(tb + (wn + 16 * i + c) * kPitch + 8 * g);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[t][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[f], x[t], acc[t][f], 0, 0, 0);
  }
  // 16 rows at a time through LDS, so that a row's results leave in 16-byte pieces beside each other
  constexpr int kPieces = kPairs ? 4 : 8;             // pieces of a row of the wave
  constexpr int kRows = 64 / kPieces;                 // rows at a time
  float* lds = staged[wave];
  const int piece = lane % kPieces, n = n0 + (kPairs ? wn / 2 : wn) + piece * 8;
  const bool live = n < p.N;
  Bias bias{};
  if (live) bias = load_bias<MODE>(p, n);
  Piece sum_a{}, sum_b{};
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int f = 0; f < 4; ++f) *(f32x4*)(lds + c * kStagePitch + 16 * f + 4 * g) = acc[t][f];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 16 / kRows; ++i) {
        const int r = i * kRows + lane / kPieces, m = m0 + wm + 16 * t + r;
        if (!live || m >= p.M) continue;
        const float* at = lds + r * kStagePitch + (kPairs ? (piece >> 1) * 32 + (piece & 1) * 8 : piece * 8);
        Piece a = load_piece_f32((const char*)at), b{};
        if constexpr (kPairs) b = load_piece_f32((const char*)(at + 16));
        finish<MODE, decltype(act)::value>(p, m, n, a, b, bias);
        if (MODE >= kGrad && p.sums) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum_a.v[j] += a.v[j], sum_b.v[j] += b.v[j];
        }
      }
    }
  });
  if constexpr (MODE >= kGrad) {
    if (p.sums) {
      const int columns = MODE == kGatedGrad ? 2 * p.N : p.N;
      float* at = p.sums + (int64_t)(blockIdx.y * 2 + (wave >> 1)) * columns + n;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        for (int over = kPieces; over < 64; over *= 2) {
          sum_a.v[j] += __shfl_xor(sum_a.v[j], over, 64);
          sum_b.v[j] += __shfl_xor(sum_b.v[j], over, 64);
        }
        if (live && lane < kPieces) {
          at[j] = sum_a.v[j];
          if (MODE == kGatedGrad) at[p.N + j] = sum_b.v[j];
        }
      }
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

ProductPlan plan_product(int M, int N, int K, bool a_across, bool b_across, int mode, bool sums) {
  ProductPlan plan{};
  plan.sum_rows = sums ? (M + kTile - 1) / kTile * 2 : 0;
  plan.total = round_up((size_t)plan.sum_rows * (mode == kGatedGrad ? 2 : 1) * N * sizeof(float));
  return plan;
}

template <bool A_ACROSS, bool B_ACROSS>
static void launch_mode(const ProductParams& p, int mode, hipStream_t s) {
  const dim3 grid((p.N + (mode == kGated ? kTile / 2 : kTile) - 1) / (mode == kGated ? kTile / 2 : kTile), (p.M + kTile - 1) / kTile);
  if (mode == kPlain) product_kernel<A_ACROSS, B_ACROSS, kPlain><<<grid, 256, 0, s>>>(p);
  else if (mode == kGated) product_kernel<A_ACROSS, B_ACROSS, kGated><<<grid, 256, 0, s>>>(p);
  else if (mode == kGrad) product_kernel<A_ACROSS, B_ACROSS, kGrad><<<grid, 256, 0, s>>>(p);
  else product_kernel<A_ACROSS, B_ACROSS, kGatedGrad><<<grid, 256, 0, s>>>(p);
}

static hipError_t launch_column_sums(const float* part, int rows, int columns, void* out, hipStream_t s) {
  column_sums_kernel<<<(columns + 31) / 32, 256, 0, s>>>(part, rows, columns, (__bf16*)out);
  return hipGetLastError();
}

hipError_t launch_product(ProductParams p, const ProductPlan& plan, bool a_across, bool b_across, int mode, void* sums, char* workspace, hipStream_t s) {
  p.sums = sums ? (float*)(workspace + plan.sums_off) : nullptr;
  if (a_across && b_across) launch_mode<true, true>(p, mode, s);
  else if (a_across) launch_mode<true, false>(p, mode, s);
  else if (b_across) launch_mode<false, true>(p, mode, s);
  else launch_mode<false, false>(p, mode, s);
  const hipError_t e = hipGetLastError();
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
      if (p.out) finish<kGrad, ACT>(p, m, n, a, b, Bias{});
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
