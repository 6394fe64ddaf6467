// Layer norm with tables (include/pkh3_rows.h), forward and backward.
//
//   forward    y = xh w[r] + b[r], xh = (x - mean) rstd
//   backward   g = dy w[r]:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw[r] = sum of dy xh, db[r] = sum of dy over the rows of table row r
//
// A row lies in the registers of the lanes that share it (a wave up to 2,048 elements, a workgroup above), 8 elements a piece, so memory is read once
// and the variance is taken about the mean.  The backward pass forms the statistics again from the row, which it needs anyway, instead of keeping them.  Both
// are bound by memory.
//
// Sums for the tables: every workgroup takes one run of rows and keeps the sums of the table row that it is at in registers (its rows come
// in runs of one table row, so they rarely change); when the table row changes, and at the end, the workgroup's lanes add up in LDS and the sums go to the
// workgroup's own slice of the workspace.  A second launch adds the slices up in their order: no atomics, the same bits every time.
#include "pkh3_rows.h"

namespace pkh3 {

constexpr int kNormThreads = 256;

// `count` values summed over the LANES lanes that share a row
template <int LANES, int COUNT>
__device__ __forceinline__ void row_sums(float (&x)[COUNT], float* lds) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) x[i] = wave_sum(x[i]);
  if constexpr (LANES == 256) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();                                  // (what the sums before these were read from)
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) lds[wave * COUNT + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) x[i] = (lds[i] + lds[COUNT + i]) + (lds[2 * COUNT + i] + lds[3 * COUNT + i]);
  }
}

template <bool F32>
__device__ __forceinline__ Piece load_row_piece(const char* row, int n) {
  return F32 ? load_piece_f32(row + (int64_t)n * 4) : load_piece(row + (int64_t)n * 2);
}
template <bool F32>
__device__ __forceinline__ void store_row_piece(char* row, int n, const Piece& p) {
  if constexpr (F32) {
    store_piece_f32(row + (int64_t)n * 4, p);
  } else {
    store_piece(row + (int64_t)n * 2, p);
  }
}

// A row of NP pieces a lane: loaded (zeros past its end), its mean taken off, and 1 / sqrt(variance + eps) returned.
template <bool F32, int LANES, int NP>
struct Row {
  Piece x[NP];
  __device__ __forceinline__ void load(const char* row, int lane, int width) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int n = (i * LANES + lane) * 8;
      x[i] = n < width ? load_row_piece<F32>(row, n) : Piece{};
    }
  }
  __device__ __forceinline__ float centre(int lane, int width, float eps, float* lds) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += x[i].v[j];
    row_sums<LANES>(s, lds);
    const float mean = s[0] / (float)width;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const bool live = (i * LANES + lane) * 8 < width;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[i].v[j] = live ? x[i].v[j] - mean : 0.f;
        s[0] += x[i].v[j] * x[i].v[j];
      }
    }
    row_sums<LANES>(s, lds);
    return 1.0f / sqrtf(s[0] / (float)width + eps);
  }
};

__device__ __forceinline__ int table_of(const NormParams& p, int row) { return p.row_index ? min(max(p.row_index[row], 0), p.tables - 1) : 0; }

template <bool F32, bool TB16, int LANES, int NP>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(NormParams p) {
  __shared__ float lds[4];
  const int lane = threadIdx.x % LANES;
  const int row = blockIdx.x * (kNormThreads / LANES) + threadIdx.x / LANES;
  if (row >= p.rows) return;                          // (whole waves, and with LANES == 256 none)
  Row<F32, LANES, NP> r;
  r.load(p.x + row * p.x_stride, lane, p.width);
  const int64_t table = (int64_t)table_of(p, row) * p.width;
  const float rstd = r.centre(lane, p.width, p.eps, lds);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int n = (i * LANES + lane) * 8;
    if (n >= p.width) break;
    Piece y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y.v[j] = r.x[i].v[j] * rstd;
    if (p.weight) {
      const Piece w = load_table(p.weight, table + n, TB16);
#pragma unroll
      for (int j = 0; j < 8; ++j) y.v[j] *= w.v[j];
    }
    if (p.bias) {
      const Piece b = load_table(p.bias, table + n, TB16);
#pragma unroll
      for (int j = 0; j < 8; ++j) y.v[j] += b.v[j];
    }
    store_row_piece<F32>(p.out + row * p.out_stride, n, y);
  }
}

// slice of a workgroup: [table][weights' sums, biases' sums][width]
__host__ __device__ inline int64_t slice_floats(int tables, int width) { return (int64_t)tables * 2 * width; }

template <bool F32, bool TB16, int LANES, int NP>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(NormParams p) {
  constexpr int kRows = kNormThreads / LANES;         // rows at a time
  __shared__ float lds[8];
  __shared__ __attribute__((aligned(16))) float staged[LANES == 64 ? 3 * 64 * 8 : 1];
  const int lane = threadIdx.x % LANES, which = threadIdx.x / LANES;
  const int first = (int)((int64_t)p.rows * blockIdx.x / p.groups), end = (int)((int64_t)p.rows * (blockIdx.x + 1) / p.groups);
  float* slice = p.part + (int64_t)blockIdx.x * slice_floats(p.tables, p.width);
  const bool sums = p.part != nullptr;
  uint64_t touched = 0;
  int at = first;
  while (at < end) {                                  // rows at .. to - 1 take table row t
    const int t = __builtin_amdgcn_readfirstlane(table_of(p, at));
    int to = end;
    if (p.row_index) {
      to = at + 1;
      while (to < end) {
        const int look = to + (int)(threadIdx.x & 63);
        const uint64_t other = __ballot(look < end && table_of(p, look) != t);
        if (other) {
          to += __builtin_ctzll(other);
          break;
        }
        to = min(to + 64, end);
      }
    }
    Piece w[NP], dw[NP], db[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int n = (i * LANES + lane) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[i].v[j] = 1.f, dw[i].v[j] = 0.f, db[i].v[j] = 0.f;
      if (p.weight && n < p.width) w[i] = load_table(p.weight, (int64_t)t * p.width + n, TB16);
    }
    for (int row = at + which; row < to; row += kRows) {
      Row<F32, LANES, NP> r, d;
      r.load(p.x + row * p.x_stride, lane, p.width);
      d.load(p.dy + row * p.dy_stride, lane, p.width);
      const float rstd = r.centre(lane, p.width, p.eps, lds);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = r.x[i].v[j] * rstd, g = d.x[i].v[j] * w[i].v[j];
          r.x[i].v[j] = xh;
          dw[i].v[j] += d.x[i].v[j] * xh;
          db[i].v[j] += d.x[i].v[j];
          d.x[i].v[j] = g;
          s[0] += g;
          s[1] += g * xh;
        }
      row_sums<LANES>(s, lds);
      const float mean_g = s[0] / (float)p.width, mean_gx = s[1] / (float)p.width;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int n = (i * LANES + lane) * 8;
        if (n >= p.width) break;
        Piece y;
#pragma unroll
        for (int j = 0; j < 8; ++j) y.v[j] = rstd * (d.x[i].v[j] - mean_g - r.x[i].v[j] * mean_gx);
        store_row_piece<F32>(p.dx + row * p.dx_stride, n, y);
      }
    }
    if (sums) {
      const bool again = (touched >> t) & 1;
      touched |= 1ull << t;
      auto put = [&](const Piece (&v)[NP], float* to_row) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          Piece sum = v[i];
          if constexpr (LANES == 64) {
            // the waves' sums meet in LDS, in their order
            __syncthreads();
            if (which) {
#pragma unroll
              for (int j = 0; j < 8; ++j) staged[((which - 1) * 8 + j) * 64 + lane] = sum.v[j];
            }
            __syncthreads();
            if (which) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum.v[j] = (sum.v[j] + staged[j * 64 + lane]) + (staged[(8 + j) * 64 + lane] + staged[(16 + j) * 64 + lane]);
          }
          const int n = (i * LANES + lane) * 8;
          if (n >= p.width) continue;
          if (again) {
            const Piece before = load_piece_f32((const char*)(to_row + n));
#pragma unroll
            for (int j = 0; j < 8; ++j) sum.v[j] += before.v[j];
          }
          store_row_piece<true>((char*)to_row, n, sum);
        }
      };
      put(dw, slice + (int64_t)t * 2 * p.width);
      put(db, slice + ((int64_t)t * 2 + 1) * p.width);
    }
    at = to;
  }
  if (sums && threadIdx.x == 0) p.touched[blockIdx.x] = touched;
}

// dweight and dbias from the slices: a workgroup is 32 columns of one table row (8 lanes of 4), 32 slices at a time
__global__ __launch_bounds__(256) void norm_sums_kernel(NormParams p) {
  __shared__ f32x4 staged[256];
  const int t = blockIdx.y, half = blockIdx.z;
  float* out = half ? p.dbias : p.dweight;
  if (!out) return;
  const int col = blockIdx.x * 32 + (threadIdx.x & 7) * 4;
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  if (col < p.width) {
    const float* at = p.part + ((int64_t)t * 2 + half) * p.width + col;
    for (int g = threadIdx.x >> 3; g < p.groups; g += 32)
      if ((p.touched[g] >> t) & 1) sum += *(const f32x4*)(at + (int64_t)g * slice_floats(p.tables, p.width));
  }
  staged[threadIdx.x] = sum;
  for (int over = 128; over >= 8; over /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < over) staged[threadIdx.x] += staged[threadIdx.x + over];
  }
  if (threadIdx.x < 8 && col < p.width) *(f32x4*)(out + (int64_t)t * p.width + col) = staged[threadIdx.x];
}

// f(type of the rows, of the tables, lanes a row, pieces a lane)
template <class F>
static void with_form(bool f32, bool tb16, int width, F&& f) {
  auto by_width = [&](auto rows32, auto tables16) {
    if (width <= 512) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (width <= 1024) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (width <= 2048) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (width <= 4096) f(rows32, tables16, std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (width <= 8192) f(rows32, tables16, std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else f(rows32, tables16, std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  };
  if (f32) tb16 ? by_width(std::true_type{}, std::true_type{}) : by_width(std::true_type{}, std::false_type{});
  else tb16 ? by_width(std::false_type{}, std::true_type{}) : by_width(std::false_type{}, std::false_type{});
}

hipError_t launch_norm(const NormParams& p, bool f32, bool tables_bf16, hipStream_t s) {
  with_form(f32, tables_bf16, p.width, [&](auto a, auto b, auto lanes, auto np) {
    constexpr int kRows = kNormThreads / decltype(lanes)::value;
    norm_kernel<decltype(a)::value, decltype(b)::value, decltype(lanes)::value, decltype(np)::value><<<(p.rows + kRows - 1) / kRows, kNormThreads, 0, s>>>(p);
  });
  return hipGetLastError();
}

// A workgroup for 16 rows while there are few, up to 1,024 of them; with many tables fewer, so that the slices stay small.
int norm_groups(int rows, int tables) {
  const int by_rows = (rows + 15) / 16, most = 8192 / tables < 1024 ? 8192 / tables : 1024;
  return by_rows < most ? by_rows : most;
}

static size_t touched_bytes(int groups) { return ((size_t)groups * 8 + 255) / 256 * 256; }

size_t norm_scratch_bytes(int rows, int width, int tables) {
  const int groups = norm_groups(rows, tables);
  return touched_bytes(groups) + ((size_t)groups * slice_floats(tables, width) * sizeof(float) + 255) / 256 * 256;
}

hipError_t launch_norm_backward(NormParams p, bool f32, bool tables_bf16, char* workspace, hipStream_t s) {
  const bool sums = p.dweight || p.dbias;
  p.groups = norm_groups(p.rows, p.tables);
  p.touched = sums ? (uint64_t*)workspace : nullptr;
  p.part = sums ? (float*)(workspace + touched_bytes(p.groups)) : nullptr;
  with_form(f32, tables_bf16, p.width, [&](auto a, auto b, auto lanes, auto np) {
    norm_backward_kernel<decltype(a)::value, decltype(b)::value, decltype(lanes)::value, decltype(np)::value><<<p.groups, kNormThreads, 0, s>>>(p);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !sums) return e;
  norm_sums_kernel<<<dim3((p.width + 31) / 32, p.tables, 2), 256, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace pkh3
