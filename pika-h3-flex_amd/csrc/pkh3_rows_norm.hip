// Layer norm with tables (include/pkh3_rows.h), forward and backward.
//
//   forward    y = xh w[r] + b[r], xh = (x - mean) rstd
//   backward   g = dy w[r]:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw[r] = sum of dy xh, db[r] = sum of dy over the rows of table row r
//
// A row lies in the registers of the lanes that share it (a wave or a workgroup), 8 elements a piece, and the next row is on its way while one is worked on, so memory is
// read once and the variance is taken about the mean.  The backward pass forms the statistics again from the row, which it needs anyway, instead of keeping them.  Both
// are bound by memory: 48,360 rows of 2,048 in bfloat16 take 84 us forward (4.7 TB/s; a copy of as many bytes takes 75) and 152 us backward
// (3.8 TB/s; 132 without sums for the tables), 15,342 rows of 1,536 in float32 39 us (4.8 TB/s) and 62 us (4.5 TB/s; 55 without sums).  15,342 rows of 2,048 in bfloat16 take 27 and 57 us (3.3 TB/s
// backward, 49 without sums): two workgroups a CU, whose registers hold two rows and the next two, and the second launch.
//
// Sums for the tables: every workgroup takes one run of rows and keeps the sums of the table row that it is at in registers (its rows come
// in runs of one table row, so they rarely change); when the table row changes, and at the end, the workgroup's lanes add up in LDS and the sums go to the
// workgroup's own slice of the workspace.  A second launch adds the slices up in their order: no atomics, the same bits every time.  What a change costs: 48,360 rows of 2,048
// that take three table rows in three runs 163 us, in runs of 64 rows 171, of 8 252, at random 820, and with another table row at every row 1,070 (one of a workgroup's
// waves has a row at a time then).  Forward: 85, 86, 91, 97 and 103 us.
#include "pkh3_rows.h"

namespace pkh3 {

constexpr int kNormThreads = 256;

// COUNT values summed over the LANES lanes that share a row (lds: COUNT floats a wave)
template <int LANES, int COUNT>
__device__ __forceinline__ void row_sums(float (&x)[COUNT], float* lds) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) x[i] = wave_sum(x[i]);
  if constexpr (LANES > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();                                  // (what the sums before these were read from)
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) lds[wave * COUNT + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      x[i] = lds[i];
      for (int w = 1; w < LANES / 64; ++w) x[i] += lds[w * COUNT + i];
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store_row_piece(char* row, int n, const Piece& p) {
  if constexpr (F32) store_piece_f32(row + (int64_t)n * 4, p);
  else store_piece(row + (int64_t)n * 2, p);
}

// A row of NP pieces a lane as it lies in memory (zeros past its end): on its way while the row before it is worked on.
template <bool F32, int LANES, int NP>
struct Raw {
  i32x4 v[NP][F32 ? 2 : 1];
  __device__ __forceinline__ void load(const char* row, int lane, int width) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int n = (i * LANES + lane) * 8;
#pragma unroll
      for (int h = 0; h < (F32 ? 2 : 1); ++h) {
        v[i][h] = i32x4{0, 0, 0, 0};
        if (n < width) v[i][h] = *(const i32x4*)(row + (int64_t)n * (F32 ? 4 : 2) + h * 16);
      }
    }
  }
  __device__ __forceinline__ Piece piece(int i) const {
    Piece p;
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) p.v[j] = __int_as_float(v[i][j >> 2][j & 3]);
    } else {
      const bf16x8 raw = __builtin_bit_cast(bf16x8, v[i][0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) p.v[j] = (float)raw[j];
    }
    return p;
  }
};

// The row with its mean taken off, and 1 / sqrt(variance + eps).
template <bool F32, int LANES, int NP>
__device__ __forceinline__ float centre(Piece (&x)[NP], const Raw<F32, LANES, NP>& raw, int lane, int width, float eps, float* lds) {
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    x[i] = raw.piece(i);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0] += x[i].v[j];
  }
  row_sums<LANES>(s, lds);
  const float mean = s[0] / (float)width;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bool live = i < NP / 2 || (i * LANES + lane) * 8 < width;   // (wider than the next smaller form, so the first half is full)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[i].v[j] = live ? x[i].v[j] - mean : 0.f;
      s[0] += x[i].v[j] * x[i].v[j];
    }
  }
  row_sums<LANES>(s, lds);
  return 1.0f / sqrtf(s[0] / (float)width + eps);
}

__device__ __forceinline__ int table_of(const NormParams& p, int row) { return p.row_index ? min(max(p.row_index[row], 0), p.tables - 1) : 0; }

template <bool TB16, int LANES, int NP>
__device__ __forceinline__ void load_table_row(Piece (&to)[NP], const char* table, int t, int lane, int width, float without) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int n = (i * LANES + lane) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) to[i].v[j] = without;
    if (table && n < width) to[i] = load_table(table, (int64_t)t * width + n, TB16);
  }
}

// rows of a workgroup: one run, dealt to its waves (or taken by all of them) in turn
struct Run {
  int first, end;
};
__device__ __forceinline__ Run run_of_rows(const NormParams& p) {
  return {(int)((int64_t)p.rows * blockIdx.x / p.groups), (int)((int64_t)p.rows * (blockIdx.x + 1) / p.groups)};
}

template <bool F32, bool TB16, int LANES, int NP>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(NormParams p) {
  constexpr int kRows = kNormThreads / LANES;         // rows at a time
  __shared__ float lds[4];
  const int lane = threadIdx.x % LANES, which = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  const Run run = run_of_rows(p);
  int row = run.first + which, held = -1;
  if (row >= run.end) return;                         // (whole waves, and with LANES == 256 all of them)
  Raw<F32, LANES, NP> raw;
  raw.load(p.x + row * p.x_stride, lane, p.width);
  Piece w[NP], b[NP];
#pragma unroll 1
  for (; row < run.end; row += kRows) {
    const int t = __builtin_amdgcn_readfirstlane(table_of(p, row));
    if (t != held) {
      load_table_row<TB16, LANES>(w, p.weight, t, lane, p.width, 1.f);
      load_table_row<TB16, LANES>(b, p.bias, t, lane, p.width, 0.f);
      held = t;
    }
    const Raw<F32, LANES, NP> now = raw;
    raw.load(p.x + min(row + kRows, run.end - 1) * p.x_stride, lane, p.width);
    Piece x[NP];
    const float rstd = centre<F32, LANES, NP>(x, now, lane, p.width, p.eps, lds);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int n = (i * LANES + lane) * 8;
      if (n >= p.width) break;
      Piece y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y.v[j] = x[i].v[j] * rstd * w[i].v[j] + b[i].v[j];
      store_row_piece<F32>(p.out + row * p.out_stride, n, y);
    }
  }
}

// slice of a workgroup: [table][weights' sums, biases' sums][width]
__host__ __device__ inline int64_t slice_floats(int tables, int width) { return (int64_t)tables * 2 * width; }

template <bool F32, bool TB16, int LANES, int NP>
__global__ __launch_bounds__(LANES > kNormThreads ? LANES : kNormThreads) void norm_backward_kernel(NormParams p) {
  constexpr int kRows = LANES > kNormThreads ? 1 : kNormThreads / LANES;   // rows at a time
  __shared__ float lds[2 * 16];
  __shared__ __attribute__((aligned(16))) float staged[LANES == 64 ? 3 * 64 * 8 : 1];
  const int lane = threadIdx.x % LANES, which = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  const auto [first, end] = run_of_rows(p);
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
    load_table_row<TB16, LANES>(w, p.weight, t, lane, p.width, 1.f);
#pragma unroll
    for (int i = 0; i < NP; ++i) dw[i] = Piece{}, db[i] = Piece{};
    // The next row on its way where the registers allow it: 48,360 rows of 2,048 in bfloat16 take 157 us so and 196 without. Four pieces of float32
    // a lane lose more by the registers (15,342 rows of 1,536: 72 us so, 55 without), and where a row has several waves others fill the gap
    // (48,360 rows of 4,096: 294 us so, 261 without; 15,342 of 8,192: 203 and 172).
    constexpr bool kAhead = LANES == 64 && (NP < 4 || !F32);
    Raw<F32, LANES, NP> raw_x, raw_dy;
    auto ask = [&](int row) {
      raw_x.load(p.x + row * p.x_stride, lane, p.width);
      raw_dy.load(p.dy + row * p.dy_stride, lane, p.width);
    };
    if (kAhead) ask(min(at + which, to - 1));
#pragma unroll 1
    for (int row = at + which; row < to; row += kRows) {
      if (!kAhead) ask(row);
      const Raw<F32, LANES, NP> x_now = raw_x, dy_now = raw_dy;
      if (kAhead) ask(min(row + kRows, to - 1));
      Piece x[NP], d[NP];
      const float rstd = centre<F32, LANES, NP>(x, x_now, lane, p.width, p.eps, lds);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        d[i] = dy_now.piece(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = x[i].v[j] * rstd, g = d[i].v[j] * w[i].v[j];
          x[i].v[j] = xh;
          dw[i].v[j] += d[i].v[j] * xh;
          db[i].v[j] += d[i].v[j];
          d[i].v[j] = g;
          s[0] += g;
          s[1] += g * xh;
        }
      }
      row_sums<LANES>(s, lds);
      const float mean_g = s[0] / (float)p.width, mean_gx = s[1] / (float)p.width;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int n = (i * LANES + lane) * 8;
        if (n >= p.width) break;
        Piece y;
#pragma unroll
        for (int j = 0; j < 8; ++j) y.v[j] = rstd * (d[i].v[j] - mean_g - x[i].v[j] * mean_gx);
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

// dweight and dbias from the slices: a workgroup is 32 columns of one table row (8 lanes of 4), 128 slices at a time, four times that asked for together
constexpr int kSumThreads = 1024;

__global__ __launch_bounds__(kSumThreads) void norm_sums_kernel(NormParams p) {
  __shared__ f32x4 staged[kSumThreads];
  const int t = blockIdx.y, half = blockIdx.z;
  float* out = half ? p.dbias : p.dweight;
  if (!out) return;
  const int col = blockIdx.x * 32 + (threadIdx.x & 7) * 4;
  const int64_t slice = slice_floats(p.tables, p.width);
  const float* at = p.part + ((int64_t)t * 2 + half) * p.width + min(col, p.width - 4);
  constexpr int kAt = kSumThreads / 8;
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  for (int g = threadIdx.x >> 3; g < p.groups; g += 4 * kAt) {
    f32x4 v[4];
    bool there[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = min(g + i * kAt, p.groups - 1);
      there[i] = g + i * kAt < p.groups && ((p.touched[from] >> t) & 1);
      v[i] = *(const f32x4*)(at + from * slice);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += there[i] ? v[i][j] : 0.f;   // (what nobody wrote may be anything)
  }
  staged[threadIdx.x] = sum;
  for (int over = kSumThreads / 2; over >= 8; over /= 2) {
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

// Workgroups of the forward pass: as many as there are rows for, up to six a CU, which then have several rows a wave, the next one on its way.
hipError_t launch_norm(NormParams p, bool f32, bool tables_bf16, hipStream_t s) {
  with_form(f32, tables_bf16, p.width, [&](auto a, auto b, auto lanes, auto np) {
    constexpr int kRows = kNormThreads / decltype(lanes)::value;
    p.groups = (p.rows + kRows - 1) / kRows < 1536 ? (p.rows + kRows - 1) / kRows : 1536;
    norm_kernel<decltype(a)::value, decltype(b)::value, decltype(lanes)::value, decltype(np)::value><<<p.groups, kNormThreads, 0, s>>>(p);
  });
  return hipGetLastError();
}

// A workgroup for 8 rows up to 512 of them, for 32 up to 1,024 (their slices are then a sixth of what the rows move); with many tables (up to 64 where there are sums) fewer, so that the slices stay small.
int norm_groups(int rows, int tables) {
  const int by_8 = (rows + 7) / 8 < 512 ? (rows + 7) / 8 : 512, by_32 = (rows + 31) / 32 < 1024 ? (rows + 31) / 32 : 1024;
  const int groups = by_8 > by_32 ? by_8 : by_32, most = 8192 / tables;
  return groups < most ? groups : most;
}

static size_t touched_bytes(int groups) { return ((size_t)groups * 8 + 255) / 256 * 256; }

size_t norm_scratch_bytes(int rows, int width, int tables) {
  const int groups = norm_groups(rows, tables);
  return touched_bytes(groups) + ((size_t)groups * slice_floats(tables, width) * sizeof(float) + 255) / 256 * 256;
}

// f(type of the rows, of the tables, lanes a row, pieces a lane) for the backward pass, which holds five times as much of a row a lane
template <class F>
static void with_backward_form(bool f32, bool tb16, int width, F&& f) {
  auto by_width = [&](auto rows32, auto tables16) {
    if (width <= 512) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (width <= 1024) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (width <= 2048) f(rows32, tables16, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (width <= 4096) f(rows32, tables16, std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (width <= 8192) f(rows32, tables16, std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else f(rows32, tables16, std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
  };
  if (f32) tb16 ? by_width(std::true_type{}, std::true_type{}) : by_width(std::true_type{}, std::false_type{});
  else tb16 ? by_width(std::false_type{}, std::true_type{}) : by_width(std::false_type{}, std::false_type{});
}

hipError_t launch_norm_backward(NormParams p, bool f32, bool tables_bf16, char* workspace, hipStream_t s) {
  const bool sums = p.dweight || p.dbias;
  p.groups = norm_groups(p.rows, sums ? p.tables : 1);
  p.touched = sums ? (uint64_t*)workspace : nullptr;
  p.part = sums ? (float*)(workspace + touched_bytes(p.groups)) : nullptr;
  with_backward_form(f32, tables_bf16, p.width, [&](auto a, auto b, auto lanes, auto np) {
    constexpr int kThreads = decltype(lanes)::value > kNormThreads ? decltype(lanes)::value : kNormThreads;
    norm_backward_kernel<decltype(a)::value, decltype(b)::value, decltype(lanes)::value, decltype(np)::value><<<p.groups, kThreads, 0, s>>>(p);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !sums) return e;
  norm_sums_kernel<<<dim3((p.width + 31) / 32, p.tables, 2), kSumThreads, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace pkh3
