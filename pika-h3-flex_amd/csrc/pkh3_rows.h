// Parameters of the kernels behind include/pkh3_rows.h, and how a product finishes its results.
#pragma once
#include "pkh3_common.h"
#include "pkh3_rows_index.h"

namespace pkh3 {

// ---- layer norm ----

struct NormParams {
  const char *x, *dy;
  char *out, *dx;
  const char *weight, *bias;     // [tables][width], or null
  const int* row_index;          // or null
  float* part;                   // backward: partial sums of the workgroups (norm_slices)
  uint64_t* touched;             // ... and which tables each of them holds
  float *dweight, *dbias;
  int64_t x_stride, out_stride, dy_stride, dx_stride;   // bytes
  int rows, width, tables, groups;
  float eps;
};

int norm_groups(int rows, int tables);              // workgroups of the backward pass, each with sums of its own
size_t norm_scratch_bytes(int rows, int width, int tables);
hipError_t launch_norm(NormParams p, bool f32, bool tables_bf16, hipStream_t s);
hipError_t launch_norm_backward(NormParams p, bool f32, bool tables_bf16, char* workspace, hipStream_t s);

// ---- products ----

struct ProductParams {
  const char *a, *b;             // [M, K] and [N, K], or across
  int64_t a_stride, b_stride;    // bytes
  const char* bias;
  const char* gate;
  const int* gate_index;
  const char* residual;
  char* pre;                     // float32
  char* out;
  float* sums;                   // partial sums of out's columns, [rows of partial sums][columns], or null
  float* part;                   // parts of the tiles that are cut: [unit][rows of a tile][columns of a tile]
  int64_t gate_stride, residual_stride, pre_stride, out_stride;   // bytes
  int M, N, K, gate_rows;
  int act, bias_bf16;
};

hipError_t launch_product(ProductParams p, const ProductPlan& plan, bool a_across, bool b_across, int mode, void* sums, char* workspace, hipStream_t s);
hipError_t launch_tiles_8(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s);
hipError_t launch_tiles_4(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s);
hipError_t launch_tiles_4x4(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s);
hipError_t launch_tiles_2x4(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s);
hipError_t launch_tiles_3x4(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s);

hipError_t launch_thin(const ProductParams& p, int mode, hipStream_t s);

int activation_grad_rows(int M);                    // rows of partial column sums of an activation's gradient
hipError_t launch_activation_grad(ProductParams p, void* sums, char* workspace, hipStream_t s);

// ---- copies ----

// The two halves of a direct-to-LDS copy: wave-uniform target and base address, per-lane byte offset.
template <int OFFSET>
__device__ __forceinline__ void copy_to(unsigned lds_addr) { asm volatile("s_add_u32 m0, %0, %1" ::"s"(lds_addr), "n"(OFFSET) : "m0", "scc"); }
__device__ __forceinline__ void copy_from(const char* g, unsigned lane_off) {
  asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(lane_off), "s"(g) : "memory");
}
// operand of s_waitcnt: at most `vm` copies and `lgkm` LDS reads still on their way
constexpr int wait_for(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }

// ---- activations ----

// exp(x); one instruction's error of 2^x (about 1 ulp) and the rounding of x log2(e)
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-x)); }

// The normal distribution's tail beyond |v|: erfc(z) / 2, z = |v| / sqrt 2, with erfc(z) = t exp(-z^2 + p(t)), t = 1 / (1 + z / 2), the form in which W. H. Press et al.,
// "Numerical Recipes", give the error function.  p is a polynomial of lower degree, fitted here to log(erfc(z) / t) + z^2 at Chebyshev points of t in [1/8, 1] (z up to 14),
// to 8e-7 of the value.  In float32 the roundings of the exponent come on top, which grow with it: 1.2e-6 of the value up to |v| of 2, 2.5e-6 up to 6, 1.1e-5 up to 13.  The
// result's own rounding to bfloat16 is 350 times that.
// (Its coefficients are those times log2(e), with -1 for the half in the last one: an activation's instructions are what a tile's results take besides memory, 256 of
// them a lane at 4 cycles each and 16 for those of exp2 and the reciprocal.)
__device__ __forceinline__ float normal_tail(float v) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.35355339059327376f * fabsf(v));
  float p = -0.274807450f;
  p = p * t + 1.10064317f;
  p = p * t - 1.47251475f;
  p = p * t + 0.530742107f;
  p = p * t - 0.0708096726f;
  p = p * t + 0.572366047f;
  p = p * t + 1.44003868f;
  p = p * t - 2.82565923f;
  return t * __builtin_amdgcn_exp2f(p - 0.5f * kLog2e * (v * v));
}

constexpr float kTanhScale = 0.79788456080286536f;   // sqrt(2 / pi)
constexpr float kTanhCube = 0.044715f;
// sigmoid(2 u), u = sqrt(2 / pi) (v + 0.044715 v^3)
__device__ __forceinline__ float tanh_gate(float v) {
  constexpr float kOnce = -2.0f * kTanhScale * kLog2e, kCubed = kOnce * kTanhCube;
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * (kOnce + kCubed * (v * v))));
}

// act(v): 0 none, 1 silu, 2 gelu, 3 gelu through tanh (as v sigmoid(2 u), which keeps its small tail exact).  Of infinities what the formulas give: +inf for +inf, and for
// -inf their infinity times zero, NaN.
template <int ACT>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == 1) return v * sigmoid_of(v);
  if constexpr (ACT == 2) return fmaxf(v, 0.f) - fabsf(fminf(v, 1e30f)) * normal_tail(v);   // (+inf: not infinity times its tail of 0)
  if constexpr (ACT == 3) return v * tanh_gate(v);
  return v;
}
// act(v) and act'(v)
template <int ACT>
__device__ __forceinline__ void act_and_slope(float v, float& value, float& slope) {
  if constexpr (ACT == 1) {
    const float q = sigmoid_of(v);
    value = v * q;
    slope = q + value * (1.0f - q);
  } else if constexpr (ACT == 2) {
    const float tail = normal_tail(v), q = v < 0.f ? tail : 1.0f - tail;
    value = v * q;
    slope = q + v * 0.39894228040143268f * exp_of(-0.5f * v * v);
  } else if constexpr (ACT == 3) {
    const float q = tanh_gate(v);
    value = v * q;
    slope = q + value * (1.0f - q) * (2.0f * kTanhScale) * (1.0f + 3.0f * kTanhCube * fminf(v * v, 1e30f));   // (no 0 times infinity far out)
  } else {
    value = v;
    slope = 1.0f;
  }
}

// ---- eight results of a row: columns n .. n + 7 of row m ----

struct Piece {
  float v[8];
};
__device__ __forceinline__ Piece load_piece(const char* at) {
  const bf16x8 raw = *(const bf16x8*)at;
  Piece p;
#pragma unroll
  for (int j = 0; j < 8; ++j) p.v[j] = (float)raw[j];
  return p;
}
__device__ __forceinline__ void store_piece(char* at, const Piece& p) {
  bf16x8 raw;
#pragma unroll
  for (int j = 0; j < 8; ++j) raw[j] = (__bf16)p.v[j];
  *(bf16x8*)at = raw;
}
__device__ __forceinline__ Piece load_piece_f32(const char* at) {
  const f32x4 lo = *(const f32x4*)at, hi = *(const f32x4*)(at + 16);
  return Piece{{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
}
__device__ __forceinline__ void store_piece_f32(char* at, const Piece& p) {
  *(f32x4*)at = f32x4{p.v[0], p.v[1], p.v[2], p.v[3]};
  *(f32x4*)(at + 16) = f32x4{p.v[4], p.v[5], p.v[6], p.v[7]};
}
__device__ __forceinline__ Piece load_table(const char* table, int64_t at, bool bf16) {
  return bf16 ? load_piece(table + at * 2) : load_piece_f32(table + at * 4);
}

// The bias of columns n .. n + 7, and of the gates' (mode kGated)
struct Bias {
  Piece a, b;
};
template <int MODE>
__device__ __forceinline__ Bias load_bias(const ProductParams& p, int n) {
  Bias bias{};
  if (MODE <= kGated && p.bias) {
    bias.a = load_table(p.bias, n, p.bias_bf16);
    if (MODE == kGated) bias.b = load_table(p.bias, p.N + n, p.bias_bf16);
  }
  return bias;
}

// Two blocks of 16 columns a lane holds four of each (4*g .. +3): after the exchange of rows of 16 lanes it holds eight columns beside each other, from
// eight_of(g) of the 32 on.
__device__ __forceinline__ int eight_of(int g) { return (g & 1) * 16 + (g >> 1) * 8; }
__device__ __forceinline__ Piece eight_columns(const f32x4& first, const f32x4& second) {
  Piece p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(first[i]), __float_as_uint(second[i]), false, false);
    p.v[i] = __uint_as_float(r[0]);
    p.v[4 + i] = __uint_as_float(r[1]);
  }
  return p;
}

// ---- from sums to results (see pkh3_product in the header) ----
// What a call has besides is a matter of constants, not of branches: behind a branch around a load the compiler waits for all accesses before it, stores
// among them, whether the load was made or not (a tile's results took 25,000 cycles that way).  Accesses past the last row or column are dropped by
// the hardware's range check for the same reason.

constexpr int kWithResidual = 1, kWithGate = 2;

// f(activation, what is there besides: as constants).  SUMS: a gradient's product, whose sums are its results.
template <int MODE, bool SUMS, class F>
__device__ __forceinline__ void with_form(const ProductParams& p, F&& f) {
  if constexpr (SUMS) return f(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
  auto by_act = [&](auto besides) {
    if (p.act == 0) f(std::integral_constant<int, 0>{}, besides);
    else if (p.act == 1) f(std::integral_constant<int, 1>{}, besides);
    else if (p.act == 2) f(std::integral_constant<int, 2>{}, besides);
    else f(std::integral_constant<int, 3>{}, besides);
  };
  if constexpr (MODE == kPlain) {
    if (p.gate && p.residual) by_act(std::integral_constant<int, kWithGate | kWithResidual>{});
    else if (p.gate) by_act(std::integral_constant<int, kWithGate>{});
    else if (p.residual) by_act(std::integral_constant<int, kWithResidual>{});
    else by_act(std::integral_constant<int, 0>{});
  } else {
    by_act(std::integral_constant<int, 0>{});
  }
}

// Rows of a matrix from one row on: up to 128 of them, whose offsets are 32 bits (strides up to 2^24 bytes).
constexpr unsigned kNowhere = 0x80000000u;          // an offset that the range check drops
struct RowsOf {
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned stride;
  __device__ __forceinline__ RowsOf(char* base, int64_t row_stride, int first)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(base + first * row_stride, 0, (int)kNowhere, 0x00020000)), stride((unsigned)row_stride) {}
  __device__ __forceinline__ i32x4 load(unsigned at) const { return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0)); }
  __device__ __forceinline__ void store(unsigned at, i32x4 v) const {
    typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc, at, 0, 0);
  }
  __device__ __forceinline__ void store_bf16(unsigned at, const Piece& p) const {
    bf16x8 raw;
#pragma unroll
    for (int j = 0; j < 8; ++j) raw[j] = (__bf16)p.v[j];
    store(at, __builtin_bit_cast(i32x4, raw));
  }
  __device__ __forceinline__ void store_f32(unsigned at, const Piece& p) const {
    store(at, __builtin_bit_cast(i32x4, f32x4{p.v[0], p.v[1], p.v[2], p.v[3]}));
    store(at + 16, __builtin_bit_cast(i32x4, f32x4{p.v[4], p.v[5], p.v[6], p.v[7]}));
  }
  __device__ __forceinline__ Piece load_f32(unsigned at) const {
    const f32x4 lo = __builtin_bit_cast(f32x4, load(at)), hi = __builtin_bit_cast(f32x4, load(at + 16));
    return Piece{{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
  }
};

// The results' rows from one on; rows counted from there.
template <int MODE>
struct Results {
  const ProductParams& p;
  RowsOf out, pre, residual;
  int rows, first;
  __device__ __forceinline__ Results(const ProductParams& params, int first_row)
      : p(params), out(params.out, params.out_stride, first_row), pre(params.pre, params.pre_stride, first_row),
        residual((char*)params.residual, params.residual_stride, first_row), rows(params.M - first_row), first(first_row) {}

  // What else a piece's results need, asked for ahead of them: the gate and the residual, or the saved sums.
  struct Plain {
    i32x4 gate, residual;
  };
  struct Grad {
    Piece z;
  };
  struct GatedGrad {
    Piece a, b;
  };
  using Extra = std::conditional_t<MODE == kGatedGrad, GatedGrad, std::conditional_t<MODE == kGrad, Grad, Plain>>;
  __device__ __forceinline__ unsigned at(const RowsOf& m, int row, int n, int size) const {
    return row < rows && n < p.N ? (unsigned)row * m.stride + (unsigned)(n * size) : kNowhere;
  }
  // The row of the gate that a row takes.
  __device__ __forceinline__ int gate_row(int row) const {
    return p.gate_index ? min(max(p.gate_index[first + min(row, rows - 1)], 0), p.gate_rows - 1) : 0;
  }
  // gate_of: gate_row(row), where there is a gate
  template <int ACT, int BESIDES>
  __device__ __forceinline__ void fetch(int row, int n, int gate_of, Extra& e) const {
    if constexpr (MODE == kGrad) {
      if constexpr (ACT != 0) e.z = pre.load_f32(at(pre, row, n, 4));
    } else if constexpr (MODE == kGatedGrad) {
      const unsigned where = at(pre, row, n, 4);
      e.a = pre.load_f32(where);
      e.b = pre.load_f32(where == kNowhere ? where : where + (unsigned)p.N * 4);
    } else {
      if constexpr (BESIDES & kWithGate) {
        e.gate = *(const i32x4*)(p.gate + gate_of * p.gate_stride + (int64_t)min(n, p.N - 8) * 2);
      }
      if constexpr (BESIDES & kWithResidual) e.residual = residual.load(at(residual, row, n, 2));
    }
  }
  // a: the sums of columns n .. n + 7, b: of the gates'.  On return what out got, for the sums of columns.  Sums that are saved for the
  // backward pass stay in float32: rounded to bfloat16 they cost its gradients half as much again as their own rounding does.
  template <int ACT, int BESIDES>
  __device__ __forceinline__ void finish(int row, int n, Piece& a, Piece& b, const Bias& bias, const Extra& e) const {
    const unsigned to = at(out, row, n, 2);
    const unsigned to_b = to == kNowhere ? to : to + (unsigned)p.N * 2;
    if constexpr (MODE <= kGated) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a.v[j] += bias.a.v[j];
      if constexpr (MODE == kGated) {
#pragma unroll
        for (int j = 0; j < 8; ++j) b.v[j] += bias.b.v[j];
      }
      if (p.pre) {
        const unsigned keep = at(pre, row, n, 4);
        pre.store_f32(keep, a);
        if constexpr (MODE == kGated) pre.store_f32(keep == kNowhere ? keep : keep + (unsigned)p.N * 4, b);
      }
      if constexpr (MODE == kGated) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a.v[j] *= act_of<ACT>(b.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a.v[j] = act_of<ACT>(a.v[j]);
        if constexpr (BESIDES & kWithGate) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a.v[j] *= (float)__builtin_bit_cast(bf16x8, e.gate)[j];
        }
        if constexpr (BESIDES & kWithResidual) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a.v[j] += (float)__builtin_bit_cast(bf16x8, e.residual)[j];
        }
      }
      out.store_bf16(to, a);
    } else if constexpr (MODE == kGrad) {
      if constexpr (ACT != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float value, slope;
          act_and_slope<ACT>(e.z.v[j], value, slope);
          a.v[j] *= slope;
        }
      }
      out.store_bf16(to, a);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float value, slope;
        act_and_slope<ACT>(e.b.v[j], value, slope);
        b.v[j] = a.v[j] * e.a.v[j] * slope;
        a.v[j] *= value;
      }
      out.store_bf16(to, a);
      out.store_bf16(to_b, b);
    }
  }
};

}  // namespace pkh3
