/*
 * pkh3_rows.h -- the feed-forward half of a transformer block on plain row-major matrices, forward and backward:
 * layer norm with its tables, and matrix products that finish their own results.
 *
 * The reference's blocks are those of the un-vendored transformer that src/pika_h3/core/loader.py:11-18 loads; of their
 * feed-forward half it names the two linear layers (`ff.net.0.proj`, `ff.net.2`, src/pika_h3/core/loader.py:9), and its patch
 * shows the modulated norm in front (patches/0001-h3-adaln-fp32.patch:34-40).
 *
 * Conventions are those of pkh3_attn.h (errors, streams, caller-owned device memory, no allocation, no synchronisation; calls may be
 * captured).  Matrices are row-major with unit column stride; row strides and widths are multiples of 8 elements, bases 16-byte
 * aligned.  What a call writes must not overlap what it reads, but for `out` of a product, which may be exactly its `residual`, and for `dx` of
 * a norm's backward pass, which may be exactly `dy` or `x`; and the `out` of a norm, which may be exactly its `x`.
 */
#ifndef PKH3_ROWS_H
#define PKH3_ROWS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm ----
 * y = (x - mean(x)) / sqrt(var(x) + eps) * weight[r] + bias[r] for every row, r its table row: row_index[row], brought into [0, tables),
 * or 0 without row_index.  Statistics are float32, the variance about the mean. */

#define PKH3_LAYER_NORM_F32 1u        /* x, out, dy and dx are float32, else bfloat16 */
#define PKH3_LAYER_NORM_TABLES_BF16 2u /* weight and bias are bfloat16, else float32 */
#define PKH3_LAYER_NORM_MAX_WIDTH 16384
#define PKH3_LAYER_NORM_MAX_TABLES 64 /* with dweight or dbias; else 65,535 */

typedef struct pkh3_norm_args {
  const void* x;                /* [rows, width] */
  const void* weight;           /* [tables, width] contiguous, or NULL: 1 */
  const void* bias;             /* the same, or NULL: 0 (not read by the backward pass) */
  const int32_t* row_index;     /* [rows], or NULL */
  void* out;                    /* forward: [rows, width] */
  const void* dy;               /* backward: gradient of out */
  void* dx;                     /* backward: gradient of x */
  float* dweight;               /* backward: [tables, width] float32, or NULL */
  float* dbias;                 /* backward: the same, or NULL */
  void* workspace;              /* backward with dweight or dbias: 256-byte aligned, pkh3_norm_workspace_bytes() */
  uint64_t workspace_bytes;
  int64_t x_stride, out_stride, dy_stride, dx_stride;
  int32_t rows, width, tables;
  float eps;
  uint32_t flags;
} pkh3_norm_args;

int pkh3_layer_norm(const pkh3_norm_args* args, void* stream);
/* dx = (g - mean(g) - xh * mean(g * xh)) / sqrt(var + eps), g = dy * weight[r], xh the normalised row; dweight[r] and dbias[r] are the sums of
 * dy * xh and of dy over the rows of table row r (zeros where there are none), added up in an order that depends on the sizes and the row index alone.  Meant for rows that
 * take the same table row for a while: with another one at every row the call takes six times as long. */
int pkh3_layer_norm_backward(const pkh3_norm_args* args, void* stream);
size_t pkh3_norm_workspace_bytes(const pkh3_norm_args* args);

/* ---- matrix products ----
 * out[m, n] = finish( sum over k of A(m, k) * B(n, k) ), bfloat16 in and out, sums in float32.  A is stored [M, K], or [K, M] with
 * PKH3_PRODUCT_A_ACROSS; B [N, K], or [K, N] with PKH3_PRODUCT_B_ACROSS.  So a linear layer's y = x W^T is (x, W), its input's gradient
 * dy W is (dy, W across), its weight's gradient dy^T x is (dy across, x across).  K alone may be any number: rows of a matrix that is stored
 * across need not come in eights.
 *
 *   plain    v = sum + bias[n]; pre[m, n] = v in float32, if given; out = residual[m, n] + gate[index[m], n] * act(v), as far as given
 *   GATED    B has 2 N rows, bias 2 N entries: a = row n, b = row N + n.  pre [M, 2 N] = (a | b), if given; out = a * act(b); no gate or residual
 *   GRAD     sum is the gradient of act(pre) and out [M, N] that of pre: out = sum * act'(pre[m, n])
 *   GRAD and GATED   pre [M, 2 N] = (a | b), out [M, 2 N]: out[m, n] = sum * act(b), out[m, N + n] = sum * a * act'(b)
 *
 * Offered are A and B along (plain, GATED), A along and B across (plain without anything besides, GRAD, GRAD and GATED), and both
 * across (plain without anything besides); of others PKH3_EUNSUPPORTED.  With GRAD, `sums`, if given, gets the sums of out's columns before they were rounded (bfloat16, N or 2 N entries). */

/* Activations.  Of an infinite sum they are what the formulas give: +inf of +inf, NaN (infinity times zero) of -inf, and slopes of NaN. */
enum {
  PKH3_ACT_NONE = 0,
  PKH3_ACT_SILU = 1,            /* v / (1 + exp(-v)) */
  PKH3_ACT_GELU = 2,            /* v * (1 + erf(v / sqrt(2))) / 2 */
  PKH3_ACT_GELU_TANH = 3        /* v * (1 + tanh(sqrt(2 / pi) * (v + 0.044715 v^3))) / 2 */
};

#define PKH3_PRODUCT_A_ACROSS 1u
#define PKH3_PRODUCT_B_ACROSS 2u
#define PKH3_PRODUCT_GATED 4u
#define PKH3_PRODUCT_GRAD 8u
#define PKH3_PRODUCT_BIAS_BF16 16u   /* bias is bfloat16, else float32 */

typedef struct pkh3_product_args {
  const void* a;
  const void* b;
  const void* bias;
  const void* gate;             /* bfloat16 [gate_rows, N] */
  const int32_t* gate_index;    /* [M], brought into [0, gate_rows); NULL: 0 */
  const void* residual;         /* bfloat16 [M, N] */
  void* pre;                    /* float32 [M, N or 2 N]: written, with GRAD read */
  void* out;
  void* sums;
  void* workspace;              /* 256-byte aligned, pkh3_product_workspace_bytes(); NULL where that is 0 */
  uint64_t workspace_bytes;
  int64_t a_stride, b_stride, gate_stride, residual_stride, pre_stride, out_stride;
  int32_t M, N, K, gate_rows;
  int32_t activation;
  uint32_t flags;
} pkh3_product_args;

int pkh3_product(const pkh3_product_args* args, void* stream);
size_t pkh3_product_workspace_bytes(const pkh3_product_args* args);

/* out = a * act'(pre) for the gradient `a` [M, N] of act(pre), with `sums` as above: what GRAD does, without a product in front.  Of the arguments a, pre (not
 * read without an activation), out (may be NULL without one, or exactly `a`), sums, workspace, strides, M, N and activation are used; the workspace is that of
 * pkh3_activation_grad_workspace_bytes(). */
int pkh3_activation_grad(const pkh3_product_args* args, void* stream);
size_t pkh3_activation_grad_workspace_bytes(const pkh3_product_args* args);

#ifdef __cplusplus
}
#endif
#endif
