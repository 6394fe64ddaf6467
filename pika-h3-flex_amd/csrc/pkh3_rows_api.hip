// C ABI of include/pkh3_rows.h: argument validation on the host, then the launches.
#include "../../include/pkh3_rows.h"
#include "../../include/pkh3_attn.h"

#include <stdarg.h>
#include <stdio.h>

#include "pkh3_internal.h"
#include "pkh3_rows.h"

using namespace pkh3;

namespace {

constexpr int kMostRows = 1 << 21, kMostStride = 1 << 22;   // rows, columns and contraction; elements between rows

int fail(int code, const char* fmt, ...) {
  char text[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return report_error(code, text);
}
int done(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(PKH3_EHIP, "%s: %s", what, hipGetErrorString(e));
  return report_error(PKH3_OK, "");
}

bool misaligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) != 0; }

// rows x cols elements of `size` bytes, `stride` elements from row to row
struct Matrix {
  const char* name;
  const void* at;
  int64_t stride;
  int rows, cols, size;
};

int check_matrix(const Matrix& m) {
  if (!m.at) return fail(PKH3_ENULL, "%s is NULL", m.name);
  if (misaligned(m.at, 16)) return fail(PKH3_EALIGN, "%s is not 16-byte aligned", m.name);
  if (m.stride % 8 || m.stride > kMostStride || (m.rows > 1 && m.stride < m.cols))
    return fail(PKH3_ESTRIDE, "%s: row stride %lld of %d columns (a multiple of 8, at most %d, rows apart from each other)", m.name, (long long)m.stride, m.cols, kMostStride);
  return PKH3_OK;
}

// Whether two matrices share a byte.  Of matrices with the same row pitch (column slices of one buffer among them) the columns are held against each other;
// of others the whole stretches.
bool overlap(const Matrix& a, const Matrix& b) {
  if (!a.at || !b.at || a.rows < 1 || b.rows < 1) return false;
  const int64_t pa = a.stride * a.size, pb = b.stride * b.size, wa = (int64_t)a.cols * a.size, wb = (int64_t)b.cols * b.size;
  const int64_t a0 = (int64_t)(uintptr_t)a.at, b0 = (int64_t)(uintptr_t)b.at;
  if (a0 + pa * (a.rows - 1) + wa <= b0 || b0 + pb * (b.rows - 1) + wb <= a0) return false;
  if (pa != pb || a.rows == 1 || b.rows == 1) return true;
  const int64_t d = ((b0 - a0) % pa + pa) % pa;
  return d < wa || d + wb > pa;
}
bool same(const Matrix& a, const Matrix& b) { return a.at == b.at && (a.stride == b.stride || a.rows == 1) && a.rows == b.rows && a.cols == b.cols && a.size == b.size; }

int apart(const Matrix& out, const Matrix& in) {
  return overlap(out, in) ? fail(PKH3_EARG, "%s overlaps %s", out.name, in.name) : PKH3_OK;
}

int check_workspace(const void* at, uint64_t have, size_t need) {
  if (!need) return PKH3_OK;
  if (!at) return fail(PKH3_EWORKSPACE, "workspace is NULL");
  if (misaligned(at, 256)) return fail(PKH3_EWORKSPACE, "workspace is not 256-byte aligned");
  if (have < need) return fail(PKH3_EWORKSPACE, "workspace too small: %llu < %zu bytes", (unsigned long long)have, need);
  return PKH3_OK;
}

// ---- layer norm ----

// sums: the tables' gradients are asked for
int check_norm_sizes(const pkh3_norm_args* a, bool sums) {
  if (!a) return fail(PKH3_ENULL, "args is NULL");
  if (a->flags & ~(PKH3_LAYER_NORM_F32 | PKH3_LAYER_NORM_TABLES_BF16)) return fail(PKH3_EARG, "unknown flag bits 0x%x", a->flags);
  if (a->rows < 0 || a->rows > kMostRows) return fail(PKH3_ESHAPE, "rows must be in [0, 2^21], got %d", a->rows);
  if (a->width < 8 || a->width > PKH3_LAYER_NORM_MAX_WIDTH || a->width % 8) return fail(PKH3_ESHAPE, "width must be a multiple of 8 in [8, %d], got %d", PKH3_LAYER_NORM_MAX_WIDTH, a->width);
  const int most = sums ? PKH3_LAYER_NORM_MAX_TABLES : 65535;
  if (a->tables < 1 || a->tables > most) return fail(PKH3_ESHAPE, "tables must be in [1, %d], got %d", most, a->tables);
  return PKH3_OK;
}

int check_norm(const pkh3_norm_args* a, bool backward) {
  int rc = check_norm_sizes(a, backward && a && (a->dweight || a->dbias));
  if (rc) return rc;
  if (!(a->eps >= 0.f) || a->eps > 3e38f) return fail(PKH3_EARG, "eps must be finite and >= 0");
  const int size = a->flags & PKH3_LAYER_NORM_F32 ? 4 : 2, tsize = a->flags & PKH3_LAYER_NORM_TABLES_BF16 ? 2 : 4;
  const Matrix x{"x", a->x, a->x_stride, a->rows, a->width, size}, dy{"dy", a->dy, a->dy_stride, a->rows, a->width, size};
  const Matrix out = backward ? Matrix{"dx", a->dx, a->dx_stride, a->rows, a->width, size} : Matrix{"out", a->out, a->out_stride, a->rows, a->width, size};
  const Matrix w{"weight", a->weight, a->width, a->tables, a->width, tsize}, b{"bias", a->bias, a->width, a->tables, a->width, tsize};
  const Matrix index{"row_index", a->row_index, 1, 1, a->row_index ? a->rows : 0, 4};
  const Matrix dw{"dweight", a->dweight, a->width, a->tables, a->width, 4}, db{"dbias", a->dbias, a->width, a->tables, a->width, 4};
  if (a->rows) {
    if ((rc = check_matrix(x)) || (rc = check_matrix(out))) return rc;
    if (backward && (rc = check_matrix(dy))) return rc;
  }
  if (a->weight && (rc = check_matrix(w))) return rc;
  if (!backward && a->bias && (rc = check_matrix(b))) return rc;
  if (misaligned(a->row_index, 4)) return fail(PKH3_EALIGN, "row_index is not 4-byte aligned");
  if (!same(out, x) && (rc = apart(out, x))) return rc;
  if ((rc = apart(out, w)) || (rc = apart(out, index))) return rc;
  if (!backward) return apart(out, b);
  if (!same(out, dy) && (rc = apart(out, dy))) return rc;
  if (a->dweight && (rc = check_matrix(dw))) return rc;
  if (a->dbias && (rc = check_matrix(db))) return rc;
  for (const Matrix& to : {dw, db})
    for (const Matrix& in : {x, dy, out, w, index})
      if ((rc = apart(to, in))) return rc;
  return apart(dw, db);
}

NormParams norm_params(const pkh3_norm_args* a) {
  const int size = a->flags & PKH3_LAYER_NORM_F32 ? 4 : 2;
  NormParams p{};
  p.x = (const char*)a->x; p.dy = (const char*)a->dy; p.out = (char*)a->out; p.dx = (char*)a->dx;
  p.weight = (const char*)a->weight; p.bias = (const char*)a->bias; p.row_index = a->row_index;
  p.dweight = a->dweight; p.dbias = a->dbias;
  p.x_stride = a->x_stride * size; p.out_stride = a->out_stride * size; p.dy_stride = a->dy_stride * size; p.dx_stride = a->dx_stride * size;
  p.rows = a->rows; p.width = a->width; p.tables = a->tables; p.eps = a->eps;
  return p;
}

// ---- products ----

int mode_of(uint32_t flags) { return (flags & PKH3_PRODUCT_GRAD ? kGrad : kPlain) + (flags & PKH3_PRODUCT_GATED ? 1 : 0); }

int check_product_sizes(const pkh3_product_args* a) {
  if (!a) return fail(PKH3_ENULL, "args is NULL");
  if (a->flags & ~(PKH3_PRODUCT_A_ACROSS | PKH3_PRODUCT_B_ACROSS | PKH3_PRODUCT_GATED | PKH3_PRODUCT_GRAD | PKH3_PRODUCT_BIAS_BF16))
    return fail(PKH3_EARG, "unknown flag bits 0x%x", a->flags);
  if (a->M < 0 || a->M > kMostRows) return fail(PKH3_ESHAPE, "M must be in [0, 2^21], got %d", a->M);
  if (a->N < 8 || a->N > kMostRows || a->N % 8) return fail(PKH3_ESHAPE, "N must be a multiple of 8 in [8, 2^21], got %d", a->N);
  if (a->K < 1 || a->K > kMostRows) return fail(PKH3_ESHAPE, "K must be in [1, 2^21], got %d", a->K);
  if (a->activation < PKH3_ACT_NONE || a->activation > PKH3_ACT_GELU_TANH) return fail(PKH3_EARG, "unknown activation %d", a->activation);
  const bool a_across = a->flags & PKH3_PRODUCT_A_ACROSS, b_across = a->flags & PKH3_PRODUCT_B_ACROSS;
  if (!product_offered(a_across, b_across, mode_of(a->flags))) return fail(PKH3_EUNSUPPORTED, "no product of these operands with flags 0x%x", a->flags);
  if (a_across && a->M % 8) return fail(PKH3_ESHAPE, "M must be a multiple of 8 where A is stored across, got %d", a->M);
  if (!a_across && a->K % 8) return fail(PKH3_ESHAPE, "K must be a multiple of 8 unless both operands are stored across, got %d", a->K);
  return PKH3_OK;
}

int check_product(const pkh3_product_args* a) {
  int rc = check_product_sizes(a);
  if (rc) return rc;
  const int mode = mode_of(a->flags), M = a->M, N = a->N, K = a->K;
  const bool gated = a->flags & PKH3_PRODUCT_GATED, grad = a->flags & PKH3_PRODUCT_GRAD;
  if (grad && a->bias) return fail(PKH3_EARG, "bias does not go with PKH3_PRODUCT_GRAD");
  if ((grad || gated) && (a->gate || a->residual)) return fail(PKH3_EARG, "gate and residual do not go with PKH3_PRODUCT_GRAD or PKH3_PRODUCT_GATED");
  if (!grad && a->sums) return fail(PKH3_EARG, "sums go with PKH3_PRODUCT_GRAD");
  if (mode == kPlain && (a->flags & PKH3_PRODUCT_B_ACROSS) && (a->bias || a->gate || a->residual || a->pre || a->activation))
    return fail(PKH3_EARG, "bias, activation, gate, residual and pre do not go with operands stored across");
  const int wide = gated ? 2 * N : N, b_rows = mode == kGated ? 2 * N : N;
  const Matrix A = a->flags & PKH3_PRODUCT_A_ACROSS ? Matrix{"a", a->a, a->a_stride, K, M, 2} : Matrix{"a", a->a, a->a_stride, M, K, 2};
  const Matrix B = a->flags & PKH3_PRODUCT_B_ACROSS ? Matrix{"b", a->b, a->b_stride, K, b_rows, 2} : Matrix{"b", a->b, a->b_stride, b_rows, K, 2};
  const Matrix out{"out", a->out, a->out_stride, M, mode == kGatedGrad ? wide : N, 2}, pre{"pre", a->pre, a->pre_stride, M, wide, 4};
  const Matrix residual{"residual", a->residual, a->residual_stride, M, N, 2}, gate{"gate", a->gate, a->gate_stride, a->gate_rows, N, 2};
  const Matrix bias{"bias", a->bias, wide, 1, wide, a->flags & PKH3_PRODUCT_BIAS_BF16 ? 2 : 4};
  const Matrix index{"gate_index", a->gate_index, 1, 1, a->gate_index ? M : 0, 4}, sums{"sums", a->sums, wide, 1, wide, 2};
  if (M && ((rc = check_matrix(A)) || (rc = check_matrix(out)))) return rc;
  if ((rc = check_matrix(B))) return rc;
  const bool pre_needed = grad && (gated || a->activation != PKH3_ACT_NONE);
  if (M && (a->pre || pre_needed) && (rc = check_matrix(pre))) return rc;
  if (M && a->residual && (rc = check_matrix(residual))) return rc;
  if (a->gate) {
    if (a->gate_rows < 1 || a->gate_rows > kMostRows) return fail(PKH3_ESHAPE, "gate_rows must be in [1, 2^21], got %d", a->gate_rows);
    if ((rc = check_matrix(gate))) return rc;
    if (misaligned(a->gate_index, 4)) return fail(PKH3_EALIGN, "gate_index is not 4-byte aligned");
  }
  if (a->bias && (rc = check_matrix(bias))) return rc;
  if (a->sums && (rc = check_matrix(sums))) return rc;
  for (const Matrix& in : {A, B, bias, gate, index, pre})
    if ((rc = apart(out, in))) return rc;
  if (!same(out, residual) && (rc = apart(out, residual))) return rc;
  if (!grad)
    for (const Matrix& in : {A, B, bias, gate, index, residual})
      if ((rc = apart(pre, in))) return rc;
  for (const Matrix& in : {A, B, pre, out})
    if ((rc = apart(sums, in))) return rc;
  return PKH3_OK;
}

ProductParams product_params(const pkh3_product_args* a) {
  ProductParams p{};
  p.a = (const char*)a->a; p.b = (const char*)a->b; p.a_stride = a->a_stride * 2; p.b_stride = a->b_stride * 2;
  p.bias = (const char*)a->bias; p.gate = (const char*)a->gate; p.gate_index = a->gate_index; p.residual = (const char*)a->residual;
  p.pre = (char*)a->pre; p.out = (char*)a->out;
  p.gate_stride = a->gate_stride * 2; p.residual_stride = a->residual_stride * 2; p.pre_stride = a->pre_stride * 4; p.out_stride = a->out_stride * 2;
  p.M = a->M; p.N = a->N; p.K = a->K; p.gate_rows = a->gate_rows;
  p.act = a->activation; p.bias_bf16 = a->flags & PKH3_PRODUCT_BIAS_BF16 ? 1 : 0;
  return p;
}

ProductPlan product_plan(const pkh3_product_args* a) {
  return plan_product(a->M, a->N, a->K, !(a->flags & (PKH3_PRODUCT_A_ACROSS | PKH3_PRODUCT_B_ACROSS)), mode_of(a->flags), a->sums != nullptr, a->flags & PKH3_PRODUCT_A_ACROSS);
}

int check_activation_sizes(const pkh3_product_args* a) {
  if (!a) return fail(PKH3_ENULL, "args is NULL");
  if (a->flags) return fail(PKH3_EARG, "unknown flag bits 0x%x", a->flags);
  if (a->M < 0 || a->M > kMostRows) return fail(PKH3_ESHAPE, "M must be in [0, 2^21], got %d", a->M);
  if (a->N < 8 || a->N > kMostRows || a->N % 8) return fail(PKH3_ESHAPE, "N must be a multiple of 8 in [8, 2^21], got %d", a->N);
  if (a->activation < PKH3_ACT_NONE || a->activation > PKH3_ACT_GELU_TANH) return fail(PKH3_EARG, "unknown activation %d", a->activation);
  return PKH3_OK;
}

size_t activation_scratch(const pkh3_product_args* a) {
  return a->sums ? ((size_t)activation_grad_rows(a->M) * a->N * sizeof(float) + 255) / 256 * 256 : 0;
}

}  // namespace

extern "C" {

int pkh3_layer_norm(const pkh3_norm_args* a, void* stream) {
  const int rc = check_norm(a, false);
  if (rc) return rc;
  if (a->rows == 0) return report_error(PKH3_OK, "");
  return done(launch_norm(norm_params(a), a->flags & PKH3_LAYER_NORM_F32, a->flags & PKH3_LAYER_NORM_TABLES_BF16, (hipStream_t)stream), "layer norm");
}

size_t pkh3_norm_workspace_bytes(const pkh3_norm_args* a) {
  if (check_norm_sizes(a, true)) return 0;
  report_error(PKH3_OK, "");
  return norm_scratch_bytes(a->rows < 1 ? 1 : a->rows, a->width, a->tables);
}

int pkh3_layer_norm_backward(const pkh3_norm_args* a, void* stream) {
  int rc = check_norm(a, true);
  if (rc) return rc;
  if (a->rows == 0) {
    if (a->dweight || a->dbias) return fail(PKH3_ESHAPE, "no rows: the tables' gradients are zeros, which this call does not write");
    return report_error(PKH3_OK, "");
  }
  if ((a->dweight || a->dbias) && (rc = check_workspace(a->workspace, a->workspace_bytes, norm_scratch_bytes(a->rows, a->width, a->tables)))) return rc;
  return done(launch_norm_backward(norm_params(a), a->flags & PKH3_LAYER_NORM_F32, a->flags & PKH3_LAYER_NORM_TABLES_BF16, (char*)a->workspace, (hipStream_t)stream),
              "layer norm backward");
}

size_t pkh3_product_workspace_bytes(const pkh3_product_args* a) {
  if (check_product_sizes(a)) return 0;
  report_error(PKH3_OK, "");
  return product_plan(a).total;
}

int pkh3_product(const pkh3_product_args* a, void* stream) {
  int rc = check_product(a);
  if (rc) return rc;
  if (a->M == 0) {
    if (a->sums) return fail(PKH3_ESHAPE, "no rows: the sums are zeros, which this call does not write");
    return report_error(PKH3_OK, "");
  }
  const ProductPlan plan = product_plan(a);
  if ((rc = check_workspace(a->workspace, a->workspace_bytes, plan.total))) return rc;
  return done(launch_product(product_params(a), plan, a->flags & PKH3_PRODUCT_A_ACROSS, a->flags & PKH3_PRODUCT_B_ACROSS, mode_of(a->flags), a->sums,
                             (char*)a->workspace, (hipStream_t)stream), "product");
}

size_t pkh3_activation_grad_workspace_bytes(const pkh3_product_args* a) {
  if (check_activation_sizes(a)) return 0;
  report_error(PKH3_OK, "");
  return activation_scratch(a);
}

int pkh3_activation_grad(const pkh3_product_args* a, void* stream) {
  int rc = check_activation_sizes(a);
  if (rc) return rc;
  const bool act = a->activation != PKH3_ACT_NONE;
  const Matrix in{"a", a->a, a->a_stride, a->M, a->N, 2}, out{"out", a->out, a->out_stride, a->M, a->N, 2}, pre{"pre", a->pre, a->pre_stride, a->M, a->N, 4};
  const Matrix sums{"sums", a->sums, a->N, 1, a->N, 2};
  if (a->M) {
    if ((rc = check_matrix(in))) return rc;
    if ((act || a->out) && (rc = check_matrix(out))) return rc;
    if (act && (rc = check_matrix(pre))) return rc;
  }
  if (a->sums && (rc = check_matrix(sums))) return rc;
  if (!same(out, in) && (rc = apart(out, in))) return rc;
  if (act && ((rc = apart(out, pre)) || (rc = apart(sums, pre)))) return rc;
  if ((rc = apart(sums, in)) || (rc = apart(sums, out))) return rc;
  if (a->M == 0) {
    if (a->sums) return fail(PKH3_ESHAPE, "no rows: the sums are zeros, which this call does not write");
    return report_error(PKH3_OK, "");
  }
  if ((rc = check_workspace(a->workspace, a->workspace_bytes, activation_scratch(a)))) return rc;
  return done(launch_activation_grad(product_params(a), a->sums, (char*)a->workspace, (hipStream_t)stream), "activation gradient");
}

}  // extern "C"
