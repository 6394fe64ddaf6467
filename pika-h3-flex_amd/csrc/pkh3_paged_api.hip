// C ABI of the paged K/V cache (include/pkh3_paged.h): argument validation on the host, then the launches.
#include "../../include/pkh3_paged.h"
#include "../../include/pkh3_attn.h"

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "pkh3_internal.h"
#include "pkh3_paged.h"

using namespace pkh3;

namespace {

static_assert(PKH3_PAGE_KEYS == kTileKeys && PKH3_PAGED_MAX_SEQUENCES == kMaxSequences, "header and kernels");

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

// Whether two of rows x heads pieces of 128 elements share an element, strides of 128 at least.  Where the outer stride passes over all of the inner pieces
// they do not (every slice of a tensor); otherwise each distance along the inner one is held against the two multiples of the outer one beside it.
bool overlaps(int64_t ss, int64_t sh, int rows, int heads) {
  if (rows < 2 || heads < 2) return false;
  const int64_t outer = ss > sh ? ss : sh, inner = ss > sh ? sh : ss;
  const int n_outer = ss > sh ? rows : heads, n_inner = ss > sh ? heads : rows;
  if ((outer - kD) / inner >= n_inner - 1) return false;
  for (int i = 1; i < n_inner; ++i) {
    const __int128 d = (__int128)inner * i, j = d / outer;
    if (j >= n_outer) return false;                        // (and all further ones are past the last of the outer)
    if (j >= 1 && d - j * outer < kD) return true;
    if (j + 1 < n_outer && (j + 1) * outer - d < kD) return true;
  }
  return false;
}

int check_rows(const char* name, const void* ptr, int64_t ss, int64_t sh, int rows, int heads, bool out) {
  if (!ptr) return fail(PKH3_ENULL, "%s is NULL", name);
  if (misaligned(ptr, 16)) return fail(PKH3_EALIGN, "%s is not 16-byte aligned", name);
  if (ss < 0 || sh < 0) return fail(PKH3_ESTRIDE, "%s: negative stride", name);
  if ((ss % 8) || (sh % 8)) return fail(PKH3_ESTRIDE, "%s: strides must be multiples of 8 elements, got (%lld, %lld)", name, (long long)ss, (long long)sh);
  if (out && (ss < kD || (heads > 1 && sh < kD) || overlaps(ss, sh, rows, heads)))
    return fail(PKH3_ESTRIDE, "%s: rows or heads that are written overlap (strides %lld, %lld)", name, (long long)ss, (long long)sh);
  return PKH3_OK;
}

enum Call { kWrite, kRead, kAttn };

// what the host can know of the sizes
int check_sizes(const pkh3_paged_args* a, Call call) {
  if (!a) return fail(PKH3_ENULL, "args is NULL");
  if (a->D != kD) return fail(PKH3_EHEADDIM, "head dim must be 128, got %d", a->D);
  if (a->flags & ~(uint32_t)(PKH3_PAGED_FP8 | PKH3_PAGED_CAUSAL)) return fail(PKH3_EARG, "unknown flag bits 0x%x", a->flags);
  if ((a->flags & PKH3_PAGED_CAUSAL) && call != kAttn) return fail(PKH3_EARG, "PKH3_PAGED_CAUSAL belongs to pkh3_paged_attn");
  if (a->B < 1 || a->B > kMaxSequences) return fail(PKH3_ESHAPE, "B must be in [1, %d], got %d", kMaxSequences, a->B);
  if (a->rows < 0 || a->rows > (1 << 24)) return fail(PKH3_ESHAPE, "rows must be in [0, 2^24], got %d", a->rows);
  if (a->kv_heads < 1 || a->kv_heads > 65535) return fail(PKH3_ESHAPE, "kv_heads must be in [1, 65535], got %d", a->kv_heads);
  if (a->table_pages < 1 || a->table_pages > (1 << 24)) return fail(PKH3_ESHAPE, "table_pages must be in [1, 2^24], got %d", a->table_pages);
  if (a->table_stride < 0) return fail(PKH3_ESTRIDE, "table: negative stride");
  if (a->n_pages < 1 || a->n_pages > 0x7fffffffll) return fail(PKH3_ESHAPE, "n_pages must be in [1, 2^31), got %lld", (long long)a->n_pages);
  const int64_t heads = call == kAttn ? a->heads : a->kv_heads;
  if (call == kAttn && (a->heads < 1 || a->heads > 65535 || a->heads % a->kv_heads))
    return fail(PKH3_ESHAPE, "heads must be a multiple of kv_heads in [1, 65535], got %d and %d", a->heads, a->kv_heads);
  if (((int64_t)a->rows + 64ll * a->B) * heads > (1ll << 30)) return fail(PKH3_ESHAPE, "(rows + 64 * B) * heads must be <= 2^30");
  if (call == kAttn && (!(a->softmax_scale == a->softmax_scale) || isinf(a->softmax_scale))) return fail(PKH3_EARG, "softmax_scale is not finite");
  if (call != kRead) {
    if (a->rope_mode < PKH3_ROPE_NONE || a->rope_mode > PKH3_ROPE_HALF) return fail(PKH3_EARG, "bad rope_mode %d", a->rope_mode);
    if (a->norm_w && !(a->norm_eps >= 0.f)) return fail(PKH3_EARG, "norm_eps must be >= 0");
  }
  return PKH3_OK;
}

int check(const pkh3_paged_args* a, Call call) {
  int rc = check_sizes(a, call);
  if (rc) return rc;
  if (!a->pages) return fail(PKH3_ENULL, "pages is NULL");
  if (misaligned(a->pages, 256)) return fail(PKH3_EALIGN, "pages is not 256-byte aligned");
  if (!a->starts || !a->lengths || !a->table) return fail(PKH3_ENULL, "starts, lengths and table must not be NULL");
  if (misaligned(a->starts, 4) || misaligned(a->lengths, 4) || misaligned(a->table, 4)) return fail(PKH3_EALIGN, "starts, lengths and table must be 4-byte aligned");
  if (call == kAttn) {
    if ((rc = check_rows("q", a->q, a->q_ss, a->q_sh, a->rows, a->heads, false))) return rc;
    if ((rc = check_rows("o", a->o, a->o_ss, a->o_sh, a->rows, a->heads, true))) return rc;
  } else {
    if ((rc = check_rows("k", a->k, a->k_ss, a->k_sh, a->rows, a->kv_heads, call == kRead))) return rc;
    if ((rc = check_rows("v", a->v, a->v_ss, a->v_sh, a->rows, a->kv_heads, call == kRead))) return rc;
  }
  if (call != kRead) {
    if (a->rope_mode != PKH3_ROPE_NONE) {
      if (!a->rope_cos || !a->rope_sin) return fail(PKH3_ENULL, "rope_mode set but a cos/sin table is NULL");
      if (misaligned(a->rope_cos, 16) || misaligned(a->rope_sin, 16)) return fail(PKH3_EALIGN, "rope tables must be 16-byte aligned");
    }
    if (a->norm_w && misaligned(a->norm_w, 16)) return fail(PKH3_EALIGN, "norm weights must be 16-byte aligned");
  }
  if (call == kRead && a->rows > 0 && a->k == a->v) return fail(PKH3_EARG, "k and v are written to one place");
  return PKH3_OK;
}

PagedParams params(const pkh3_paged_args* a) {
  PagedParams p{};
  p.pages = (char*)a->pages; p.n_pages = a->n_pages;
  p.page_stride = (int64_t)a->kv_heads * (a->flags & PKH3_PAGED_FP8 ? kPageRecord8 : kPageRecord16);
  p.starts = a->starts; p.lengths = a->lengths; p.table = a->table; p.table_stride = a->table_stride;
  p.B = a->B; p.table_pages = a->table_pages; p.rows = a->rows; p.H = a->kv_heads;
  p.q = (const char*)a->q; p.k = (char*)a->k; p.v = (char*)a->v; p.o = (char*)a->o;
  p.q_ss = a->q_ss * 2; p.q_sh = a->q_sh * 2; p.k_ss = a->k_ss * 2; p.k_sh = a->k_sh * 2;
  p.v_ss = a->v_ss * 2; p.v_sh = a->v_sh * 2; p.o_ss = a->o_ss * 2; p.o_sh = a->o_sh * 2;
  p.norm_w = a->norm_w; p.eps = a->norm_eps; p.rope_mode = a->rope_mode; p.cos_t = a->rope_cos; p.sin_t = a->rope_sin;
  p.causal = (a->flags & PKH3_PAGED_CAUSAL) ? 1 : 0;
  return p;
}

size_t scratch(const pkh3_paged_args* a) {
  return (paged_attn_scratch(a->rows, a->B, a->kv_heads, a->heads / a->kv_heads, a->table_pages, a->flags & PKH3_PAGED_FP8) * sizeof(float) + 255) / 256 * 256;
}

}  // namespace

extern "C" {

size_t pkh3_paged_record_bytes(uint32_t flags) {
  if (flags & ~(uint32_t)(PKH3_PAGED_FP8 | PKH3_PAGED_CAUSAL)) {
    fail(PKH3_EARG, "unknown flag bits 0x%x", flags);
    return 0;
  }
  return flags & PKH3_PAGED_FP8 ? kPageRecord8 : kPageRecord16;
}

int pkh3_paged_write(const pkh3_paged_args* a, void* stream) {
  const int rc = check(a, kWrite);
  if (rc) return rc;
  if (a->rows == 0) return report_error(PKH3_OK, "");
  return done(launch_paged_write(params(a), a->flags & PKH3_PAGED_FP8, (hipStream_t)stream), "paged write");
}

int pkh3_paged_read(const pkh3_paged_args* a, void* stream) {
  const int rc = check(a, kRead);
  if (rc) return rc;
  if (a->rows == 0) return report_error(PKH3_OK, "");
  return done(launch_paged_read(params(a), a->flags & PKH3_PAGED_FP8, (hipStream_t)stream), "paged read");
}

size_t pkh3_paged_workspace_bytes(const pkh3_paged_args* a) {
  if (check_sizes(a, kAttn)) return 0;
  return scratch(a);
}

int pkh3_paged_attn(const pkh3_paged_args* a, void* stream) {
  const int rc = check(a, kAttn);
  if (rc) return rc;
  if (!a->workspace) return fail(PKH3_EWORKSPACE, "workspace is NULL");
  if (misaligned(a->workspace, 256)) return fail(PKH3_EWORKSPACE, "workspace is not 256-byte aligned");
  if (a->workspace_bytes < scratch(a)) return fail(PKH3_EWORKSPACE, "workspace too small: %zu < %zu bytes", a->workspace_bytes, scratch(a));
  if (a->rows == 0) return report_error(PKH3_OK, "");
  PagedParams p = params(a);
  p.G = make_group(a->heads / a->kv_heads);
  p.c = (a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / sqrtf((float)kD)) * kLog2e;
  p.cuts = (i32x4*)a->workspace;
  p.partials = (float*)a->workspace + 4 * kMaxShares;
  return done(launch_paged_attn(p, a->flags & PKH3_PAGED_FP8, (hipStream_t)stream), "paged attention");
}

}  // extern "C"
