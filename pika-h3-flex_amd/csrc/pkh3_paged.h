// The paged K/V cache: layout of its records, and how the kernels find their way through a batch of sequences whose rows,
// lengths and pages are known on the device only.
#pragma once
#include "pkh3_common.h"
#include "pkh3_paged_index.h"

namespace pkh3 {

// A record: one page (64 keys) of one kv head.  bf16: the K tile and the V tile of pkh3_common.h.  e4m3: K as its fp8 K tile,
// V as images of two 16-column blocks side by side, then an exponent byte (E8M0) per key for K and one for V:
//   V byte ((half*4 + dbp)*64 + l)*16 + 8*par + j holds V[32*half + v_image_key(g, j)][16*(2*dbp + par) + c] / scale,
// so that 16 bytes of a lane become its two 16-byte pieces of bf16 images, of K as of V.
constexpr int kPageRecord16 = kKTileBytes + kVTileBytes;
constexpr int kPageScales = 2 * kTileKeys;
constexpr int kPageRecord8 = kK8TileBytes + kVTileBytes / 2 + kPageScales;
constexpr int kMaxSequences = 1024;
static_assert(kPageKeys == kTileKeys, "a page is a tile of keys");

struct PagedParams {
  char* pages;
  int64_t n_pages, page_stride;      // bytes from page to page; a head's record follows the one before it
  const int* starts;
  const int* lengths;
  const int* table;
  int64_t table_stride;
  int B, table_pages, rows, H;       // H: heads of the cache
  // rows in (write: k; attn: q) and out
  const char* q;
  char* k;
  char* v;
  char* o;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;   // bytes
  const float* norm_w;
  float eps;
  int rope_mode;
  const float* cos_t;
  const float* sin_t;
  int heads_per_wg, groups;          // write, read
  int whole;                         // attn: no unit is cut (short tables), and there is no second launch
  Group G;                           // attn: query heads of one of the cache's
  float c;                           // attn: softmax scale * log2(e)
  int causal;
  i32x4* cuts;                       // attn: where runs begin inside a unit, and ...
  float* partials;                   // ... the parts of units (see pkh3_paged_attn.hip)
};

__device__ __forceinline__ Sequence sequence(const PagedParams& p, int b) {
  return make_sequence(p.starts[b], p.starts[b + 1], p.lengths[b], p.rows, p.table_pages);
}
// the same of a wave-uniform sequence, and the page of its tile (or -1), through the scalar cache
__device__ __forceinline__ int uniform_int(const int* p, int64_t i) { return ((const __attribute__((address_space(4))) int*)p)[i]; }
__device__ __forceinline__ Sequence uniform_sequence(const PagedParams& p, int b) {
  return make_sequence(uniform_int(p.starts, b), uniform_int(p.starts, b + 1), uniform_int(p.lengths, b), p.rows, p.table_pages);
}
// .. and both as a write takes them
template <bool WRITES>
__device__ __forceinline__ Sequence moved_sequence(const PagedParams& p, int b) {
  return WRITES ? make_written(p.starts[b], p.starts[b + 1], p.lengths[b], p.rows, p.table_pages) : sequence(p, b);
}
template <bool WRITES>
__device__ __forceinline__ Sequence uniform_moved_sequence(const PagedParams& p, int b) {
  return WRITES ? make_written(uniform_int(p.starts, b), uniform_int(p.starts, b + 1), uniform_int(p.lengths, b), p.rows, p.table_pages) : uniform_sequence(p, b);
}
__device__ __forceinline__ int uniform_page(const PagedParams& p, int b, int tile) {
  if (tile < 0 || tile >= p.table_pages) return -1;
  return page_in_pool(uniform_int(p.table, (int64_t)b * p.table_stride + tile), p.n_pages);
}

// cum[b + 1] = the sum of cum[1 .. b + 1], cum[0] = 0, by the first wave; every wave goes through the barriers
__device__ __forceinline__ void prefix_sums(int64_t* cum, int B) {
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int64_t before = 0;
    for (int at = 0; at < B; at += 64) {
      const int b = at + lane;
      int64_t x = b < B ? cum[b + 1] : 0;
      for (int d = 1; d < 64 && d < B; d <<= 1) {
        const int64_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
      x += before;
      if (b < B) cum[b + 1] = x;
      before = __shfl(x, 63);
    }
    if (lane == 0) cum[0] = 0;
  }
  __syncthreads();
}
// the sequence b with cum[b] <= pos < cum[b + 1], for 0 <= pos < cum[B]
__device__ __forceinline__ int find_sequence(const int64_t* cum, int B, int64_t pos) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= pos) lo = mid;
    else hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// eight e4m3 bytes of a lane times a power of two, exact in bf16 (a scale's smallest products, below 2^-126, may become 0)
__device__ __forceinline__ bf16x8 expand_fp8(int lo, int hi, float scale) {
  bf16x8 out;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const unsigned src = w == 0 ? lo : hi;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, true);
    out[4 * w] = a[0], out[4 * w + 1] = a[1], out[4 * w + 2] = b[0], out[4 * w + 3] = b[1];
  }
  return out;
}
__device__ __forceinline__ float exponent_scale(unsigned byte) { return __uint_as_float(byte << 23); }
// the same of eight keys' values, each times its own scale (exponent bytes e[0], e[1])
__device__ __forceinline__ bf16x8 expand_fp8_keys(int lo, int hi, const unsigned (&e)[2]) {
  bf16x8 out;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned src = j < 4 ? lo : hi;
    const float scale = exponent_scale((e[j >> 2] >> (8 * (j & 3))) & 0xffu);
    const bf16x2 both = (j & 2) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, false);
    out[j] = both[j & 1];
  }
  return out;
}

hipError_t launch_paged_write(const PagedParams& p, bool fp8, hipStream_t st);
hipError_t launch_paged_read(const PagedParams& p, bool fp8, hipStream_t st);
hipError_t launch_paged_attn(const PagedParams& p, bool fp8, hipStream_t st);
// scratch of the attention call in floats, from the sizes that the host knows
size_t paged_attn_scratch(int rows, int B, int H, int G, int table_pages, bool fp8);

}  // namespace pkh3
