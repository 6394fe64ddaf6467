// Writing the paged K/V cache and reading it back.  Both are one pass over rows and pages, bound by HBM: 15,342 rows of 24 heads in e4m3 are
// written in 59 to 67 us (norm, rotation, rounding; 288 MB, 4.3 to 4.9 TB/s) and read back in 47 to 48 (284 MB, 5.9 TB/s).  A few rows are a launch:
// 4.4 and 3.7 us.
//
// A workgroup takes one 64-key tile of one sequence for `heads_per_wg` heads, its K or its V (by the parity of blockIdx.x), as the
// K/V pass of the dense calls does: rows as they lie in memory, turned around in LDS into the lane order of the operand images.
// Which tile that is follows from the batch's arrays: every workgroup adds the tiles of all sequences up and looks itself up there.
// A tile of which the call has all 64 rows is written as whole images; of any other tile no byte of another key is touched -- a K piece
// of 16 bytes belongs to one key, a V piece to eight, so at the ends of a chunk V goes out value by value.
#include "pkh3_paged.h"
#include "pkh3_internal.h"

namespace pkh3 {

// The tile that a workgroup works on, and whose it is.
struct Item {
  int b;
  TileRows t;
};
template <bool WRITES>
__device__ __forceinline__ bool find_tile(const PagedParams& p, int64_t* cum, int nth, Item& it) {
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) cum[b + 1] = tiles_of_rows(moved_sequence<WRITES>(p, b));
  prefix_sums(cum, p.B);
  if (nth >= cum[p.B]) return false;
  it.b = find_sequence(cum, p.B, nth);
  it.t = tile_rows(uniform_moved_sequence<WRITES>(p, it.b), __builtin_amdgcn_readfirstlane((int)(nth - cum[it.b])));
  return true;
}

__device__ __forceinline__ float row_max16(float x) {   // over the 16 lanes of a row
  x = max_with<0xB1>(x);
  x = max_with<0x4E>(x);
  x = max_with<0x141>(x);
  return max_with<0x140>(x);
}
// What is not finite is stored as NaN and counts as nothing for the scale.  The conversion does that with NaN, and the largest magnitude passes over it; a
// largest magnitude of infinity says that the careful way is needed.
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// x / scale to e4m3; what is not finite becomes NaN
__device__ __forceinline__ float to_quantise(float x, float inv) { return fabsf(x) < INFINITY ? x * inv : __builtin_nanf(""); }
// a row's scale: 2^-126 to 2^120 for finite values, so that its inverse is a normal number as well
__device__ __forceinline__ float key_scale(float amax) { return fp8_block_scale(amax, true); }

template <bool FP8>
__device__ __forceinline__ void write_k(const PagedParams& p, const TileRows& t, char* page, int h0, int n_heads, char* turn) {
  const int lane = threadIdx.x & 63, kb = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int place = kb * 16 + c;
  const bool mine = place >= t.p0 && place < t.p1;
  int src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) src[i] = t.row0 + min(max(kb * 16 + 4 * i + g, t.p0), t.p1 - 1);
  const char* x0 = p.k + (int64_t)h0 * p.k_sh;
  Rows16 next, cos, sin;
  ask_rows16(next, x0, p.k_ss, src, lane);
  NormLanes norm;
  load_norm_lanes(norm, p.norm_w, lane);
  RopeQuarter rope;
  if (p.rope_mode != 0) {
    ask_rows16(cos, (const char*)p.cos_t, kD / 2 * sizeof(float), src, lane);
    ask_rows16(sin, (const char*)p.sin_t, kD / 2 * sizeof(float), src, lane);
    turn_table(cos, rope.c, p.rope_mode, turn, lane);
    turn_table(sin, rope.s, p.rope_mode, turn, lane);
  }
#pragma unroll 1
  for (int hi = 0; hi < n_heads; ++hi) {
    char* record = page + (int64_t)(h0 + hi) * (FP8 ? kPageRecord8 : kPageRecord16);
    bf16x8 raw[4];
    float x[32];
    turn_elements(next, raw, turn, lane);
    if (hi + 1 < n_heads) ask_rows16(next, x0 + (int64_t)(hi + 1) * p.k_sh, p.k_ss, src, lane);
    norm_row(x, raw, p.norm_w != nullptr, p.eps, norm, 1.0f);
    rope_row(x, p.rope_mode, rope);
    if constexpr (!FP8) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        bf16x8 w;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = (__bf16)x[ks * 8 + j];
        if (mine) *(bf16x8*)(record + ((((kb >> 1) * 4 + ks) * 2 + (kb & 1)) * 64 + lane) * 16) = w;
      }
    } else {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
      if (__any(!(amax < INFINITY))) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          amax = fmaxf(amax, finite_magnitude(x[i]));
          x[i] = to_quantise(x[i], 1.0f);
        }
      }
      const float scale = key_scale(max_across_groups(amax));
      const float inv = 1.0f / scale;
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        const i32x2 q0 = quant_fp8_piece(x + 16 * c2, inv), q1 = quant_fp8_piece(x + 16 * c2 + 8, inv);
        if (mine) *(i32x4*)(record + ((kb * 2 + c2) * 64 + lane) * 16) = i32x4{q0[0], q0[1], q1[0], q1[1]};
      }
      if (mine && g == 0) record[kK8TileBytes + kVTileBytes / 2 + place] = (char)e8m0_of(scale);
    }
  }
}

// V: wave (half, odd) takes 32 keys of the even or odd heads; through 8 KiB of LDS of its own, from where transposing reads give it back in
// the images' order (see v_tile of the dense calls' K/V pass).
template <bool FP8>
__device__ __forceinline__ void write_v(const PagedParams& p, const TileRows& t, char* page, int h0, int n_heads, char* lds, float* inv_scale) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave & 1, first = wave >> 1;
  const int g = lane >> 4, c = lane & 15;
  char* mine = lds + wave * 8192;
  float* inv_of = inv_scale + wave * 32;
  if (half * 32 >= t.p1 || half * 32 + 32 <= t.p0 || first >= n_heads) return;
  const bool whole = t.p0 <= half * 32 && t.p1 >= half * 32 + 32;
  const char* vr[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    vr[i] = p.v + (int64_t)(t.row0 + min(max(half * 32 + 4 * i + g, t.p0), t.p1 - 1)) * p.v_ss + 16 * c;
  auto fetch = [&](bf16x8 (&raw)[8], int hi) {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = *(const bf16x8*)(vr[i] + (int64_t)(h0 + hi) * p.v_sh);
  };
  bf16x8 next[8];
  fetch(next, first);
#pragma unroll 1
  for (int hi = first; hi < n_heads; hi += 2) {
    char* record = page + (int64_t)(h0 + hi) * (FP8 ? kPageRecord8 : kPageRecord16);
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf((float)next[i][j]));
        if (__any(!(amax < INFINITY))) {
          amax = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            amax = fmaxf(amax, finite_magnitude((float)next[i][j]));
            next[i][j] = (__bf16)to_quantise((float)next[i][j], 1.0f);
          }
        }
        const float scale = key_scale(row_max16(amax));
        const int place = half * 32 + 4 * i + g;
        if (c == 0) {
          inv_of[4 * i + g] = 1.0f / scale;
          if (place >= t.p0 && place < t.p1) record[kK8TileBytes + kVTileBytes / 2 + 64 + place] = (char)e8m0_of(scale);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + g;
      *(bf16x8*)(mine + r * 256 + ((c ^ (2 * (r & 7))) * 16)) = next[i];
    }
    if (hi + 2 < n_heads) fetch(next, hi + 2);
    float inv[8];
    if constexpr (FP8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = inv_of[v_image_key(g, j)];
    }
    i32x2 bytes[2];
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      bf16x8 img;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int r = 16 * kb + 4 * g + (c >> 2);      // the row this lane names, columns 16*db + 4*(c%4) .. +3
        const auto w = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(mine + r * 256 + ((db ^ (r & 7)) * 32) + 8 * (c & 3)));
#pragma unroll
        for (int j = 0; j < 4; ++j) img[4 * kb + j] = w[j];
      }
      if constexpr (!FP8) {
        __bf16* to = (__bf16*)(record + kKTileBytes + ((half * 8 + db) * 64 + lane) * 16);
        if (whole) {
          *(bf16x8*)to = img;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int place = half * 32 + v_image_key(g, j);
            if (place >= t.p0 && place < t.p1) to[j] = img[j];
          }
        }
      } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)img[j] * inv[j];
        bytes[db & 1] = quant_fp8_piece(x, 1.0f);
        if (db & 1) {
          char* to = record + kK8TileBytes + ((half * 4 + (db >> 1)) * 64 + lane) * 16;
          if (whole) {
            *(i32x4*)to = i32x4{bytes[0][0], bytes[0][1], bytes[1][0], bytes[1][1]};
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int place = half * 32 + v_image_key(g, j);
              if (place >= t.p0 && place < t.p1) {
                to[j] = (char)(bytes[0][j >> 2] >> (8 * (j & 3)));
                to[8 + j] = (char)(bytes[1][j >> 2] >> (8 * (j & 3)));
              }
            }
          }
        }
      }
    }
  }
}

template <bool FP8>
__global__ __launch_bounds__(256, 3) void paged_write_kernel(PagedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[4 * 8192];
  __shared__ float inv_scale[4 * 32];
  static_assert((kMaxSequences + 1) * sizeof(int64_t) <= sizeof(lds), "the sums lie where the rows are turned around afterwards");
  const int side = blockIdx.x & 1, group = (blockIdx.x >> 1) % p.groups, nth = (blockIdx.x >> 1) / p.groups;
  Item it;
  if (!find_tile<true>(p, (int64_t*)lds, nth, it)) return;
  __syncthreads();
  const TileRows& t = it.t;
  const int64_t id = uniform_page(p, it.b, t.tile);
  if (id < 0 || t.p0 >= t.p1) return;
  char* page = p.pages + id * p.page_stride;
  const int h0 = group * p.heads_per_wg, n_heads = min(p.heads_per_wg, p.H - h0);
  if (side == 0) write_k<FP8>(p, t, page, h0, n_heads, lds + (threadIdx.x >> 6) * 4096);
  else write_v<FP8>(p, t, page, h0, n_heads, lds, inv_scale);
}

// ---- reading back ----

// sixteen rows of 256 bytes out of a wave's LDS (chunk j of row r at chunk j ^ r) to the call's rows
__device__ __forceinline__ void store_rows16(const char* turn, char* out, int64_t row_bytes, const TileRows& t, int place0, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * i + (lane >> 4), place = place0 + r;
    const i32x4 v = *(const i32x4*)(turn + r * 256 + (((lane & 15) ^ r) * 16));
    if (place >= t.p0 && place < t.p1) *(i32x4*)(out + (int64_t)(t.row0 + place) * row_bytes + (lane & 15) * 16) = v;
  }
}

template <bool FP8>
__device__ __forceinline__ void read_k(const PagedParams& p, const TileRows& t, const char* page, int h0, int n_heads, char* turn) {
  const int lane = threadIdx.x & 63, kb = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  if (kb * 16 >= t.p1 || kb * 16 + 16 <= t.p0) return;
#pragma unroll 1
  for (int hi = 0; hi < n_heads; ++hi) {
    bf16x8 piece[4];
    if (!page) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) piece[ks] = bf16x8{};
    } else if constexpr (!FP8) {
      const char* record = page + (int64_t)(h0 + hi) * kPageRecord16;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) piece[ks] = *(const bf16x8*)(record + ((((kb >> 1) * 4 + ks) * 2 + (kb & 1)) * 64 + lane) * 16);
    } else {
      const char* record = page + (int64_t)(h0 + hi) * kPageRecord8;
      const float scale = exponent_scale((unsigned char)record[kK8TileBytes + kVTileBytes / 2 + kb * 16 + c]);
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        const i32x4 w = *(const i32x4*)(record + ((kb * 2 + c2) * 64 + lane) * 16);
        piece[2 * c2] = expand_fp8(w[0], w[1], scale);
        piece[2 * c2 + 1] = expand_fp8(w[2], w[3], scale);
      }
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) *(bf16x8*)(turn + c * 256 + (((4 * ks + g) ^ c) * 16)) = piece[ks];
    store_rows16(turn, p.k + (int64_t)(h0 + hi) * p.k_sh, p.k_ss, t, kb * 16, lane);
  }
}

// V: the images go to LDS as they are, and the transposing read turns 4 columns x 16 keys of them at a time: lane 4*r + m of the 16-lane group g
// names the keys 16*kb + 4*m .. +3 of column 16*db + 4*g + r, and lane c gets the columns 16*db + 4*g .. +3 of key 16*kb + c.
template <bool FP8>
__device__ __forceinline__ void read_v(const PagedParams& p, const TileRows& t, const char* page, int h0, int n_heads, char* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave & 1, first = wave >> 1;
  const int g = lane >> 4, c = lane & 15;
  char* mine = lds + wave * 8192;
  if (half * 32 >= t.p1 || half * 32 + 32 <= t.p0) return;
#pragma unroll 1
  for (int hi = first; hi < n_heads; hi += 2) {
    bf16x8 img[8];
    if (!page) {
#pragma unroll
      for (int db = 0; db < 8; ++db) img[db] = bf16x8{};
    } else if constexpr (!FP8) {
      const char* record = page + (int64_t)(h0 + hi) * kPageRecord16 + kKTileBytes;
#pragma unroll
      for (int db = 0; db < 8; ++db) img[db] = *(const bf16x8*)(record + ((half * 8 + db) * 64 + lane) * 16);
    } else {
      const char* record = page + (int64_t)(h0 + hi) * kPageRecord8 + kK8TileBytes;
      const unsigned* exps = (const unsigned*)(record + kVTileBytes / 2 + 64 + half * 32);
      unsigned e[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) e[kb] = exps[4 * kb + g];
#pragma unroll
      for (int dbp = 0; dbp < 4; ++dbp) {
        const i32x4 w = *(const i32x4*)(record + ((half * 4 + dbp) * 64 + lane) * 16);
#pragma unroll
        for (int par = 0; par < 2; ++par) img[2 * dbp + par] = expand_fp8_keys(w[2 * par], w[2 * par + 1], e);
      }
    }
#pragma unroll
    for (int db = 0; db < 8; ++db) *(bf16x8*)(mine + (db * 64 + lane) * 16) = img[db];
    bf16x4 out[2][8];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const auto w = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(mine + (db * 64 + 16 * (c & 3) + 4 * g + (c >> 2)) * 16 + 8 * kb));
#pragma unroll
        for (int j = 0; j < 4; ++j) out[kb][db][j] = w[j];
      }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int db = 0; db < 8; ++db)
        *(bf16x4*)(mine + kb * 4096 + c * 256 + (((2 * db + (g >> 1)) ^ c) * 16) + 8 * (g & 1)) = out[kb][db];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) store_rows16(mine + kb * 4096, p.v + (int64_t)(h0 + hi) * p.v_sh, p.v_ss, t, half * 32 + kb * 16, lane);
  }
}

template <bool FP8>
__global__ __launch_bounds__(256, 3) void paged_read_kernel(PagedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[4 * 8192];
  const int side = blockIdx.x & 1, group = (blockIdx.x >> 1) % p.groups, nth = (blockIdx.x >> 1) / p.groups;
  Item it;
  if (!find_tile<false>(p, (int64_t*)lds, nth, it)) return;
  __syncthreads();
  const TileRows& t = it.t;
  const int64_t id = uniform_page(p, it.b, t.tile);
  const char* page = id < 0 ? nullptr : p.pages + id * p.page_stride;
  const int h0 = group * p.heads_per_wg, n_heads = min(p.heads_per_wg, p.H - h0);
  if (side == 0) read_k<FP8>(p, t, page, h0, n_heads, lds + (threadIdx.x >> 6) * 4096);
  else read_v<FP8>(p, t, page, h0, n_heads, lds);
}

// Heads a workgroup: fewer than eight where eight would leave CUs without one.
static hipError_t split_heads(PagedParams& p, int64_t tiles) {
  int cus = 0;
  const hipError_t e = device_cu_count(&cus);
  if (e != hipSuccess) return e;
  int per = p.H < 8 ? p.H : 8;
  while (per > 1 && 2 * tiles * ((p.H + per - 1) / per) < 8 * (int64_t)cus) per = (per + 1) / 2;
  p.heads_per_wg = per;
  p.groups = (p.H + per - 1) / per;
  return hipSuccess;
}

hipError_t launch_paged_write(const PagedParams& given, bool fp8, hipStream_t st) {
  PagedParams p = given;
  const int64_t tiles = most_tiles(p.rows, p.B);
  const hipError_t e = split_heads(p, tiles);
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(2 * tiles * p.groups));
  if (fp8) hipLaunchKernelGGL(paged_write_kernel<true>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_write_kernel<false>, grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_paged_read(const PagedParams& given, bool fp8, hipStream_t st) {
  PagedParams p = given;
  const int64_t tiles = most_tiles(p.rows, p.B);
  const hipError_t e = split_heads(p, tiles);
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(2 * tiles * p.groups));
  if (fp8) hipLaunchKernelGGL(paged_read_kernel<true>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_read_kernel<false>, grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace pkh3
