// What a wave of the attention kernels is made of: its state for 32 queries, copies of key tiles from memory to LDS, and S^T of a tile or half a
// tile that lies there.  For the dense and block-sparse kernels and for those of the paged cache.
#pragma once
#include <float.h>

#include "pkh3_common.h"

namespace pkh3 {

constexpr float kRescaleSlack = 8.0f;  // the running max is only raised when exceeded by 2^8
// The running max before the first key.  Finite: keys whose logits are all -inf then weigh exp2(-inf - max) = 0, wherever
// among a wave's keys they lie, and two shares without a key meet as exp2(0) times a row sum of 0.
constexpr float kNoMax = -FLT_MAX;

#define PKH3_SGB(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)
// Each tile loop ends on an MFMA into the O^T accumulators.  The compiler was seen to place the register
// copies that merge the two loop variants (v_mov_b64 reading the accumulator's last registers) four scalar
// instructions after that MFMA, before its result is written back; the block-sparse kernel then returned a stale
// O^T block.  32 idle issue cycles after every loop let the last MFMA retire whatever follows.  The accumulators
// are operands of the statement, so every read or copy of them the compiler emits after the loop is ordered
// after the idle cycles.
#define PKH3_MFMA_DRAIN(W)                                                                                               \
  asm volatile("s_nop 15\n\ts_nop 15"                                                                                    \
               : "+v"((W).o[0][0]), "+v"((W).o[0][1]), "+v"((W).o[1][0]), "+v"((W).o[1][1]), "+v"((W).o[2][0]),          \
                 "+v"((W).o[2][1]), "+v"((W).o[3][0]), "+v"((W).o[3][1]), "+v"((W).o[4][0]), "+v"((W).o[4][1]),          \
                 "+v"((W).o[5][0]), "+v"((W).o[5][1]), "+v"((W).o[6][0]), "+v"((W).o[6][1]), "+v"((W).o[7][0]),          \
                 "+v"((W).o[7][1])::"memory")
constexpr int kSgMfma = 0x008, kSgDsRead = 0x100;

__device__ __forceinline__ void lds_dma16(const char* g, unsigned lane_off, char* l) {
  // 64 lanes x 16 B, global -> LDS without passing through VGPRs: lane i copies g[lane_off_i .. +16) to
  // l + i*16.  `g` and `l` are wave-uniform (the address arithmetic stays on the scalar unit), `lane_off` is
  // the per-lane byte offset.
  // Issued through inline assembly on purpose: once the compiler sees a direct-to-LDS load it stops trusting
  // the in-order LDS counter and turns every later wait on an LDS read into lgkmcnt(0), which serialises the
  // operand image reads.  Completion is tracked by hand: the s_waitcnt vmcnt(0) at the top of each tile loop.
  const unsigned lds_addr = (unsigned)(size_t)(__attribute__((address_space(3))) char*)l;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(lane_off), "s"(g), "s"(lds_addr)
               : "memory", "m0");
}

// Wave-uniform reads of tables earlier kernels wrote (tile lists, fp8 scales): through the scalar cache, so
// they count on lgkmcnt and never make the wave wait for its outstanding HBM->LDS copies (vmcnt).
template <typename T>
__device__ __forceinline__ T uniform_load(const T* p, int i) {
  return ((const __attribute__((address_space(4))) T*)p)[i];
}

// Per-wave state.  Lane (c = l % 16, g = l / 16) works for the two queries 16*qb + c, qb = 0, 1, of the wave's 32.
template <bool FP8>
struct WaveState {
  bf16x8 qf[FP8 ? 1 : 2][FP8 ? 1 : 4];  // bf16 Q images (qb, ks): Q'[16*qb + c][32*ks + 8*g + j]
  i32x8 q8[FP8 ? 2 : 1];                // fp8 Q images (qb): bytes 8*ks + j = element 32*ks + 8*g + j
  f32x4 s[4][2];                        // S^T of the tile (kb, qb): keys 16*kb + 4*g + i
  f32x4 o[8][2];                        // O^T accumulators (db, qb): head-dim rows 16*db + 4*g + i
  bf16x8 vf[8];                         // V images of the first 32 keys, fetched while QK^T finishes
  float m[2], l[2];                     // per query block: running row max (scaled, log2 domain), this lane group's row sum
  int qe;                               // fp8 with power-of-two scales: exponent byte (E8M0) of the Q block's scale
};

// Consecutive MFMAs share an operand where they can: the two query blocks of an image come in turn (0 1, 1 0, 0 1 ..), so that only
// one of the operands changes from one to the next.  Less toggles in the matrix unit, at a clock that is set by power: 480p 19.82 ->
// 19.66 ms, 768p 130.1 -> 128.9, 14,830 + 512 rows 2,149 -> 2,138 us, with the projection's GEMMs (the same) a block of them 3,168 -> 3,145
// (means of two comparisons on one card); fp8 and short calls the same.
#define PKH3_MFMA16(A, B, C) __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, B, C, 0, 0, 0)
// format codes 0/0 = e4m3 x e4m3; scale operands 0 select the unscaled form of the instruction
#define PKH3_MFMA16_F8(A, B, C) __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, C, 0, 0, 0, 0, 0, 0)
// the scaled form: the product is multiplied by 2^(EA - 127) * 2^(EB - 127), EA / EB = byte 0 of each lane's scale
// operand (every lane passes the same exponents: one scale per 64-row block, not per 32 elements)
#define PKH3_MFMA16_F8S(A, B, C, EA, EB) __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, C, 0, 0, 0, EA, 0, EB)

// S^T = K' Q'^T for the 64 keys of one tile: image i of the K tile is (half, ks, kb2) = (i >> 3, (i >> 1) & 3, i & 1)
// and feeds the two query blocks, so four accumulators rotate inside each half.  LDS reads run 8 images ahead of
// the MFMAs that consume them; the tail of the MFMA chain covers the first V image reads.
// LEAN (three waves per SIMD, 168 VGPRs): the reads run only 4 images ahead and V is left to the P.V loop.
// AHEAD: images the LEAN reads run ahead (the copies of the loop that run once per workgroup take 2 and fit the registers)
// POW2 (fp8): the block scales are powers of two and go into the MFMA as its scale operands (`ke`: exponent byte of
// this K tile's scale), so S^T leaves the MFMA dequantised.
// MASKED (lean bf16 form): the sums start from -inf instead of 0 for keys from `lim` on, which costs the softmax nothing.
template <bool FP8, bool LEAN, int AHEAD = 4, bool POW2 = false, bool MASKED = false>
__device__ __forceinline__ void qk_tile(WaveState<FP8>& w, const char* kbuf, const char* vbuf, int lane, int ke = 0, int lim = 0) {
  static_assert(!MASKED || (!FP8 && LEAN), "the forms that ask for it");
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (MASKED) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.s[kb][0][i] = w.s[kb][1][i] = 16 * kb + 4 * (lane >> 4) + i >= lim ? -INFINITY : 0.f;
  }
  if constexpr (!FP8 && LEAN) {
    bf16x8 kf[16];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) kf[i] = *(const bf16x8*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int ks = (i >> 1) & 3, kb = 2 * (i >> 3) + (i & 1);
#pragma unroll
      for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.s[kb][qb] = PKH3_MFMA16(kf[i], w.qf[qb][ks], ks == 0 && !MASKED ? zero : w.s[kb][qb]);
      if (i + AHEAD < 16) kf[i + AHEAD] = *(const bf16x8*)(kbuf + ((i + AHEAD) * 64 + lane) * 16);
    }
    PKH3_SGB(kSgDsRead, AHEAD);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      PKH3_SGB(kSgMfma, 2);
      if (i + AHEAD < 16) PKH3_SGB(kSgDsRead, 1);
    }
  } else if constexpr (!FP8) {
    bf16x8 kf[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[i] = *(const bf16x8*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int ks = (i >> 1) & 3, kb = 2 * (i >> 3) + (i & 1);
#pragma unroll
      for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.s[kb][qb] = PKH3_MFMA16(kf[i], w.qf[qb][ks], ks == 0 ? zero : w.s[kb][qb]);
      if (i < 8)
        kf[i + 8] = *(const bf16x8*)(kbuf + ((i + 8) * 64 + lane) * 16);
      else
        w.vf[i - 8] = *(const bf16x8*)(vbuf + ((i - 8) * 64 + lane) * 16);
    }
    PKH3_SGB(kSgDsRead, 8);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      PKH3_SGB(kSgMfma, 2);
      PKH3_SGB(kSgDsRead, 1);
    }
  } else {
    i32x4 kc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) kc[i] = *(const i32x4*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const i32x4 a0 = kc[2 * kb], a1 = kc[2 * kb + 1];
      const i32x8 a = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
        w.s[kb][qb] = POW2 ? PKH3_MFMA16_F8S(a, w.q8[qb], zero, ke, w.qe) : PKH3_MFMA16_F8(a, w.q8[qb], zero);
      // the MFMA chain covers the first V image reads: 8 images, or 4 where registers are short (LEAN)
      if constexpr (LEAN) {
        w.vf[kb] = *(const bf16x8*)(vbuf + (kb * 64 + lane) * 16);
      } else {
        w.vf[2 * kb] = *(const bf16x8*)(vbuf + ((2 * kb) * 64 + lane) * 16);
        w.vf[2 * kb + 1] = *(const bf16x8*)(vbuf + ((2 * kb + 1) * 64 + lane) * 16);
      }
    }
  }
}

// ---- 32-key half tiles: the short-key form of the dense kernel, phase 2 of the block-sparse one ----
// S^T (32 keys x 32 queries) into w.s[AT..AT + 1]; kbuf/vbuf point at this half's K images (8 bf16 / 4 fp8 chunks)
// and V images (8).
// LEAN (three waves per SIMD): the K reads run 4 images ahead and only the fp8 path prefetches V (4 images).
template <bool FP8, bool LEAN = false, bool POW2 = false, int AT = 0>
__device__ __forceinline__ void qk_half(WaveState<FP8>& w, const char* kbuf, const char* vbuf, int lane, int ke = 0) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (!FP8 && LEAN) {
    bf16x8 kf[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) kf[i] = *(const bf16x8*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.s[AT + (i & 1)][qb] = PKH3_MFMA16(kf[i], w.qf[qb][i >> 1], i < 2 ? zero : w.s[AT + (i & 1)][qb]);
      if (i + 4 < 8) kf[i + 4] = *(const bf16x8*)(kbuf + ((i + 4) * 64 + lane) * 16);
    }
  } else if constexpr (!FP8) {
    bf16x8 kf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[i] = *(const bf16x8*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int q = 0, qb = i & 1; q < 2; ++q, qb ^= 1) w.s[AT + (i & 1)][qb] = PKH3_MFMA16(kf[i], w.qf[qb][i >> 1], i < 2 ? zero : w.s[AT + (i & 1)][qb]);
      w.vf[i] = *(const bf16x8*)(vbuf + (i * 64 + lane) * 16);
    }
  } else {
    i32x4 kc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kc[i] = *(const i32x4*)(kbuf + (i * 64 + lane) * 16);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const i32x4 a0 = kc[2 * kb], a1 = kc[2 * kb + 1];
      const i32x8 a = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
        w.s[AT + kb][qb] = POW2 ? PKH3_MFMA16_F8S(a, w.q8[qb], zero, ke, w.qe) : PKH3_MFMA16_F8(a, w.q8[qb], zero);
#pragma unroll
      for (int i = 0; i < (LEAN ? 2 : 4); ++i) {
        const int v = (LEAN ? 2 : 4) * kb + i;
        w.vf[v] = *(const bf16x8*)(vbuf + (v * 64 + lane) * 16);
      }
    }
  }
}

}  // namespace pkh3
