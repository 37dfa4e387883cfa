// Shared pieces of the MXFP4 kernels (mxfp4_ops.hip, gemm_mxfp4.hip).
#pragma once
#include "common.h"

namespace {

typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));

// the e8m0 byte of a block whose largest magnitude has the float bits `amax`
__device__ __forceinline__ uint32_t mxfp4_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = (int)((amax + 0x200000u) >> 23) - 2;   // biased by 127
  return (uint32_t)min(max(e, 0), 252);
}

// eight values of a block with scale byte e8 -> their codes, the first in the lowest nibble.  v_cvt_scalef32_pk_fp4_f32 rounds to nearest even and
// stops at 6 (checked for every bf16 value); the scale is applied by v_ldexp in front of it, which is exact over the whole exponent range.
__device__ __forceinline__ uint32_t mxfp4_encode8(const float* f, uint32_t e8) {
  if (e8 == 255u) return 0u;
  const int sh = 127 - (int)e8;
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, ldexpf(f[0], sh), ldexpf(f[1], sh), 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, ldexpf(f[2], sh), ldexpf(f[3], sh), 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, ldexpf(f[4], sh), ldexpf(f[5], sh), 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, ldexpf(f[6], sh), ldexpf(f[7], sh), 1.0f, 3);
  return c;
}
// the values they stand for
__device__ __forceinline__ void mxfp4_decode8(uint32_t c, uint32_t e8, float* f) {
  const int sh = (int)e8 - 127;
#define MX_PAIR(B)                                                             \
  {                                                                            \
    const wan_f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, B);  \
    f[2 * B] = e8 == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(v[0], sh);   \
    f[2 * B + 1] = e8 == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(v[1], sh); \
  }
  MX_PAIR(0) MX_PAIR(1) MX_PAIR(2) MX_PAIR(3)
#undef MX_PAIR
}

// D += A B over 128 values with both blocks' scales; T, U: the bytes of sy, sx.  Accumulators pinned to the accumulator file (builtin MFMAs had them copied
// back and forth: 92 register moves a stage of 32 MFMAs)
template <int T, int U>
__device__ __forceinline__ void mfma_mx(f32x4& acc, const mx_u4& ya, const mx_u4& xb, uint32_t sy, uint32_t sx) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
               : "+a"(acc)
               : "v"(ya), "v"(xb), "v"(sy), "v"(sx), "n"(T & 1), "n"(U & 1), "n"(T >> 1), "n"(U >> 1));
}
// One LDS-DMA piece (16 bytes a lane, 1 KB a wave) as inline asm: hipcc's waitcnt pass does not see it, completion is counted by hand
__device__ __forceinline__ void mx_dma16(uint32_t voff, const mx_u4& rsrc, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ mx_u4 mx_rsrc(const char* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)base;
  mx_u4 r;
  r[0] = (uint32_t)b;
  r[1] = (uint32_t)(b >> 32) & 0xffffu;  // stride 0
  r[2] = bytes;                          // beyond: zeros
  r[3] = 0x00020000u;
  return r;
}

__device__ __forceinline__ float mx_gelu_tanh(float x) {
  const float c = -2.0f * 0.7978845608028654f * 1.4426950408889634f;  // -2 sqrt(2/pi) log2(e)
  const float t = __builtin_fmaf(x * x, 0.044715f * c, c);
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * t));
}

}  // namespace

// a product's operands as the kernels see them: Y = the rows of the output, X = its columns (the transposed form: weights, tokens)
struct MxGemm {
  const uint8_t *A, *As, *W, *Ws;
  int64_t M, N;
  int K, kt;
  const bf16_t* bias;
  bf16_t* C;
  int64_t ldc;
  const bf16_t *R, *mod, *e;
  int n_mod, gate_idx;
  int64_t rows_per_batch;
};
