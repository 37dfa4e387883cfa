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

__device__ __forceinline__ float mx_gelu_tanh(float x) {
  const float c = -2.0f * 0.7978845608028654f * 1.4426950408889634f;  // -2 sqrt(2/pi) log2(e)
  const float t = __builtin_fmaf(x * x, 0.044715f, 1.0f);
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * t * c));
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
