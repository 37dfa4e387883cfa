// Shared pieces of the MXFP4 kernels (mxfp4_ops.hip, gemm_mxfp4.hip).
#pragma once
#include "common.h"

namespace {

typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));

// where the scale byte of (row, block j of the row) lies; kt = tiles of 8 blocks along K
__device__ __forceinline__ int64_t mxfp4_scale_at(int64_t row, int j, int kt) {
  const int r = (int)(row & 127);
  return ((row >> 7) * kt + (j >> 3)) * 1024 + (j & 3) * 256 + (r >> 3) * 16 + ((j >> 2) & 1) * 8 + (r & 7);
}

// the e8m0 byte of a block whose largest magnitude has the float bits `amax`
__device__ __forceinline__ uint32_t mxfp4_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = (int)((amax + 0x200000u) >> 23) - 2;   // biased by 127
  return (uint32_t)min(max(e, 0), 252);
}

__device__ __forceinline__ uint32_t mxfp4_code(float y) {
  const float a = fabsf(y);
  const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c | (__float_as_uint(y) >> 31 << 3);
}

// eight values of a block -> their codes (lowest nibble first) and the block's scale byte
__device__ __forceinline__ uint32_t mxfp4_encode8(const float* f, uint32_t amax, uint32_t& codes) {
  const uint32_t e8 = mxfp4_scale(amax);
  codes = 0;
  if (e8 != 255u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) codes |= mxfp4_code(ldexpf(f[i], 127 - (int)e8)) << (4 * i);
  }
  return e8;
}

__device__ __forceinline__ float mxfp4_value(uint32_t code) {
  const uint32_t m = code & 7u;
  const float a = m < 4u ? 0.5f * (float)m : (m == 4u ? 2.f : m == 5u ? 3.f : m == 6u ? 4.f : 6.f);
  return (code & 8u) ? -a : a;
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
