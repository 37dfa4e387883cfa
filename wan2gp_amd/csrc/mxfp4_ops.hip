// Microscaled 4-bit floating point (OCP MX: e2m1 elements, one power of two per 32 of them) for gfx950: quantisation and expansion.  The product is
// gemm_mxfp4.hip's.
//
// A block is 32 consecutive values of a row.  Its scale 2^e: e = floor(log2 amax) - 2, one more where amax >= 1.75 of its power of two -- the grid
// ends at 6, so without that step everything from 7 up (an eighth of all block maxima) would be cut by up to a quarter of its value.  Elements are
// rounded to nearest even onto 0, .5, 1, 1.5, 2, 3, 4, 6.  e is kept in [-127, 125] (at 126 a 4 would stand for 2^128).  A block that holds an inf or
// a NaN gets the scale byte 255, NaN: it has to show in the product.
//
// codes  [rows][K / 2] bytes, the even element in the low nibble.
// scales in the order in which the matrix instruction's lanes want them: tiles of 128 rows x 8 blocks (256 values of K), 1,024 bytes each, row tiles
//        outside; inside a tile the byte of row r, block j lies at [j & 3][r >> 3][j >> 2][r & 7].  A lane (row group n, block group g) of
//        gemm_mxfp4.hip then has all its scales of a k-stage -- eight rows, two blocks -- in ONE 16-byte load.  Bytes past the matrix are 0.
#include "mxfp4.h"

namespace {

// Four lanes share a block: 16-byte loads of 8 values that are contiguous across the wave (a lane of its own per block would read 64-byte runs at a
// stride of 64).
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const bf16_t* __restrict__ x, int64_t row_stride, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t M, int K,
                                                         int kt /* tiles along K */) {
  const int nb = kt * 8;                                  // blocks of a row, the padding included
  const int64_t t = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2);
  const int64_t row = t / nb;
  const int j = (int)(t - row * nb), part = threadIdx.x & 3;
  if (row >= (M + 127) / 128 * 128) return;               // (whole groups of four lanes)
  const bool live = row < M && j * 32 < K;
  uint32_t e8 = 0;
  if (live) {
    float f[8];
    unpack8(*reinterpret_cast<const uint4*>(x + row * row_stride + j * 32 + part * 8), f);
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(f[i]) & 0x7fffffffu);
    a = max(a, (uint32_t)__shfl_xor((int)a, 1, 64));
    a = max(a, (uint32_t)__shfl_xor((int)a, 2, 64));
    uint32_t c;
    e8 = mxfp4_encode8(f, a, c);
    codes[(row * K + j * 32) / 8 + part] = c;
  }
  if (part == 0) scales[mxfp4_scale_at(row, j, kt)] = (uint8_t)e8;
}

__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, bf16_t* __restrict__ out, int64_t M, int K, int kt) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // eight values
  const int per = K / 8;
  const int64_t row = i / per;
  if (row >= M) return;
  const int c = (int)(i - row * per);
  const uint32_t w = codes[i];
  const uint32_t e8 = scales[mxfp4_scale_at(row, c >> 2, kt)];
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = e8 == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(mxfp4_value((w >> (4 * k)) & 15u), (int)e8 - 127);
  *reinterpret_cast<uint4*>(out + i * 8) = pack8(f);
}

}  // namespace

extern "C" int64_t wan_mxfp4_scale_bytes(int64_t rows, int64_t K) {
  if (rows < 1 || K < 1) return 0;
  return (rows + 127) / 128 * ((K + 255) / 256) * 1024;
}

extern "C" int wan_mxfp4_quantize(const wan_bf16* x, int64_t row_stride, uint8_t* codes, uint8_t* scales, int64_t M, int K, void* stream) {
  WAN_REQUIRE(x && codes && scales, "wan_mxfp4_quantize: null pointer");
  WAN_REQUIRE(M >= 1 && K >= 32 && K % 32 == 0, "wan_mxfp4_quantize: M=%lld must be positive, K=%d a positive multiple of 32", (long long)M, K);
  WAN_REQUIRE(row_stride >= K && row_stride % 8 == 0, "wan_mxfp4_quantize: the row stride %lld must be a multiple of 8 elements, at least K", (long long)row_stride);
  WAN_REQUIRE((((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) == 0, "wan_mxfp4_quantize: pointers must be 16-byte aligned");
  const int kt = (K + 255) / 256;
  const int64_t blocks = (M + 127) / 128 * 128 * kt * 8;
  WAN_REQUIRE(blocks / 64 < ((int64_t)1 << 31), "wan_mxfp4_quantize: grid too large");
  hipLaunchKernelGGL(mxfp4_quant_kernel, dim3((unsigned)(blocks / 64)), dim3(256), 0, as_stream(stream), x, row_stride, reinterpret_cast<uint32_t*>(codes), scales, M, K, kt);
  WAN_LAUNCH_CHECK();
  return 0;
}

extern "C" int wan_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, wan_bf16* out, int64_t M, int K, void* stream) {
  WAN_REQUIRE(codes && scales && out, "wan_mxfp4_dequantize: null pointer");
  WAN_REQUIRE(M >= 1 && K >= 32 && K % 32 == 0, "wan_mxfp4_dequantize: M=%lld must be positive, K=%d a positive multiple of 32", (long long)M, K);
  WAN_REQUIRE((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15) == 0, "wan_mxfp4_dequantize: pointers must be 16-byte aligned");
  const int64_t n = (M * (K / 8) + 255) / 256;
  WAN_REQUIRE(n < ((int64_t)1 << 31), "wan_mxfp4_dequantize: grid too large");
  hipLaunchKernelGGL(mxfp4_dequant_kernel, dim3((unsigned)n), dim3(256), 0, as_stream(stream), reinterpret_cast<const uint32_t*>(codes), scales, out, M, K, (K + 255) / 256);
  WAN_LAUNCH_CHECK();
  return 0;
}
