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

// One wave per 8 rows x 256 columns: four 16-byte loads per lane (two whole rows of 512 bytes a load), four lanes to a block, its maximum through two
// quad exchanges.  The 64 scale bytes are 8 consecutive ones for each block of the tile: lanes l and l + 32 hold the even and the odd rows, one
// exchange makes them dwords.  75,600 x 5,120: 183 us = 5.3 TB/s of rows, codes and scales (byte stores and comparisons against the grid: 329 us).
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const bf16_t* __restrict__ x, int64_t row_stride, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t M, int K,
                                                         int kt, int64_t groups) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane & 31, hi = lane >> 5;
  const int64_t r8 = w / kt;                              // group of 8 rows
  const int s = (int)(w - r8 * kt);                       // tile along K
  if (r8 >= groups) return;                               // (whole waves)
  const int col = s * 256 + c * 8;
  const bool in = col < K;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r8 * 8 + 2 * i + hi;
    v[i] = make_uint4(0, 0, 0, 0);
    if (in && row < M) v[i] = *reinterpret_cast<const uint4*>(x + row * row_stride + col);
  }
  uint32_t e8[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r8 * 8 + 2 * i + hi;
    float f[8];
    unpack8(v[i], f);
    uint32_t a = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) a = max(a, __float_as_uint(f[k]) & 0x7fffffffu);
    a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true));   // quad_perm [1, 0, 3, 2]
    a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4e, 0xf, 0xf, true));   // quad_perm [2, 3, 0, 1]
    const uint32_t e = mxfp4_scale(a);
    e8[i] = in && row < M ? e : 0u;
    if (in && row < M) codes[(row * K + col) / 8] = mxfp4_encode8(f, e);
  }
  const uint32_t own = e8[0] | e8[1] << 8 | e8[2] << 16 | e8[3] << 24;
  const uint32_t other = (uint32_t)__shfl_xor((int)own, 32, 64);
  const uint32_t even = hi ? other : own, odd = hi ? own : other;
  // rows 0 .. 3 from the lower lane, 4 .. 7 from the upper one
  const uint32_t word = hi ? __builtin_amdgcn_perm(odd, even, 0x07030602u) : __builtin_amdgcn_perm(odd, even, 0x05010400u);
  const int j = c >> 2;
  if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(scales + ((r8 >> 4) * kt + s) * 1024 + (j & 3) * 256 + (r8 & 15) * 16 + (j >> 2) * 8 + hi * 4) = word;
}

__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, bf16_t* __restrict__ out, int64_t M, int K, int kt,
                                                           int64_t groups) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane & 31, hi = lane >> 5, j = c >> 2;
  const int64_t r8 = w / kt;
  const int s = (int)(w - r8 * kt);
  const int col = s * 256 + c * 8;
  if (r8 >= groups || col >= K) return;
  const uint2 e = *reinterpret_cast<const uint2*>(scales + ((r8 >> 4) * kt + s) * 1024 + (j & 3) * 256 + (r8 & 15) * 16 + (j >> 2) * 8);   // the eight rows' scales
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r8 * 8 + 2 * i + hi;
    q[i] = row < M ? codes[(row * K + col) / 8] : 0u;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r8 * 8 + 2 * i + hi;
    const uint32_t e8 = (i < 2 ? e.x : e.y) >> (16 * (i & 1) + 8 * hi) & 255u;
    float f[8];
    mxfp4_decode8(q[i], e8, f);
    if (row < M) *reinterpret_cast<uint4*>(out + row * K + col) = pack8(f);
  }
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
  const int64_t groups = (M + 127) / 128 * 16, wgs = (groups * kt + 3) / 4;   // (the padding rows' scales are written too)
  WAN_REQUIRE(wgs < ((int64_t)1 << 31), "wan_mxfp4_quantize: grid too large");
  hipLaunchKernelGGL(mxfp4_quant_kernel, dim3((unsigned)wgs), dim3(256), 0, as_stream(stream), x, row_stride, reinterpret_cast<uint32_t*>(codes), scales, M, K, kt, groups);
  WAN_LAUNCH_CHECK();
  return 0;
}

extern "C" int wan_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, wan_bf16* out, int64_t M, int K, void* stream) {
  WAN_REQUIRE(codes && scales && out, "wan_mxfp4_dequantize: null pointer");
  WAN_REQUIRE(M >= 1 && K >= 32 && K % 32 == 0, "wan_mxfp4_dequantize: M=%lld must be positive, K=%d a positive multiple of 32", (long long)M, K);
  WAN_REQUIRE((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15) == 0, "wan_mxfp4_dequantize: pointers must be 16-byte aligned");
  const int kt = (K + 255) / 256;
  const int64_t groups = (M + 7) / 8, wgs = (groups * kt + 3) / 4;
  WAN_REQUIRE(wgs < ((int64_t)1 << 31), "wan_mxfp4_dequantize: grid too large");
  hipLaunchKernelGGL(mxfp4_dequant_kernel, dim3((unsigned)wgs), dim3(256), 0, as_stream(stream), reinterpret_cast<const uint32_t*>(codes), scales, out, M, K, kt, groups);
  WAN_LAUNCH_CHECK();
  return 0;
}
