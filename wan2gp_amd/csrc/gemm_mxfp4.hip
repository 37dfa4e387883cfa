// Linear on MXFP4 operands for gfx950: C[M, N] = epilogue(A W^T + bias), A and W as wan_mxfp4_quantize leaves them, fp32 accumulation on
// v_mfma_scale_f32_16x16x128_f8f6f4 (which applies both blocks' scales itself), bf16 out.
//
// A lane (n = lane & 15, g = lane >> 4) of the instruction supplies row n, values 32 g .. 32 g + 31 of its 128 -- one block, 16 bytes, one scale
// byte.  A k-stage is 256 values = 128 bytes of a row = 8 blocks; step ks of it takes blocks 4 ks + g.
// Row r of a 128-row panel is lane row n = r >> 3 of tile t = r & 7, for both operands: a lane then owns the 8 consecutive columns 8 n .. 8 n + 7 of
// the output (one 16-byte store), and 8 consecutive rows' scales.
#include "mxfp4.h"

namespace {

typedef int mx_i8 __attribute__((ext_vector_type(8)));

// ---- the general kernel: any M and N, K % 32 == 0; 128 x 128 tiles, 4 waves of 64 x 64 -----------------------------------------------------
template <int EPI>   // WAN_EPI_TRANSPOSED: the bias runs along the rows
__global__ __launch_bounds__(256) void gemm_mxfp4_kernel(MxGemm p) {
  __shared__ __attribute__((aligned(16))) char smem[2][2][128 * 144];   // [stage][operand], rows of 128 B at a pitch of 144 B
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int wy = wave >> 1, wx = wave & 1;
  const int tx = (int)((p.N + 127) / 128), id = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t y0 = (int64_t)(id / tx) * 128, x0 = (int64_t)(id % tx) * 128;
  const int pitch = p.K / 2;
  mx_u4 ra[4], rw[4];
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = i * 256 + tid, row = q >> 3, c = s * 128 + (q & 7) * 16;
      ra[i] = rw[i] = mx_u4{0, 0, 0, 0};
      if (c < pitch) {
        ra[i] = *reinterpret_cast<const mx_u4*>(p.A + min(y0 + row, p.M - 1) * pitch + c);
        rw[i] = *reinterpret_cast<const mx_u4*>(p.W + min(x0 + row, p.N - 1) * pitch + c);
      }
    }
  };
  auto store = [&](int st) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = i * 256 + tid;
      *reinterpret_cast<mx_u4*>(&smem[st][0][(q >> 3) * 144 + (q & 7) * 16]) = ra[i];
      *reinterpret_cast<mx_u4*>(&smem[st][1][(q >> 3) * 144 + (q & 7) * 16]) = rw[i];
    }
  };
  f32x4 acc[4][4] = {};
  load(0);
  for (int s = 0; s < p.kt; ++s) {
    store(s & 1);
    __syncthreads();
    if (s + 1 < p.kt) load(s + 1);
    const char* sa = smem[s & 1][0];
    const char* sw = smem[s & 1][1];
    const int64_t at = (int64_t)s * 1024 + (g * 16 + n) * 16;
    const mx_u4 qa = *reinterpret_cast<const mx_u4*>(p.As + (y0 >> 7) * p.kt * 1024 + at);
    const mx_u4 qw = *reinterpret_cast<const mx_u4*>(p.Ws + (x0 >> 7) * p.kt * 1024 + at);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      mx_i8 fa[4] = {}, fw[4] = {};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        // tile t of the wave's half of the panel: rows 8 n + 4 half + t
        const mx_u4 a = *reinterpret_cast<const mx_u4*>(sa + (8 * n + 4 * wy + t) * 144 + (4 * ks + g) * 16);
        const mx_u4 w = *reinterpret_cast<const mx_u4*>(sw + (8 * n + 4 * wx + t) * 144 + (4 * ks + g) * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) { fa[t][k] = (int)a[k]; fw[t][k] = (int)w[k]; }
      }
      const int sca = (int)qa[2 * ks + wy], scw = (int)qw[2 * ks + wx];   // byte t: tile t of this half
#define MX_ROW(T)                                                                                                                        \
  acc[T][0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa[T], fw[0], acc[T][0], 4, 4, T, sca, 0, scw);                            \
  acc[T][1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa[T], fw[1], acc[T][1], 4, 4, T, sca, 1, scw);                            \
  acc[T][2] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa[T], fw[2], acc[T][2], 4, 4, T, sca, 2, scw);                            \
  acc[T][3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa[T], fw[3], acc[T][3], 4, 4, T, sca, 3, scw);
      MX_ROW(0) MX_ROW(1) MX_ROW(2) MX_ROW(3)
#undef MX_ROW
    }
  }
  // lane (n, g), tile (a, w), register i: row 8 (4 g + i) + 4 wy + a, column 8 n + 4 wx + w
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t y = y0 + 8 * (4 * g + i) + 4 * wy + a;
      if (y >= p.M) continue;
      const int64_t bidx = EPI == WAN_EPI_GATE_RES && p.gate_idx >= 0 ? y / p.rows_per_batch : 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int64_t x = x0 + 8 * n + 4 * wx + w;
        if (x >= p.N) continue;
        float o = acc[a][w][i];
        if (p.bias != nullptr) o += bf2f(p.bias[EPI == WAN_EPI_TRANSPOSED ? y : x]);
        if (EPI == WAN_EPI_GELU_TANH) o = mx_gelu_tanh(o);
        if (EPI == WAN_EPI_GATE_RES) {
          float gate = 1.f;
          if (p.gate_idx >= 0) gate = bf2f(p.mod[(int64_t)p.gate_idx * p.N + x]) + bf2f(p.e[(bidx * p.n_mod + p.gate_idx) * p.N + x]);
          o = __builtin_fmaf(o, gate, bf2f(p.R[y * p.ldc + x]));
        }
        p.C[y * p.ldc + x] = f2bf(o);
      }
    }
}

}  // namespace

int wan_gemm_mxfp4m_try(const MxGemm& p, int epilogue, hipStream_t st);   // gemm_mxfp4m.hip

extern "C" int64_t wan_gemm_mxfp4_scratch_bytes(int64_t M, int N, int K, int epilogue) { return 0; }

extern "C" int wan_gemm_mxfp4(const uint8_t* A, const uint8_t* a_scales, const uint8_t* W, const uint8_t* w_scales, const wan_bf16* bias, wan_bf16* C, int64_t ldc, int64_t M, int N, int K,
                              int epilogue, const wan_bf16* R, const wan_bf16* mod, const wan_bf16* e, int n_mod, int gate_idx, int64_t rows_per_batch, void* scratch, int64_t scratch_bytes,
                              void* stream) {
  WAN_REQUIRE(A && a_scales && W && w_scales && C, "wan_gemm_mxfp4: null operand");
  WAN_REQUIRE(M >= 1 && N >= 1 && K >= 32 && K % 32 == 0, "wan_gemm_mxfp4: M=%lld and N=%d must be positive, K=%d a positive multiple of 32", (long long)M, N, K);
  WAN_REQUIRE((((uintptr_t)A | (uintptr_t)a_scales | (uintptr_t)W | (uintptr_t)w_scales | (uintptr_t)C) & 15) == 0, "wan_gemm_mxfp4: pointers must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  const bool tr = epilogue == WAN_EPI_TRANSPOSED;
  WAN_REQUIRE(ldc >= (tr ? M : N), "wan_gemm_mxfp4: ldc=%lld is smaller than a row of the output", (long long)ldc);
  MxGemm p = {tr ? W : A, tr ? w_scales : a_scales, tr ? A : W, tr ? a_scales : w_scales, tr ? N : M, tr ? M : N, K, (K + 255) / 256, bias, C, ldc, R, mod, e, n_mod, gate_idx, rows_per_batch > 0 ? rows_per_batch : 1};
  if (epilogue == WAN_EPI_GATE_RES) {
    WAN_REQUIRE(R != nullptr, "wan_gemm_mxfp4: GATE_RES needs the residual R");
    WAN_REQUIRE(gate_idx < 0 || (mod && e && gate_idx < n_mod && rows_per_batch > 0), "wan_gemm_mxfp4: bad gate args");
  }
  WAN_REQUIRE(epilogue >= WAN_EPI_NONE && epilogue <= WAN_EPI_TRANSPOSED, "wan_gemm_mxfp4: unknown epilogue %d", epilogue);
  const int rc = wan_gemm_mxfp4m_try(p, epilogue, st);
  if (rc >= 0) return rc;
  const int64_t tiles = ((p.M + 127) / 128) * ((p.N + 127) / 128);
  WAN_REQUIRE(tiles < ((int64_t)1 << 31), "wan_gemm_mxfp4: grid too large");
  const dim3 grid((unsigned)tiles), wg(256);
  switch (epilogue) {
    case WAN_EPI_NONE: hipLaunchKernelGGL(gemm_mxfp4_kernel<WAN_EPI_NONE>, grid, wg, 0, st, p); break;
    case WAN_EPI_GELU_TANH: hipLaunchKernelGGL(gemm_mxfp4_kernel<WAN_EPI_GELU_TANH>, grid, wg, 0, st, p); break;
    case WAN_EPI_GATE_RES: hipLaunchKernelGGL(gemm_mxfp4_kernel<WAN_EPI_GATE_RES>, grid, wg, 0, st, p); break;
    default: hipLaunchKernelGGL(gemm_mxfp4_kernel<WAN_EPI_TRANSPOSED>, grid, wg, 0, st, p); break;
  }
  WAN_LAUNCH_CHECK();
  return 0;
}
