// Linear on MXFP4 operands for gfx950: C[M, N] = epilogue(A W^T + bias), A and W as wan_mxfp4_quantize leaves them, fp32 accumulation on
// v_mfma_scale_f32_16x16x128_f8f6f4 (which applies both blocks' scales itself), bf16 out.
//
// A lane (n = lane & 15, g = lane >> 4) of the instruction supplies row n, values 32 g .. 32 g + 31 of its 128 -- one block, 16 bytes, one scale
// byte.  A k-stage is 256 values = 128 bytes of a row = 8 blocks; step ks of it takes blocks 4 ks + g.
// Row r of a 128-row panel is lane row n = r >> 3 of tile t = r & 7, for both operands: a lane then owns the 8 consecutive columns 8 n .. 8 n + 7 of
// the output (one 16-byte store), and 8 consecutive rows' scales.
#include "mxfp4.h"

namespace {

typedef __attribute__((address_space(3))) const char mxg_lds_cchar;
typedef __attribute__((address_space(3))) const mx_u4 mxg_lds_u4;
typedef __attribute__((address_space(3))) const uint32_t mxg_lds_u32;

constexpr int MXG_OP = 128 * 128, MXG_STAGE = 2 * MXG_OP + 2 * 1024, MXG_NST = 4;   // bytes: an operand's stage, a stage (both operands' rows and scales), ring

__device__ __forceinline__ void unpack4(const uint2& v, float* f) {
  f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
}

// the fp32 epilogue of one element at (row y, column x)
template <int EPI>
__device__ __forceinline__ bf16_t mxg_finish(const MxGemm& p, float o, int64_t y, int64_t x) {
  if (p.bias != nullptr) o += bf2f(p.bias[EPI == WAN_EPI_TRANSPOSED ? y : x]);
  if (EPI == WAN_EPI_GELU_TANH) o = mx_gelu_tanh(o);
  if (EPI == WAN_EPI_GATE_RES) {
    float gate = 1.f;
    if (p.gate_idx >= 0) gate = bf2f(p.mod[(int64_t)p.gate_idx * p.N + x]) + bf2f(p.e[(y / p.rows_per_batch * p.n_mod + p.gate_idx) * p.N + x]);
    o = __builtin_fmaf(o, gate, bf2f(p.R[y * p.ldc + x]));
  }
  return f2bf(o);
}

struct MxgFrags {
  mx_u4 y[4], x[4];
};
// MFMA m = 0 .. 15 of a k-step: y tile m >> 2, x tile m & 3
template <int M0, class F>
__device__ __forceinline__ void mxg_run(f32x4 (&acc)[4][4], const MxgFrags& f, uint32_t sy, uint32_t sx, F&& gap) {
  if constexpr (M0 < 16) {
    mfma_mx<(M0 >> 2), (M0 & 3)>(acc[M0 >> 2][M0 & 3], f.y[M0 >> 2], f.x[M0 & 3], sy, sx);
    __builtin_amdgcn_sched_barrier(0);
    gap(M0);
    __builtin_amdgcn_sched_barrier(0);
    mxg_run<M0 + 1>(acc, f, sy, sx, gap);
  }
}

// ---- any M and N, K % 32 == 0: 128 x 128 tiles, 4 waves of 64 x 64, a ring of four k-stages filled by LDS-DMA ------------------
// Rows and scales both go through the ring (gemm_mxfp4m.hip has no LDS left for the scales): every wait is counted by hand, nine pieces a stage and
// wave.  PARTS: this launch is one of several parts along K (few tiles: the CUs that have none take a part of the others' stages), and leaves its sums
// in fp32 at part [parts][M][N]; mxg_join_kernel adds them up in order.
template <int EPI, bool PARTS>
__global__ __launch_bounds__(256) void gemm_mxfp4_kernel(MxGemm p, int parts, float* __restrict__ part) {
  __shared__ __attribute__((aligned(16))) char smem[MXG_NST * MXG_STAGE];
  mxg_lds_cchar* lds = (mxg_lds_cchar*)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wy = wave >> 1, wx = wave & 1;
  // XCD-contiguous ids, then groups of eight tile rows walked column by column: what runs on an XCD at a time shares few panels of its L2
  const int ty = (int)((p.M + 127) / 128), tx = (int)((p.N + 127) / 128);
  const int wg = xcd_remap(blockIdx.x, gridDim.x);
  const int id = PARTS ? wg / parts : wg, pt = PARTS ? wg - id * parts : 0;
  const int first = id / (8 * tx) * 8, gsz = min(ty - first, 8), in_g = id - first * tx;
  const int64_t y0 = (int64_t)(first + in_g % gsz) * 128, x0 = (int64_t)(in_g / gsz) * 128;
  const int s0 = PARTS ? (int)((int64_t)p.kt * pt / parts) : 0, s1 = PARTS ? (int)((int64_t)p.kt * (pt + 1) / parts) : p.kt;
  const int pitch = p.K / 2;

  // piece i of a wave: image rows (i * 4 + wave) * 8 .. + 7, eight lanes a row; image row 16 t + n = row 8 n + t of the panel; chunk swizzle as gemm_mxfp4m.hip
  uint32_t yofs[4], xofs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (i * 256 + tid) >> 3, lch = (tid & 7) ^ ((row >> 1) & 7);
    const int r = 8 * (row & 15) + (row >> 4);
    yofs[i] = (uint32_t)(min(y0 + r, p.M - 1) - y0) * (uint32_t)pitch + lch * 16;   // past the matrix: its last row again, never stored
    xofs[i] = (uint32_t)(min(x0 + r, p.N - 1) - x0) * (uint32_t)pitch + lch * 16;
  }
  const char* yb = reinterpret_cast<const char*>(p.A) + y0 * pitch;
  const char* xb = reinterpret_cast<const char*>(p.W) + x0 * pitch;
  const uint32_t ylen = (uint32_t)min((p.M - y0) * pitch, (int64_t)0xffffff00), xlen = (uint32_t)min((p.N - x0) * pitch, (int64_t)0xffffff00);   // (a tile's reach is below 2^31)
  const char* sb = (wave & 1) ? reinterpret_cast<const char*>(p.Ws + (x0 >> 7) * p.kt * 1024) : reinterpret_cast<const char*>(p.As + (y0 >> 7) * p.kt * 1024);
  // past a row's end: the next row's codes, whose scale bytes are 0 on both sides (gemm_mxfp4m.hip); past the buffer's: zeros
  struct Fetch {
    mx_u4 y, x, s;
    uint32_t at, sat;
  };
  auto plan = [&](int s, int st) {
    Fetch f;
    f.y = mx_rsrc(yb + (uint32_t)s * 128u, ylen - (uint32_t)s * 128u);
    f.x = mx_rsrc(xb + (uint32_t)s * 128u, xlen - (uint32_t)s * 128u);
    f.s = mx_rsrc(sb + (uint32_t)s * 1024u, 1024u);
    f.at = lds0 + st + wave * 1024;
    f.sat = lds0 + st + 2 * MXG_OP + (wave & 1) * 1024;   // (waves 2, 3: the same bytes again)
    return f;
  };
  auto piece = [&](const Fetch& f, int i) {
    if (i < 4) mx_dma16(yofs[i & 3], f.y, f.at + (i & 3) * 4096);
    else if (i < 8) mx_dma16(xofs[i & 3], f.x, f.at + MXG_OP + (i & 3) * 4096);
    else mx_dma16((uint32_t)lane * 16u, f.s, f.sat);
  };
  auto fetch = [&](int s, int slot) {
    const Fetch f = plan(s, slot * MXG_STAGE);
#pragma unroll
    for (int i = 0; i < 9; ++i) piece(f, i);
  };
  // fragment addresses inside a stage: one per (operand, k-step), the tiles 2 KB apart
  uint32_t ya[2], xa[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const uint32_t ch = (uint32_t)((4 * ks + g) ^ ((n >> 1) & 7)) * 16u;
    ya[ks] = (uint32_t)((4 * wy * 16 + n) * 128) + ch;
    xa[ks] = (uint32_t)(MXG_OP + (4 * wx * 16 + n) * 128) + ch;
  }
  const uint32_t sca[2] = {(uint32_t)(2 * MXG_OP + (g * 16 + n) * 16 + wy * 4), (uint32_t)(2 * MXG_OP + 1024 + (g * 16 + n) * 16 + wx * 4)};
  auto frag = [&](MxgFrags& f, int st, int ks, int r) {
    if (r < 4) f.y[r] = *(mxg_lds_u4*)(lds + st + ya[ks] + r * 2048);
    else f.x[r - 4] = *(mxg_lds_u4*)(lds + st + xa[ks] + (r - 4) * 2048);
  };
  // the dwords of a lane's 16 scale bytes that belong to the wave's half of the panel, one per k-step (byte t: tile t)
  auto scales = [&](int st, int op, uint32_t (&q)[2]) {
    q[0] = *(mxg_lds_u32*)(lds + st + sca[op]);
    q[1] = *(mxg_lds_u32*)(lds + st + sca[op] + 8);
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
      asm volatile("" : "+a"(acc[a][b]));
    }
#pragma unroll
  for (int i = 0; i < MXG_NST; ++i) fetch(min(s0 + i, s1 - 1), i);
  asm volatile("s_waitcnt vmcnt(27)" ::: "memory");   // the first stage
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  MxgFrags f0, f1;
  uint32_t sy[2], sx[2], ny[2], nx[2];
  scales(0, 0, sy);
  scales(0, 1, sx);
#pragma unroll
  for (int r = 0; r < 8; ++r) frag(f0, 0, 0, r);
  int st = 0;
  // a stage: k-step 0's 16 MFMAs with k-step 1's fragment reads between them; then everybody has read the stage (barrier) and the next one has landed;
  // k-step 1's MFMAs with the next stage's first fragments, its scales, and the DMA of the stage four ahead into this one's place
  for (int s = s0; s < s1; ++s) {
    const int nst = st + MXG_STAGE == MXG_NST * MXG_STAGE ? 0 : st + MXG_STAGE;
    asm volatile("s_nop 1" : "+v"(sy[0]), "+v"(sy[1]), "+v"(sx[0]), "+v"(sx[1]));   // (a register copy in front of an MFMA that reads it: hipcc pads nothing around asm)
    mxg_run<0>(acc, f0, sy[0], sx[0], [&](int m) __attribute__((always_inline)) {
      if (m < 8) frag(f1, st, 1, m);
    });
    asm volatile("s_waitcnt vmcnt(18) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const Fetch fx = plan(min(s + MXG_NST, s1 - 1), st);
    mxg_run<0>(acc, f1, sy[1], sx[1], [&](int m) __attribute__((always_inline)) {
      if (m == 0) scales(nst, 0, ny);
      if (m == 1) scales(nst, 1, nx);
      if (m >= 2 && m < 10) frag(f0, nst, 0, m - 2);
      if (m < 9) piece(fx, m);
    });
    sy[0] = ny[0]; sy[1] = ny[1]; sx[0] = nx[0]; sx[1] = nx[1];
    st = nst;
  }
  // the last DMA (the LDS is released at the end); the last MFMAs -> accumulator reads
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
  // lane (n, g), tile (a, w), register i: row 8 (4 g + i) + 4 wy + a, columns 8 n + 4 wx .. + 3
  const int64_t x = x0 + 8 * n + 4 * wx;
  if (PARTS) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int a = r & 3, i = r >> 2;
      const int64_t y = y0 + 8 * (4 * g + i) + 4 * wy + a;
      if (y >= p.M || x >= p.N) continue;
      float* o = part + ((int64_t)pt * p.M + y) * p.N + x;
      if ((p.N & 3) == 0) *reinterpret_cast<float4*>(o) = make_float4(acc[a][0][i], acc[a][1][i], acc[a][2][i], acc[a][3][i]);
      else {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (x + w < p.N) o[w] = acc[a][w][i];
      }
    }
    return;
  }
  // four columns at a time where every pointer allows 8-byte accesses; what a row needs is loaded ahead of the rows' arithmetic and stores (element by
  // element, with the bias read again for each, the epilogue took 3 us of a 13-us call)
  const bool quad = x + 4 <= p.N && ((p.N | p.ldc) & 3) == 0 && (((uintptr_t)p.C | (uintptr_t)p.bias | (uintptr_t)p.R | (uintptr_t)p.mod | (uintptr_t)p.e) & 7) == 0;
  if (quad) {
    float bc[4] = {0.f, 0.f, 0.f, 0.f}, mc[4];
    if (EPI != WAN_EPI_TRANSPOSED && p.bias != nullptr) unpack4(*reinterpret_cast<const uint2*>(p.bias + x), bc);
    const bool gated = EPI == WAN_EPI_GATE_RES && p.gate_idx >= 0;
    if (gated) unpack4(*reinterpret_cast<const uint2*>(p.mod + (int64_t)p.gate_idx * p.N + x), mc);
    uint2 res[16], ec[16];
    float br[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t y = min(y0 + 8 * (4 * g + (r >> 2)) + 4 * wy + (r & 3), p.M - 1);
      if (EPI == WAN_EPI_GATE_RES) res[r] = *reinterpret_cast<const uint2*>(p.R + y * p.ldc + x);
      if (gated) ec[r] = *reinterpret_cast<const uint2*>(p.e + (y / p.rows_per_batch * p.n_mod + p.gate_idx) * p.N + x);
      if (EPI == WAN_EPI_TRANSPOSED) br[r] = p.bias != nullptr ? bf2f(p.bias[y]) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int a = r & 3, i = r >> 2;
      const int64_t y = y0 + 8 * (4 * g + i) + 4 * wy + a;
      float v[4], rv[4], ev[4];
      if (EPI == WAN_EPI_GATE_RES) unpack4(res[r], rv);
      if (gated) unpack4(ec[r], ev);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        v[w] = acc[a][w][i] + (EPI == WAN_EPI_TRANSPOSED ? br[r] : bc[w]);
        if (EPI == WAN_EPI_GELU_TANH) v[w] = mx_gelu_tanh(v[w]);
        if (EPI == WAN_EPI_GATE_RES) v[w] = __builtin_fmaf(v[w], gated ? mc[w] + ev[w] : 1.f, rv[w]);
      }
      if (y < p.M) *reinterpret_cast<uint2*>(p.C + y * p.ldc + x) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int a = r & 3, i = r >> 2;
    const int64_t y = y0 + 8 * (4 * g + i) + 4 * wy + a;
    if (y >= p.M) continue;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (x + w < p.N) p.C[y * p.ldc + x + w] = mxg_finish<EPI>(p, acc[a][w][i], y, x + w);
  }
}

// four columns of a row a thread (32-bit indices: problems in parts have fewer than 2^31 elements, mxg_plan)
template <int EPI>
__global__ __launch_bounds__(256) void mxg_join_kernel(MxGemm p, int parts, const float* __restrict__ part) {
  const uint32_t n = (uint32_t)p.N, quads = (n + 3) / 4;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const uint32_t y = i / quads, x = (i - y * quads) * 4;
  if (y >= (uint32_t)p.M) return;
  const float* src = part + (y * n + x);
  const int64_t step = p.M * p.N;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if ((n & 3) == 0) {
    for (int k = 0; k < parts; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(src + k * step);
      o[0] += v.x; o[1] += v.y; o[2] += v.z; o[3] += v.w;
    }
  } else {
    for (int k = 0; k < parts; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (x + w < n) o[w] += src[k * step + w];
  }
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (x + w < n) p.C[y * p.ldc + x + w] = mxg_finish<EPI>(p, o[w], y, x + w);
}

// ---- up to 16 rows: the weights straight from memory ------------------------------------------------------------------------------------
// One workgroup per 128-row panel of the weights, wave t of each half of K its rows 8 n + t: a lane's 16 bytes of codes are one block, its 16 bytes of scales the eight waves' (byte t & 3 of
// dwords t >> 2 and 2 + (t >> 2)).  The activations -- bf16 rows that are quantised here (X), or codes and scales -- lie in the LDS as a whole.  The weights of four
// stages (8 KB a wave) are in flight while the four before are multiplied, the first ones in front of the quantisation.  Bound by the weights' bytes: 30,720 x 5,120 for one
// row in 15.7 us, 5.3 TB/s.
constexpr int MXR_ROWS = 16, MXR_LDS = 144 * 1024;
struct MxRows {
  const bf16_t* x;   // null: A, As
  int64_t x_row;
  const uint8_t *A, *As, *W, *Ws;
  int64_t N;
  int M;
};
__host__ __device__ constexpr int mxr_pitch(int K) { return K / 2 + 16; }         // (a row's 16 bytes more: the rows of a fragment read start at other banks)
__host__ __device__ constexpr int mxr_scales(int K) { return (K / 32 + 15) & ~15; }

typedef int mx_i8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ mx_i8 mx_wide(const mx_u4& v) { return mx_i8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }   // (of which a 4-bit operand reads the first four)

template <int EPI>
__global__ __launch_bounds__(1024) void gemm_mxfp4_rows_kernel(MxRows r, MxGemm p) {
  extern __shared__ __attribute__((aligned(16))) char rows_lds[];   // codes [M][pitch], scale bytes [M][scales]
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int t = __builtin_amdgcn_readfirstlane((tid >> 6) & 7), half = __builtin_amdgcn_readfirstlane(tid >> 9);
  const int K = p.K, kt = p.kt, blocks = K / 32, pitch = mxr_pitch(K), sp = mxr_scales(K);
  uint8_t* codes = reinterpret_cast<uint8_t*>(rows_lds);
  uint8_t* scales = codes + r.M * pitch;
  const int64_t col = (int64_t)blockIdx.x * 128 + 8 * n + t;
  const uint8_t* w = r.W + min(col, r.N - 1) * (K / 2) + 16 * g;                   // past the matrix: its last row again, never stored
  const uint8_t* ws = r.Ws + (int64_t)blockIdx.x * kt * 1024 + lane * 16;
  struct Batch {
    mx_u4 c[4][2], s[4];
  };
  const int first = kt * half / 2, end = kt * (half + 1) / 2;
  auto fetch = [&](Batch& b, int s0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i;
      if (s < end) b.s[i] = *reinterpret_cast<const mx_u4*>(ws + (int64_t)s * 1024);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        b.c[i][ks] = mx_u4{0u, 0u, 0u, 0u};
        if (s < end && 8 * s + 4 * ks + g < blocks) b.c[i][ks] = *reinterpret_cast<const mx_u4*>(w + s * 128 + ks * 64);
      }
    }
  };
  Batch cur, nxt;
  fetch(cur, first);
  for (int i = tid; i < r.M * blocks; i += 1024) {
    const int m = i / blocks, j = i - m * blocks;
    mx_u4 c;
    uint32_t e;
    if (r.x != nullptr) {
      const bf16_t* x = r.x + m * r.x_row + j * 32;
      uint32_t a = 0;
      float f[32];
#pragma unroll
      for (int q = 0; q < 4; ++q) unpack8(*reinterpret_cast<const uint4*>(x + 8 * q), f + 8 * q);
#pragma unroll
      for (int q = 0; q < 32; ++q) a = max(a, __float_as_uint(f[q]) & 0x7fffffffu);
      e = mxfp4_scale(a);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t v = mxfp4_encode8(f + 8 * q, e);
        c[q] = v;
      }
    } else {
      c = *reinterpret_cast<const mx_u4*>(r.A + (int64_t)m * (K / 2) + j * 16);
      e = r.As[(j >> 3) * 1024 + (j & 3) * 256 + (m >> 3) * 16 + ((j >> 2) & 1) * 8 + (m & 7)];
    }
    *reinterpret_cast<mx_u4*>(codes + m * pitch + j * 16) = c;
    scales[m * sp + j] = (uint8_t)e;
  }
  __syncthreads();
  const int m = min(n, r.M - 1);   // (rows past the last: that one again, never stored)
  const uint8_t* xc = codes + m * pitch + 16 * g;
  const uint8_t* xs = scales + m * sp + g;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int sh = 8 * (t & 3);
  const bool upper = t >= 4;
  for (int s0 = first; s0 < end; s0 += 4) {
    if (s0 + 4 < end) fetch(nxt, s0 + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i;
      if (s >= end) break;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const int j = 8 * s + 4 * ks;
        const bool in = j + g < blocks;
        mx_u4 a = mx_u4{0u, 0u, 0u, 0u};
        uint32_t sa = 0;
        if (in) {
          a = *reinterpret_cast<const mx_u4*>(xc + j * 16);
          sa = xs[j];
        }
        const uint32_t word = upper ? cur.s[i][2 * ks + 1] : cur.s[i][2 * ks];
        const uint32_t sw = in ? word >> sh : 0u;
        // (the builtin: one chain of products, where hipcc's own wait states between them cost nothing)
        if (EPI == WAN_EPI_TRANSPOSED) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_wide(cur.c[i][ks]), mx_wide(a), acc, 4, 4, 0, (int)sw, 0, (int)sa);
        else acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_wide(a), mx_wide(cur.c[i][ks]), acc, 4, 4, 0, (int)sa, 0, (int)sw);
      }
    }
    cur = nxt;
  }
  __syncthreads();   // (the codes are read)
  f32x4* sums = reinterpret_cast<f32x4*>(rows_lds);
  if (half == 1) sums[tid - 512] = acc;
  __syncthreads();
  if (half == 1) return;
  acc += sums[tid];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (EPI == WAN_EPI_TRANSPOSED) {   // register i: weight row 8 (4 g + i) + t, token n
      const int64_t y = (int64_t)blockIdx.x * 128 + 8 * (4 * g + i) + t;
      if (y < r.N && n < r.M) p.C[y * p.ldc + n] = mxg_finish<EPI>(p, acc[i], y, n);
    } else {
      const int y = 4 * g + i;
      if (y < r.M && col < r.N) p.C[y * p.ldc + col] = mxg_finish<EPI>(p, acc[i], y, col);
    }
  }
}

// Which kernel, and in how many parts along K: 0 = the 256 x 256 tiles of gemm_mxfp4m.hip, n = 128 x 128 tiles in n parts.  The least of what the
// three were measured to take, in us: a round of up to 256 big tiles 8.5 + 1.2 a stage, of small ones 5.5 + 0.52 a stage, a join 5 and the partial
// sums' bytes.  Both sides, M x N x K: 512 x 5,120 x 5,120 (40 big tiles) 29.3 big, 15.8 small; 1,024 x 5,120 x 13,824 (80) 68.5 and 62.2;
// 1,560 x 5,120 x 5,120 (140) 34.3 and 46.6;
// 16 x 5,120 x 5,120 (small, 40 tiles) in one part 13.3, in five 10.8; 512 x 1,536 x 5,120 (48) 13.6 and 17.2.
int mxg_plan(int64_t M, int64_t N, int kt) {
  const int64_t big = ((M + 255) / 256) * ((N + 255) / 256), small = ((M + 127) / 128) * ((N + 127) / 128);
  double best = (8.5 + 1.2 * kt) * (double)((big + 255) / 256);
  int plan = 0;
  for (int parts = 1; parts <= 16 && 2 * parts <= (kt > 2 ? kt : 2); ++parts) {
    if (parts > 1 && small * parts > 512) break;
    const double t = (5.5 + 0.52 * ((kt + parts - 1) / parts)) * (double)((small * parts + 255) / 256) + (parts > 1 ? 5.0 + 1.4e-6 * parts * (double)(M * N) : 0.0);
    if (t < best) { best = t; plan = parts; }
  }
  return plan;
}

template <int EPI>
int mxg_launch(const MxGemm& p, int parts, float* scratch, hipStream_t st) {
  const int64_t tiles = ((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (parts <= 1) {
    hipLaunchKernelGGL((gemm_mxfp4_kernel<EPI, false>), dim3((unsigned)tiles), dim3(256), 0, st, p, 1, scratch);
  } else {
    hipLaunchKernelGGL((gemm_mxfp4_kernel<EPI, true>), dim3((unsigned)(tiles * parts)), dim3(256), 0, st, p, parts, scratch);
    hipLaunchKernelGGL(mxg_join_kernel<EPI>, dim3((unsigned)((p.M * ((p.N + 3) / 4) + 255) / 256)), dim3(256), 0, st, p, parts, (const float*)scratch);
  }
  WAN_LAUNCH_CHECK();
  return 0;
}

// Whether a problem of few rows takes that kernel.  A workgroup streams its panel at the 30 GB/s that one CU gets, so few panels of long rows are better cut along K, the more so the
// more rows each workgroup has to quantise.  In us with the quantisation, this kernel and the others, M x N x K: 1 x 1,536 x 1,536 5.4 and 9.1; 16 x 1,536 x 1,536 7.6 and 9.6;
// 1 x 5,120 x 5,120 13.0 and 12.2; 16 x 5,120 x 5,120 16.8 and 13.8; 1 x 5,120 x 13,824 30.9 and 17.0.  With panels for most CUs: 1 x 30,720 x 5,120 15.7 and 19.3;
// 4 x 13,824 x 5,120 15.5 and 16.6; 16 x 13,824 x 5,120 18.2 and 17.2.
bool mxr_fits(int64_t M, int64_t N, int K) {
  if (M > MXR_ROWS || M * (mxr_pitch(K) + mxr_scales(K)) > MXR_LDS) return false;
  return K <= 4608 - 128 * M || (M <= 8 && N >= 96 * 128);
}

int mxr_launch(const bf16_t* x, int64_t x_row, const uint8_t* A, const uint8_t* As, const uint8_t* W, const uint8_t* Ws, int64_t M, int64_t N, const MxGemm& p, int epilogue, hipStream_t st) {
  const MxRows r = {x, x_row, A, As, W, Ws, N, (int)M};
  const dim3 grid((unsigned)((N + 127) / 128)), wg(1024);
  const unsigned need = (unsigned)(M * (mxr_pitch(p.K) + mxr_scales(p.K))), lds = need > 8192 ? need : 8192;   // (the second half's sums: 8 KB)
  switch (epilogue) {
    case WAN_EPI_NONE: hipLaunchKernelGGL(gemm_mxfp4_rows_kernel<WAN_EPI_NONE>, grid, wg, lds, st, r, p); break;
    case WAN_EPI_GELU_TANH: hipLaunchKernelGGL(gemm_mxfp4_rows_kernel<WAN_EPI_GELU_TANH>, grid, wg, lds, st, r, p); break;
    case WAN_EPI_GATE_RES: hipLaunchKernelGGL(gemm_mxfp4_rows_kernel<WAN_EPI_GATE_RES>, grid, wg, lds, st, r, p); break;
    default: hipLaunchKernelGGL(gemm_mxfp4_rows_kernel<WAN_EPI_TRANSPOSED>, grid, wg, lds, st, r, p); break;
  }
  WAN_LAUNCH_CHECK();
  return 0;
}

}  // namespace

int wan_gemm_mxfp4m_try(const MxGemm& p, int epilogue, hipStream_t st);   // gemm_mxfp4m.hip

extern "C" int64_t wan_gemm_mxfp4_scratch_bytes(int64_t M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || mxr_fits(M, N, K)) return 0;
  const int parts = mxg_plan(M, N, (K + 255) / 256);
  return parts <= 1 ? 0 : (int64_t)parts * M * N * 4;
}

// Whether the output shares memory with x: workgroups may read x while others already write.  (Rows side by side in one buffer share a range, but no element.)
static bool mx_overlaps(const wan_bf16* x, int64_t x_row, const wan_bf16* C, int64_t ldc, int64_t M, int N, int K, int epilogue) {
  const bool tr = epilogue == WAN_EPI_TRANSPOSED;
  const uintptr_t x0 = (uintptr_t)x, x1 = x0 + ((M - 1) * x_row + K) * 2, c0 = (uintptr_t)C, c1 = c0 + ((tr ? N - 1 : M - 1) * ldc + (tr ? M : N)) * 2;
  if (x1 <= c0 || c1 <= x0) return false;
  if (tr || x_row != ldc || M == 1) return true;
  const int64_t d = ((int64_t)(c0 / 2) - (int64_t)(x0 / 2)) % ldc, at = d < 0 ? d + ldc : d;   // C's first column, counted from x's
  return !(at >= K && at + N <= ldc);
}
// ... and with one of the small operands, or the weights
static bool mx_touches(const wan_bf16* C, int64_t ldc, int64_t M, int N, int epilogue, const void* p, int64_t bytes) {
  const bool tr = epilogue == WAN_EPI_TRANSPOSED;
  const uintptr_t c0 = (uintptr_t)C, c1 = c0 + ((tr ? N - 1 : M - 1) * ldc + (tr ? M : N)) * 2, p0 = (uintptr_t)p;
  return p != nullptr && p0 < c1 && c0 < p0 + bytes;
}

static int mx_gemm_check(const uint8_t* A, const uint8_t* a_scales, const uint8_t* W, const uint8_t* w_scales, const wan_bf16* bias, wan_bf16* C, int64_t ldc, int64_t M, int N, int K, int epilogue,
                         const wan_bf16* R, const wan_bf16* mod, const wan_bf16* e, int n_mod, int gate_idx, int64_t rows_per_batch) {
  WAN_REQUIRE(A && a_scales && W && w_scales && C, "wan_gemm_mxfp4: null operand");
  WAN_REQUIRE(M >= 1 && N >= 1 && K >= 32 && K % 32 == 0, "wan_gemm_mxfp4: M=%lld and N=%d must be positive, K=%d a positive multiple of 32", (long long)M, N, K);
  WAN_REQUIRE((((uintptr_t)A | (uintptr_t)a_scales | (uintptr_t)W | (uintptr_t)w_scales | (uintptr_t)C) & 15) == 0, "wan_gemm_mxfp4: pointers must be 16-byte aligned");
  WAN_REQUIRE(K <= (1 << 23), "wan_gemm_mxfp4: K=%d exceeds the kernels' 32-bit offsets inside a tile", K);
  WAN_REQUIRE(epilogue >= WAN_EPI_NONE && epilogue <= WAN_EPI_TRANSPOSED, "wan_gemm_mxfp4: unknown epilogue %d", epilogue);
  WAN_REQUIRE(ldc >= (epilogue == WAN_EPI_TRANSPOSED ? M : N), "wan_gemm_mxfp4: ldc=%lld is smaller than a row of the output", (long long)ldc);
  if (epilogue == WAN_EPI_GATE_RES) {
    WAN_REQUIRE(R != nullptr, "wan_gemm_mxfp4: GATE_RES needs the residual R");
    WAN_REQUIRE(gate_idx < 0 || (mod && e && gate_idx < n_mod && rows_per_batch > 0), "wan_gemm_mxfp4: bad gate args");
  }
  WAN_REQUIRE(((M + 127) / 128) * (((int64_t)N + 127) / 128) < ((int64_t)1 << 27) && M * N < ((int64_t)1 << 39), "wan_gemm_mxfp4: grid too large");   // (16 parts, 256 elements a workgroup)
  return 0;
}

// One workgroup's output would be another's operand.  (A residual that is the output itself is read by the lane alone that writes its place.)
static int mx_gemm_aliases(const uint8_t* W, const uint8_t* w_scales, const wan_bf16* bias, const wan_bf16* C, int64_t ldc, int64_t M, int N, int K, int epilogue, const wan_bf16* R,
                           const wan_bf16* mod, const wan_bf16* e, int n_mod, int gate_idx, int64_t rows_per_batch) {
  WAN_REQUIRE(!mx_touches(C, ldc, M, N, epilogue, W, (int64_t)N * (K / 2)) && !mx_touches(C, ldc, M, N, epilogue, w_scales, wan_mxfp4_scale_bytes(N, K)) &&
                  !mx_touches(C, ldc, M, N, epilogue, bias, (int64_t)N * 2),
              "wan_gemm_mxfp4: the output must not overlap the weights or the bias");
  if (epilogue != WAN_EPI_GATE_RES) return 0;
  WAN_REQUIRE(R == C || !mx_overlaps(R, ldc, C, ldc, M, N, N, epilogue), "wan_gemm_mxfp4: an output that overlaps the residual must be the residual");
  WAN_REQUIRE(gate_idx < 0 || (!mx_touches(C, ldc, M, N, epilogue, mod, (int64_t)n_mod * N * 2) &&
                               !mx_touches(C, ldc, M, N, epilogue, e, (M + rows_per_batch - 1) / rows_per_batch * n_mod * N * 2)),
              "wan_gemm_mxfp4: the output must not overlap the gate");
  return 0;
}

extern "C" int wan_gemm_mxfp4(const uint8_t* A, const uint8_t* a_scales, const uint8_t* W, const uint8_t* w_scales, const wan_bf16* bias, wan_bf16* C, int64_t ldc, int64_t M, int N, int K,
                              int epilogue, const wan_bf16* R, const wan_bf16* mod, const wan_bf16* e, int n_mod, int gate_idx, int64_t rows_per_batch, void* scratch, int64_t scratch_bytes,
                              void* stream) {
  const int bad = mx_gemm_check(A, a_scales, W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
  if (bad != 0) return bad;
  const int64_t need = wan_gemm_mxfp4_scratch_bytes(M, N, K);
  WAN_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0), "wan_gemm_mxfp4: needs 16-byte aligned scratch of %lld bytes", (long long)need);
  const int alias = mx_gemm_aliases(W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
  if (alias != 0) return alias;
  WAN_REQUIRE(!mx_touches(C, ldc, M, N, epilogue, A, M * (K / 2)) && !mx_touches(C, ldc, M, N, epilogue, a_scales, wan_mxfp4_scale_bytes(M, K)),
              "wan_gemm_mxfp4: the output must not overlap the quantised rows");
  const bool tr = epilogue == WAN_EPI_TRANSPOSED;
  hipStream_t st = as_stream(stream);
  const MxGemm p = {tr ? W : A, tr ? w_scales : a_scales, tr ? A : W, tr ? a_scales : w_scales, tr ? N : M, tr ? M : N, K, (K + 255) / 256, bias, C, ldc, R, mod, e, n_mod, gate_idx,
                    rows_per_batch > 0 ? rows_per_batch : 1};
  if (mxr_fits(M, N, K)) return mxr_launch(nullptr, 0, A, a_scales, W, w_scales, M, N, p, epilogue, st);
  const int plan = mxg_plan(M, N, p.kt);
  if (plan == 0) {
    const int rc = wan_gemm_mxfp4m_try(p, epilogue, st);
    if (rc >= 0) return rc;   // (else an alignment that it does not take)
  }
  float* ws = reinterpret_cast<float*>(scratch);
  switch (epilogue) {
    case WAN_EPI_NONE: return mxg_launch<WAN_EPI_NONE>(p, plan, ws, st);
    case WAN_EPI_GELU_TANH: return mxg_launch<WAN_EPI_GELU_TANH>(p, plan, ws, st);
    case WAN_EPI_GATE_RES: return mxg_launch<WAN_EPI_GATE_RES>(p, plan, ws, st);
    default: return mxg_launch<WAN_EPI_TRANSPOSED>(p, plan, ws, st);
  }
}

// the quantised rows and their scales in front of the product's own scratch
static int64_t mx_linear_codes(int64_t M, int K) { return (M * (K / 2) + 255) / 256 * 256; }

extern "C" int64_t wan_linear_mxfp4_scratch_bytes(int64_t M, int N, int K) {
  if (M < 1 || N < 1 || K < 32 || K % 32 != 0 || mxr_fits(M, N, K)) return 0;
  return mx_linear_codes(M, K) + wan_mxfp4_scale_bytes(M, K) + wan_gemm_mxfp4_scratch_bytes(M, N, K);
}

extern "C" int wan_linear_mxfp4(const wan_bf16* x, int64_t x_row, const uint8_t* W, const uint8_t* w_scales, const wan_bf16* bias, wan_bf16* C, int64_t ldc, int64_t M, int N, int K, int epilogue,
                                const wan_bf16* R, const wan_bf16* mod, const wan_bf16* e, int n_mod, int gate_idx, int64_t rows_per_batch, void* scratch, int64_t scratch_bytes, void* stream) {
  WAN_REQUIRE(M >= 1 && N >= 1 && K >= 32 && K % 32 == 0, "wan_linear_mxfp4: M=%lld and N=%d must be positive, K=%d a positive multiple of 32", (long long)M, N, K);
  WAN_REQUIRE(x != nullptr, "wan_linear_mxfp4: null pointer");
  WAN_REQUIRE(x_row >= K && x_row % 8 == 0, "wan_linear_mxfp4: the row stride %lld must be a multiple of 8 elements, at least K", (long long)x_row);
  WAN_REQUIRE(((uintptr_t)x & 15) == 0, "wan_linear_mxfp4: pointers must be 16-byte aligned");
  if (mxr_fits(M, N, K)) {   // nothing of the quantised rows leaves the kernel
    const uint8_t* some = reinterpret_cast<const uint8_t*>(x);
    const int rc = mx_gemm_check(some, some, W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
    if (rc != 0) return rc;
    WAN_REQUIRE(!mx_overlaps(x, x_row, C, ldc, M, N, K, epilogue), "wan_linear_mxfp4: the output must not overlap x");
    const int alias = mx_gemm_aliases(W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
    if (alias != 0) return alias;
    const MxGemm p = {nullptr, nullptr, nullptr, nullptr, M, N, K, (K + 255) / 256, bias, C, ldc, R, mod, e, n_mod, gate_idx, rows_per_batch > 0 ? rows_per_batch : 1};
    return mxr_launch(x, x_row, nullptr, nullptr, W, w_scales, M, N, p, epilogue, as_stream(stream));
  }
  const int64_t need = wan_linear_mxfp4_scratch_bytes(M, N, K);
  WAN_REQUIRE(scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0, "wan_linear_mxfp4: needs 16-byte aligned scratch of %lld bytes", (long long)need);
  uint8_t* codes = reinterpret_cast<uint8_t*>(scratch);
  uint8_t* scales = codes + mx_linear_codes(M, K);
  uint8_t* rest = scales + wan_mxfp4_scale_bytes(M, K);
  // (the product's arguments are checked by a call that may refuse them: in front of the first launch)
  const int rc = mx_gemm_check(codes, scales, W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
  if (rc != 0) return rc;
  WAN_REQUIRE(!mx_overlaps(x, x_row, C, ldc, M, N, K, epilogue), "wan_linear_mxfp4: the output must not overlap x");
  const int alias = mx_gemm_aliases(W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch);
  if (alias != 0) return alias;
  const int rq = wan_mxfp4_quantize(x, x_row, codes, scales, M, K, stream);
  if (rq != 0) return rq;
  return wan_gemm_mxfp4(codes, scales, W, w_scales, bias, C, ldc, M, N, K, epilogue, R, mod, e, n_mod, gate_idx, rows_per_batch, rest, scratch_bytes - (rest - codes), stream);
}
