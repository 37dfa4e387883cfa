// The MXFP4 Linear (gemm_mxfp4.hip) for many tiles: 256 x 256 x 256 tiles on gemm256m.hip's stage discipline.
//
// Half a byte per element makes a k-stage of 256 values exactly gemm256m's 128-byte rows: unit images (256 rows x 128 B), swizzle, ring of five 32-KB
// units, fragment reads and register-direct stores carry over, and a k-step of 128 is 64 MFMAs of 16 cycles (v_mfma_scale_f32_16x16x128_f8f6f4 on
// two fp4 operands) where gemm256m's of 32 is 64 MFMAs of 16 cycles -- four times the FLOP on the same bytes and issue slots.  What differs:
//   * both operands' image rows are (slab, t, n) = row slab * 128 + 8 n + t: a lane's eight scales of an operand and k-step are then 8 consecutive
//     bytes of mxfp4_ops.hip's scale tiles, and all of a stage's one 16-byte load (dword 2 ks + (t >> 2), byte t & 3: the instruction picks the
//     byte).  y tile a, register i of lane (n, g) is row 8 (4 g + i) + a.
//   * the LDS is full, so the scales go straight to registers: stage S + 1's are loaded at the start of stage S.  hipcc counts these loads and not
//     the LDS-DMA beside them, so it waits for them with vmcnt(0) wherever they are first touched: that is done at the sync point, where the DMA in
//     flight is oldest -- all sixteen pieces of X_{S+2} and Y_{S+3} are issued right behind the sync point P_S, none in k-step 0, and have
//     80 MFMAs (1,280 cycles) by then.
//   * K need not be a multiple of 256: what a row's last stage reads past the row is the next row's codes (the buffer's end reads as zeros), and the
//     scale bytes there are 0 on both sides -- (6 * 2^-127)^2 is 0 in fp32.
#include "mxfp4.h"

namespace {

typedef __attribute__((address_space(3))) const char mxm_lds_cchar;
typedef __attribute__((address_space(3))) const mx_u4 mxm_lds_u4;

constexpr int MXM_BM = 256, MXM_BN = 256, MXM_ROW = 128;   // tile, bytes of a row's stage
constexpr int MXM_UNIT = 256 * MXM_ROW;                    // one operand of one stage
constexpr int MXM_NU = 5;                                  // unit u (Y_S = 2 S, X_S = 2 S + 1) lives in slot u % 5

struct MxmFrags {
  mx_u4 y[8], x[8];
};

// MFMA m of a k-step: y tile m >> 3, x tile m & 7
template <int KS, int M0, int M1, class F>
__device__ __forceinline__ void mxm_run(f32x4 (&acc)[8][8], const MxmFrags& f, const mx_u4& sy, const mx_u4& sx, F&& gap) {
  if constexpr (M0 < M1) {
    mfma_mx<(M0 >> 3) & 3, M0 & 3>(acc[M0 >> 3][M0 & 7], f.y[M0 >> 3], f.x[M0 & 7], sy[2 * KS + (M0 >> 5)], sx[2 * KS + ((M0 & 7) >> 2)]);
    __builtin_amdgcn_sched_barrier(0);
    gap(M0);
    __builtin_amdgcn_sched_barrier(0);
    mxm_run<KS, M0 + 1, M1>(acc, f, sy, sx, gap);
  }
}

// EPI: WAN_EPI_TRANSPOSED = the bias along the rows
template <int EPI>
__global__ __launch_bounds__(256) void gemm_mxfp4m_kernel(MxGemm p, int tiles_y, int tiles_x, int group) {
  __shared__ __attribute__((aligned(16))) char smem[MXM_NU * MXM_UNIT];
  mxm_lds_cchar* lds = (mxm_lds_cchar*)smem;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wy = wave >> 1, wx = wave & 1;
  const int l15 = lane & 15, lg = lane >> 4;

  // XCD-contiguous ids, then groups of `group` tile rows walked column by column: the tiles that run at a time share few panels
  const int wg = xcd_remap(blockIdx.x, tiles_y * tiles_x);
  const int per_group = group * tiles_x;
  const int gidx = wg / per_group;
  const int first_y = gidx * group;
  const int gsz = min(tiles_y - first_y, group);
  const int in_g = wg - gidx * per_group;
  const int64_t y0 = (int64_t)(first_y + in_g % gsz) * MXM_BM;
  const int64_t x0 = (int64_t)(in_g / gsz) * MXM_BN;

  // DMA plan: piece i of wave w fills the 16-byte slots q = i * 256 + w * 64 + lane; image row q >> 3, physical chunk q & 7 = logical ^ ((row >> 1) & 7)
  const int pitch = p.K / 2;
  uint32_t yofs[8], xofs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = i * 256 + tid;
    const int row = q >> 3, lch = (q & 7) ^ ((row >> 1) & 7);
    const int r = (row >> 7) * 128 + 8 * (row & 15) + ((row >> 4) & 7);
    yofs[i] = (uint32_t)(min(y0 + r, p.M - 1) - y0) * (uint32_t)pitch + lch * 16;   // past the matrix: its last row again, never stored
    xofs[i] = (uint32_t)(min(x0 + r, p.N - 1) - x0) * (uint32_t)pitch + lch * 16;
  }
  const char* ybase = reinterpret_cast<const char*>(p.A) + y0 * pitch;
  const char* xbase = reinterpret_cast<const char*>(p.W) + x0 * pitch;
  uint32_t yrec = (uint32_t)min((p.M - y0) * pitch, (int64_t)0xffffff00);
  uint32_t xrec = (uint32_t)min((p.N - x0) * pitch, (int64_t)0xffffff00);
  const uint32_t smem_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const int nk = p.kt;
  int ky = 0, kx = 0;  // the stages the two streams point at; they stop at the last one
  auto y_piece = [&](int slot, int i) { mx_dma16(yofs[i], mx_rsrc(ybase, yrec), smem_lds + slot * MXM_UNIT + (i * 256 + wave * 64) * 16); };
  auto x_piece = [&](int slot, int i) { mx_dma16(xofs[i], mx_rsrc(xbase, xrec), smem_lds + slot * MXM_UNIT + (i * 256 + wave * 64) * 16); };
  auto y_advance = [&]() { const int s = ky + 1 < nk ? MXM_ROW : 0; ybase += s; yrec -= s; ky += s ? 1 : 0; };
  auto x_advance = [&]() { const int s = kx + 1 < nk ? MXM_ROW : 0; xbase += s; xrec -= s; kx += s ? 1 : 0; };

  // the lane's scales: 16 bytes a stage of each operand's 128-row panel
  const mx_u4* ysc = reinterpret_cast<const mx_u4*>(p.As + min((y0 >> 7) + wy, (p.M - 1) >> 7) * nk * 1024) + lg * 16 + l15;
  const mx_u4* xsc = reinterpret_cast<const mx_u4*>(p.Ws + min((x0 >> 7) + wx, (p.N - 1) >> 7) * nk * 1024) + lg * 16 + l15;

  // fragment addresses: one base register per (operand, k-step, 64-KB window) and immediates (gemm256m.hip)
  const int sw = (l15 >> 1) & 7;
  uint32_t ybw[2][3], xbw[2][3];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      ybw[ks][w] = (uint32_t)((((wy * 128 + l15) * 128 + ((lg ^ sw) << 4)) ^ (ks << 6)) + w * 65536);
      xbw[ks][w] = (uint32_t)((((wx * 128 + l15) * 128 + ((lg ^ sw) << 4)) ^ (ks << 6)) + w * 65536);
      asm volatile("" : "+v"(ybw[ks][w]), "+v"(xbw[ks][w]));
    }
  auto load_frag = [&](MxmFrags& f, int sy, int sx, int ks, int r) {
    if (r < 8) {
      const int u = sy * MXM_UNIT + r * 2048;
      f.y[r] = *(mxm_lds_u4*)(lds + ybw[ks][u >> 16] + (u & 0xffff));
    } else {
      const int u = sx * MXM_UNIT + (r - 8) * 2048;
      f.x[r - 8] = *(mxm_lds_u4*)(lds + xbw[ks][u >> 16] + (u & 0xffff));
    }
  };
  // the order of a k-step's 16 fragment reads: y 1 .. 7, x 1 .. 7, x 0, y 0 -- what its first MFMA needs comes last, so that ONE wait covers all
  auto ord = [](int i) constexpr { return i < 7 ? 1 + i : i < 14 ? 2 + i : i == 14 ? 8 : 0; };

  mx_u4 sy = ysc[0], sx = xsc[0];
  asm volatile("" : "+v"(sy), "+v"(sx));
#pragma unroll
  for (int i = 0; i < 8; ++i) y_piece(0, i);
  y_advance();
#pragma unroll
  for (int i = 0; i < 8; ++i) x_piece(1, i);
  x_advance();
#pragma unroll
  for (int i = 0; i < 8; ++i) y_piece(2, i);
  y_advance();
#pragma unroll
  for (int i = 0; i < 8; ++i) x_piece(3, i);
  x_advance();
#pragma unroll
  for (int i = 0; i < 8; ++i) y_piece(4, i);
  y_advance();
  f32x4 acc[8][8];
#pragma unroll
  for (int a = 0; a < 8; ++a)
#pragma unroll
    for (int b = 0; b < 8; ++b) {
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[a][b][r] = 0.f;
      asm volatile("" : "+a"(acc[a][b]));
    }
  asm volatile("s_waitcnt vmcnt(24)" ::: "memory");  // stage 0 landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  MxmFrags f0, f1;
#pragma unroll
  for (int r = 0; r < 16; ++r) load_frag(f0, 0, 1, 0, ord(r));
  // Stage S = 5 i + J: Y in slot 2J % 5, X in (2J + 1) % 5.
  //   k-step 0 (f0): stage S + 1's scales behind MFMA 0, k-step 1's fragments behind MFMA 1, 3, .., 31
  //   k-step 1 (f1): MFMAs 0 .. 15 bare
  //   P_S: everything landed, stage S fully read + barrier
  //   MFMAs 16 .. 63: X_{S+2} -> slot of Y_S behind 16, 19, .., 37, Y_{S+3} -> slot of X_S behind 40, 43, .., 61; stage S + 1's first fragments
  //                   in the other gaps up to MFMA 39
  mx_u4 ny, nx;
#define MXM_STAGE(J)                                                                                                             \
  if (__builtin_expect(kt + (J) < nk, 1)) {                                                                                      \
    constexpr int J_ = (J);                                                                                                      \
    constexpr int SY = (2 * J_) % 5, SX = (2 * J_ + 1) % 5, NY = (2 * J_ + 2) % 5, NX = (2 * J_ + 3) % 5;                         \
    mxm_run<0, 0, 64>(acc, f0, sy, sx, [&](int m) __attribute__((always_inline)) {                                               \
      if (m == 0) {                                                                                                              \
        const int64_t at = (int64_t)min(kt + J_ + 1, nk - 1) * 64;                                                               \
        ny = ysc[at];                                                                                                            \
        nx = xsc[at];                                                                                                            \
      }                                                                                                                          \
      if ((m & 1) == 1 && m < 32) load_frag(f1, SY, SX, 1, ord(m >> 1));                                                         \
    });                                                                                                                          \
    mxm_run<1, 0, 16>(acc, f1, sy, sx, [](int) {});                                                                              \
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                                                                  \
    __builtin_amdgcn_s_barrier();                                                                                                \
    asm volatile("" : "+v"(ny), "+v"(nx)::"memory");                                                                             \
    mxm_run<1, 16, 64>(acc, f1, sy, sx, [&](int m) __attribute__((always_inline)) {                                              \
      const int q = (m - 16) / 3, r = (m - 16) % 3;                                                                              \
      if (r == 0 && q < 8) x_piece(SY, q);                                                                                       \
      if (r == 0 && q >= 8) y_piece(SX, q - 8);                                                                                  \
      if (r != 0 && q < 8) load_frag(f0, NY, NX, 0, ord(2 * q + r - 1));                                                         \
    });                                                                                                                          \
    x_advance();                                                                                                                 \
    y_advance();                                                                                                                 \
    sy = ny;                                                                                                                     \
    sx = nx;                                                                                                                     \
    asm volatile("s_nop 1" : "+v"(sy), "+v"(sx)); /* a register copy in front of an MFMA that reads it: hipcc pads nothing around asm */ \
  }
  for (int kt = 0; kt < nk; kt += 5) {
    MXM_STAGE(0)
    MXM_STAGE(1)
    MXM_STAGE(2)
    MXM_STAGE(3)
    MXM_STAGE(4)
  }
#undef MXM_STAGE
  // trailing DMA (the LDS is released at the end); the last MFMAs -> accumulator reads
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");

  // ---- epilogue: straight from the registers.  Rows past the matrix fall outside the descriptors' num_records; a lane's 8 columns are inside or
  // outside as a whole (N % 8 == 0), outside: an offset past num_records --------------------------------------------------------------------
  uint32_t lane_e;  // an opaque lane id: derived from threadIdx the epilogue's offsets are hoisted in front of the MFMA loop and spilled
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
  const uint32_t ne = lane_e & 15u, ge = lane_e >> 4;
  const uint32_t colb = (uint32_t)(wx * 128) * 2u + ne * 16u;
  const int64_t rows_valid = min(p.M - y0, (int64_t)MXM_BM);
  const uint32_t onum = (uint32_t)((rows_valid - 1) * p.ldc * 2 + MXM_BN * 2);
  const uint32_t ldo2 = (uint32_t)(p.ldc * 2);
  const __amdgpu_buffer_rsrc_t odesc = __builtin_amdgcn_make_buffer_rsrc((void*)(p.C + y0 * p.ldc + x0), 0, (int)onum, 0x00020000);
  const __amdgpu_buffer_rsrc_t rdesc = __builtin_amdgcn_make_buffer_rsrc((void*)((EPI == WAN_EPI_GATE_RES ? p.R : p.C) + y0 * p.ldc + x0), 0, (int)onum, 0x00020000);
  const uint32_t row_lane = (uint32_t)(wy * 128) + 32u * ge;
  const bool col_in = x0 + wx * 128 + 8 * (int64_t)ne + 8 <= p.N;
  const uint32_t lane_off = col_in ? row_lane * ldo2 + colb : 0x80000000u;
  float bcol[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (EPI != WAN_EPI_TRANSPOSED && p.bias != nullptr && col_in) unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.bias + x0) + colb), bcol);
  // gates: a 256-row tile touches at most two batches (rows_per_batch >= 256)
  float gA[8], gB[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) gA[j] = gB[j] = 1.f;
  uint32_t rb = 0xffffffffu;
  auto gate_row = [&](int64_t bidx, float* gq) {
    float mv[8], ev[8];
    unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.mod + (int64_t)p.gate_idx * p.N + x0) + colb), mv);
    unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.e + (bidx * p.n_mod + p.gate_idx) * p.N + x0) + colb), ev);
#pragma unroll
    for (int j = 0; j < 8; ++j) gq[j] = mv[j] + ev[j];
  };
  if (EPI == WAN_EPI_GATE_RES && p.gate_idx >= 0 && col_in) {
    const int64_t b0 = y0 / p.rows_per_batch;
    const int64_t yb = (b0 + 1) * p.rows_per_batch;
    gate_row(b0, gA);
    if (yb < y0 + rows_valid) {
      rb = (uint32_t)(yb - y0);
      gate_row(b0 + 1, gB);
    }
  }
  typedef unsigned int mxm_st4 __attribute__((__vector_size__(16)));
  auto rload = [&](int a, int i) -> uint4 {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rdesc, (int)(lane_off + (uint32_t)(8 * i + a) * ldo2), 0, 0));
  };
  uint4 rq[3][4] = {};   // residual rows of the next two y tiles are in flight while one is converted
  if (EPI == WAN_EPI_GATE_RES) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { rq[0][i] = rload(0, i); rq[1][i] = rload(1, i); }
  }
#pragma unroll
  for (int a = 0; a < 8; ++a) {
    if (EPI == WAN_EPI_GATE_RES && a + 2 < 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) rq[(a + 2) % 3][i] = rload(a + 2, i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t rit = (uint32_t)(8 * i + a);
      float brow = 0.f;
      if (EPI == WAN_EPI_TRANSPOSED && p.bias != nullptr) brow = bf2f(p.bias[min(y0 + row_lane + rit, p.M - 1)]);
      float v[8], rv[8];
      if (EPI == WAN_EPI_GATE_RES) unpack8(rq[a % 3][i], rv);
      const bool second = row_lane + rit >= rb;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        float o = acc[a][t][i] + (EPI == WAN_EPI_TRANSPOSED ? brow : bcol[t]);
        if (EPI == WAN_EPI_GELU_TANH) o = mx_gelu_tanh(o);
        if (EPI == WAN_EPI_GATE_RES) o = __builtin_fmaf(o, second ? gB[t] : gA[t], rv[t]);
        v[t] = o;
      }
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(mxm_st4, pack8(v)), odesc, (int)(lane_off + rit * ldo2), 0, 0);
      if (EPI == WAN_EPI_GELU_TANH) __builtin_amdgcn_sched_barrier(0);  // 8 GELUs' temporaries at a time
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace

// -1: the problem does not fit this kernel (gemm_mxfp4.hip's takes it)
int wan_gemm_mxfp4m_try(const MxGemm& p, int epilogue, hipStream_t st) {
  if (p.N % 8 != 0 || p.ldc % 8 != 0) return -1;   // a lane stores 8 columns or none
  if (((uintptr_t)p.C | (uintptr_t)p.R | (uintptr_t)p.mod | (uintptr_t)p.e) & 15) return -1;
  if (epilogue != WAN_EPI_TRANSPOSED && ((uintptr_t)p.bias & 15)) return -1;
  if (epilogue == WAN_EPI_GATE_RES && p.gate_idx >= 0 && p.rows_per_batch < MXM_BM) return -1;
  if (256 * (int64_t)(p.K / 2) + 256 >= ((int64_t)1 << 31) || 256 * p.ldc * 2 + 512 >= ((int64_t)1 << 31)) return -1;   // 32-bit offsets inside a tile
  const int64_t ty = (p.M + MXM_BM - 1) / MXM_BM, tx = (p.N + MXM_BN - 1) / MXM_BN;
  if (ty * tx >= ((int64_t)1 << 31)) return -1;
  const dim3 grid((unsigned)(ty * tx)), wg(256);
  const int group = epilogue == WAN_EPI_TRANSPOSED ? 8 : 4;
  switch (epilogue) {
    case WAN_EPI_NONE: hipLaunchKernelGGL(gemm_mxfp4m_kernel<WAN_EPI_NONE>, grid, wg, 0, st, p, (int)ty, (int)tx, group); break;
    case WAN_EPI_GELU_TANH: hipLaunchKernelGGL(gemm_mxfp4m_kernel<WAN_EPI_GELU_TANH>, grid, wg, 0, st, p, (int)ty, (int)tx, group); break;
    case WAN_EPI_GATE_RES: hipLaunchKernelGGL(gemm_mxfp4m_kernel<WAN_EPI_GATE_RES>, grid, wg, 0, st, p, (int)ty, (int)tx, group); break;
    default: hipLaunchKernelGGL(gemm_mxfp4m_kernel<WAN_EPI_TRANSPOSED>, grid, wg, 0, st, p, (int)ty, (int)tx, group); break;
  }
  WAN_LAUNCH_CHECK();
  return 0;
}
