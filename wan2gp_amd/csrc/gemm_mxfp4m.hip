// The MXFP4 Linear (gemm_mxfp4.hip) for many tiles: 256 x 256 x 256 tiles on gemm256m.hip's stage discipline.
//
// Half a byte per element makes a k-stage of 256 values exactly gemm256m's 128-byte rows: unit images (256 rows x 128 B), swizzle, ring of five 32-KB
// units, fragment reads and register-direct stores carry over, and a k-step of 128 is 64 MFMAs of 16 cycles (v_mfma_scale_f32_16x16x128_f8f6f4 on
// two fp4 operands) where gemm256m's of 32 is 64 MFMAs of 16 cycles -- four times the FLOP on the same bytes and issue slots.  What differs:
//   * one workgroup a CU takes one tile after the other, and the streams of units run on into the next tile: its first stages land and this tile's stores
//     drain while the other of the two is worked on (a workgroup a tile: 32,760 x 8,960 x 1,536 297 us, so 242; with the GELU 356 and 292).  The tile
//     loop has one stage body, and one more for a tile's first stage, with the ring slots in scalar registers.
//   * both operands' image rows are (slab, t, n) = row slab * 128 + 8 n + t: a lane's eight scales of an operand and k-step are then 8 consecutive
//     bytes of mxfp4_ops.hip's scale tiles, and all of a stage's one 16-byte load (dword 2 ks + (t >> 2), byte t & 3: the instruction picks the
//     byte).  y tile a, register i of lane (n, g) is row 8 (4 g + i) + a.
//   * the LDS is full, so the scales go straight to registers: stage S + 1's are loaded at the start of stage S.  hipcc counts these loads and not
//     the LDS-DMA beside them, so it waits for them with vmcnt(0) wherever they are first touched: that is done at the sync point, where the DMA in
//     flight is oldest -- all sixteen pieces of X_{S+2} and Y_{S+3} are issued right behind the sync point P_S, none in k-step 0, and have
//     80 MFMAs (1,280 cycles) by then.
//   * K need not be a multiple of 256: what a row's last stage reads past the row is the next row's codes (the buffer's end reads as zeros), and the
//     scale bytes there are 0 on both sides -- (6 * 2^-127)^2 is 0 in fp32.
//   * stores are non-temporal: 256 tiles are 32 MB, more than the L2 keeps for whoever reads them (with ordinary stores 5 % slower).
// Bound by the card's power where K is long: 75,600 x 5,120 x 13,824 with the gated residual in 2.15 - 2.30 ms by the card, 4.7 - 5.0 PFLOP/s, 66 % of the cycles on the matrix pipe
// (1.6 GHz in the counters' run); a bare stream of these MFMAs on normally distributed blocks runs at 6.97 PFLOP/s (8.92 on zeros: the operands' power), 1.54 ms.  Where K is short, by the epilogue: at K = 1,536 the GELU's
// 48 VALU cycles an element are as much as the products' (290 us, 3.1 PFLOP/s, 37 % of the cycles on the matrix pipe).
#include "mxfp4.h"

#include <type_traits>

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

  // A workgroup takes every step-th tile of its XCD's contiguous range of ids; ids run through groups of `group` tile rows column by column, so that the
  // tiles that an XCD works on at a time share few panels
  const int tiles = tiles_y * tiles_x;
  const int xcd = blockIdx.x & 7, qt = tiles >> 3, rt = tiles & 7;
  const int first = xcd < rt ? xcd * (qt + 1) : rt * (qt + 1) + (xcd - rt) * qt, end = first + qt + (xcd < rt ? 1 : 0);
  const int step = ((int)gridDim.x >> 3) + (xcd < ((int)gridDim.x & 7) ? 1 : 0);
  int tile = first + (blockIdx.x >> 3);
  const int per_group = group * tiles_x;
  struct Tile {
    int y, x;   // in units of 256
  };
  auto decode = [&](int t) -> Tile {
    const int gi = t / per_group, fy = gi * group, gsz = min(tiles_y - fy, group), in_g = t - gi * per_group, x = in_g / gsz;
    return {__builtin_amdgcn_readfirstlane(fy + in_g - x * gsz), __builtin_amdgcn_readfirstlane(x)};
  };

  // DMA plan: piece i of wave w fills the 16-byte slots q = i * 256 + w * 64 + lane; image row q >> 3, physical chunk q & 7 = logical ^ ((row >> 1) & 7).
  // Rows past the matrix lie past the descriptor's end: zeros, never stored
  const int pitch = p.K / 2;
  uint32_t ofs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = i * 256 + tid;
    const int row = q >> 3, lch = (q & 7) ^ ((row >> 1) & 7);
    const int r = (row >> 7) * 128 + 8 * (row & 15) + ((row >> 4) & 7);
    ofs[i] = (uint32_t)r * (uint32_t)pitch + lch * 16;
    asm volatile("" : "+v"(ofs[i]));
  }
  const uint32_t smem_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 1024;
  const int nk = p.kt;
  // The streams of Y units, X units and scales run ahead of the products, through the stages of one tile after the other: the next tile's first stages are
  // on their way while this one's epilogue runs.  Past the last tile they stay at its last stage.
  struct Stream {
    const char* base;
    uint32_t rec;
    int tile, k;
  };
  auto enter = [&](Stream& st, int t, bool is_y) {
    const Tile at = decode(t);
    const int64_t r0 = (int64_t)(is_y ? at.y : at.x) * 256, rows = (is_y ? p.M : p.N) - r0;
    st.base = reinterpret_cast<const char*>(is_y ? p.A : p.W) + r0 * pitch;
    st.rec = (uint32_t)min(rows * pitch, (int64_t)0xffffff00);
    st.tile = t;
    st.k = 0;
  };
  auto advance = [&](Stream& st, bool is_y) {
    if (st.k + 1 < nk) {
      st.base += MXM_ROW;
      st.rec -= MXM_ROW;
      ++st.k;
    } else if (st.tile + step < end) {
      enter(st, st.tile + step, is_y);
    }
  };
  auto piece = [&](const Stream& st, uint32_t slot, int i) { mx_dma16(ofs[i], mx_rsrc(st.base, st.rec), smem_lds + slot + i * 4096); };
  // a lane's scales: 16 bytes a stage of each operand's 128-row panel
  struct Scales {
    const char *y, *x;
    int tile, k;
  };
  auto enter_scales = [&](Scales& st, int t) {
    const Tile at = decode(t);
    st.y = reinterpret_cast<const char*>(p.As) + min((int64_t)at.y * 2 + wy, (p.M - 1) >> 7) * nk * 1024;
    st.x = reinterpret_cast<const char*>(p.Ws) + min((int64_t)at.x * 2 + wx, (p.N - 1) >> 7) * nk * 1024;
    st.tile = t;
    st.k = 0;
  };
  auto advance_scales = [&](Scales& st) {
    if (st.k + 1 < nk) {
      st.y += 1024;
      st.x += 1024;
      ++st.k;
    } else if (st.tile + step < end) {
      enter_scales(st, st.tile + step);
    }
  };
  auto scale_of = [&](const char* q) { return *reinterpret_cast<const mx_u4*>(q + lane * 16); };

  // fragment addresses: one base per (operand, k-step), the tiles 2 KB apart
  const int sw = (l15 >> 1) & 7;
  uint32_t ybw[2], xbw[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    ybw[ks] = (uint32_t)(((wy * 128 + l15) * 128 + ((lg ^ sw) << 4)) ^ (ks << 6));
    xbw[ks] = (uint32_t)(((wx * 128 + l15) * 128 + ((lg ^ sw) << 4)) ^ (ks << 6));
  }
  auto load_frag = [&](MxmFrags& f, uint32_t ya, uint32_t xa, int r) {
    if (r < 8) f.y[r] = *(mxm_lds_u4*)(lds + ya + r * 2048);
    else f.x[r - 8] = *(mxm_lds_u4*)(lds + xa + (r - 8) * 2048);
  };
  // the order of a k-step's 16 fragment reads: y 1 .. 7, x 1 .. 7, x 0, y 0 -- what its first MFMA needs comes last, so that ONE wait covers all
  auto ord = [](int i) constexpr { return i < 7 ? 1 + i : i < 14 ? 2 + i : i == 14 ? 8 : 0; };
  auto next_slot = [](uint32_t s) -> uint32_t { return s + MXM_UNIT == MXM_NU * MXM_UNIT ? 0u : s + MXM_UNIT; };

  Stream ys, xs;
  Scales ss;
  enter(ys, tile, true);
  enter(xs, tile, false);
  enter_scales(ss, tile);
  mx_u4 sy = scale_of(ss.y), sx = scale_of(ss.x);
  advance_scales(ss);
  mx_u4 ny = scale_of(ss.y), nx = scale_of(ss.x);   // the next stage's
  asm volatile("" : "+v"(sy), "+v"(sx), "+v"(ny), "+v"(nx));
  advance_scales(ss);
#pragma unroll
  for (int u = 0; u < 5; ++u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) piece((u & 1) ? xs : ys, u * MXM_UNIT, i);
    if (u & 1) advance(xs, false);
    else advance(ys, true);
  }
  asm volatile("s_waitcnt vmcnt(8)" ::: "memory");   // stages 0 and 1 landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  MxmFrags f0, f1;
#pragma unroll
  for (int r = 0; r < 16; ++r) load_frag(f0, ybw[0], xbw[0] + MXM_UNIT, ord(r));
  uint32_t slot_y = 0, slot_x = MXM_UNIT;   // of the current stage
  uint32_t y1 = ybw[1], x1 = xbw[1] + MXM_UNIT, yn = 0, xn = 0;   // its k-step 1's fragments, the next stage's k-step 0's
  auto load_bias = [&](int64_t x) -> uint4 {   // of this lane's columns
    const int64_t c = x + wx * 128 + 8 * l15;
    return EPI != WAN_EPI_TRANSPOSED && p.bias != nullptr && c + 8 <= p.N ? *reinterpret_cast<const uint4*>(p.bias + c) : make_uint4(0u, 0u, 0u, 0u);
  };
  Tile at = decode(tile);
  uint4 bias = load_bias((int64_t)at.x * MXM_BN);
  asm volatile("" : "+v"(bias.x), "+v"(bias.y), "+v"(bias.z), "+v"(bias.w));   // (waited for here: in the loop hipcc then waits for what is older than the stores)
  for (;;) {
    f32x4 acc[8][8];
    {
      float bcol[8];   // the sums start at the bias of their column: an addition an element less in the epilogue
      unpack8(bias, bcol);
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          acc[a][b] = f32x4{bcol[b], bcol[b], bcol[b], bcol[b]};
          asm volatile("" : "+a"(acc[a][b]));
        }
    }
    asm volatile("s_nop 1" ::: "memory");   // (in front of the first MFMA that reads them: hipcc pads nothing around asm)
    // Stage S: Y in slot 2 S % 5, X in (2 S + 1) % 5 (S counted over the tiles).
    //   k-step 0 (f0): stage S + 1's scales behind MFMA 0, k-step 1's fragments behind MFMA 1, 3, .., 31
    //   k-step 1 (f1): MFMAs 0 .. 15 bare
    //   P_S: everything landed, stage S fully read + barrier
    //   MFMAs 16 .. 63: X_{S+2} -> slot of Y_S behind 16, 19, .., 37, Y_{S+3} -> slot of X_S behind 40, 43, .., 61; stage S + 1's first fragments
    //                   in the other gaps up to MFMA 39
    // What a stage leaves to the next one is moved in the gaps too: between the stages it would hold the MFMAs up.
    // A tile's first stage has its successor's scales and units from in front of the epilogue, and waits for no store of it: what is waited for is older than the
    // 32 stores (in front of the first tile there are none, and nothing is waited for that has not landed).
    auto stage = [&](auto is_first) __attribute__((always_inline)) {
      constexpr bool FIRST = decltype(is_first)::value;
      uint32_t next_y, next_x;
      mxm_run<0, 0, 64>(acc, f0, sy, sx, [&](int m) __attribute__((always_inline)) {
        if (!FIRST && m == 0) {
          sy[2] = ny[2]; sy[3] = ny[3]; sx[2] = nx[2]; sx[3] = nx[3];
          ny = scale_of(ss.y);
          nx = scale_of(ss.x);
        }
        if ((m & 1) == 1 && m < 32) load_frag(f1, y1, x1, ord(m >> 1));
        if (m == 34) next_y = next_slot(slot_x);
        if (m == 36) next_x = next_slot(next_y);
        if (m == 38) { yn = ybw[0] + next_y; xn = xbw[0] + next_x; }
        if (m == 40) { y1 = ybw[1] + next_y; x1 = xbw[1] + next_x; }
        if (!FIRST && m == 44) advance_scales(ss);
      });
      mxm_run<1, 0, 16>(acc, f1, sy, sx, [](int) {});
      if (FIRST) asm volatile("s_waitcnt vmcnt(32) lgkmcnt(0)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" : "+v"(ny), "+v"(nx)::"memory");
      mxm_run<1, 16, 64>(acc, f1, sy, sx, [&](int m) __attribute__((always_inline)) {
        const int q = (m - 16) / 3, r = (m - 16) % 3;
        if (r == 0 && q < 8) piece(xs, slot_y, q);
        if (r == 0 && q >= 8) piece(ys, slot_x, q - 8);
        if (r != 0 && q < 8) load_frag(f0, yn, xn, ord(2 * q + r - 1));
        if (m == 42) advance(xs, false);
        if (m == 45) { sy[0] = ny[0]; sy[1] = ny[1]; sx[0] = nx[0]; sx[1] = nx[1]; }
        if (m == 62) {
          advance(ys, true);
          slot_y = next_y;
          slot_x = next_x;
        }
      });
    };
    stage(std::true_type{});
#pragma unroll 1
    for (int k = 1; k < nk; ++k) stage(std::false_type{});
    // the last MFMAs -> accumulator reads
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    sy[2] = ny[2]; sy[3] = ny[3]; sx[2] = nx[2]; sx[3] = nx[3];
    ny = scale_of(ss.y);
    nx = scale_of(ss.x);
    advance_scales(ss);
    const int64_t y0 = (int64_t)at.y * MXM_BM, x0 = (int64_t)at.x * MXM_BN;
    tile += step;
    if (tile < end) {
      at = decode(tile);
      bias = load_bias((int64_t)at.x * MXM_BN);
    }

    // ---- epilogue: straight from the registers.  The descriptors end with the tile's last column of the matrix's last row: what a row past the matrix would store
    // (or read of the residual) begins a whole pitch behind that row's start, and ldc >= N is no less than the tile's columns, however few they are.  A lane's 8
    // columns are inside or outside as a whole (N % 8 == 0), outside: an offset past num_records ----------------------------------------------------------------
    // (its arguments are read from the kernel's again: held across the loop they take the scalar registers that the streams need)
    typedef __attribute__((address_space(4))) const MxGemm mxm_args;
    mxm_args* pe = (mxm_args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(pe));
    uint32_t lane_e;  // an opaque lane id: derived from threadIdx the epilogue's offsets are hoisted in front of the MFMA loop and spilled
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
    const uint32_t ne = lane_e & 15u, ge = lane_e >> 4;
    const uint32_t colb = (uint32_t)(wx * 128) * 2u + ne * 16u;
    const int64_t rows_valid = min(pe->M - y0, (int64_t)MXM_BM);
    const uint32_t onum = (uint32_t)((rows_valid - 1) * pe->ldc * 2 + min(pe->N - x0, (int64_t)MXM_BN) * 2);
    const uint32_t ldo2 = (uint32_t)(pe->ldc * 2);
    const __amdgpu_buffer_rsrc_t odesc = __builtin_amdgcn_make_buffer_rsrc((void*)(pe->C + y0 * pe->ldc + x0), 0, (int)onum, 0x00020000);
    const __amdgpu_buffer_rsrc_t rdesc = __builtin_amdgcn_make_buffer_rsrc((void*)((EPI == WAN_EPI_GATE_RES ? pe->R : pe->C) + y0 * pe->ldc + x0), 0, (int)onum, 0x00020000);
    const uint32_t row_lane = (uint32_t)(wy * 128) + 32u * ge;
    const bool col_in = x0 + wx * 128 + 8 * (int64_t)ne + 8 <= pe->N;
    const uint32_t lane_off = col_in ? row_lane * ldo2 + colb : 0x80000000u;
    // gates: a 256-row tile touches at most two batches (rows_per_batch >= 256)
    float gA[8], gB[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) gA[j] = gB[j] = 1.f;
    uint32_t rb = 0xffffffffu;
    auto gate_row = [&](int64_t bidx, float* gq) {
      float mv[8], ev[8];
      unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(pe->mod + (int64_t)pe->gate_idx * pe->N + x0) + colb), mv);
      unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(pe->e + (bidx * pe->n_mod + pe->gate_idx) * pe->N + x0) + colb), ev);
#pragma unroll
      for (int j = 0; j < 8; ++j) gq[j] = mv[j] + ev[j];
    };
    if (EPI == WAN_EPI_GATE_RES && pe->gate_idx >= 0 && col_in) {
      const int64_t b0 = y0 / pe->rows_per_batch;
      const int64_t yb = (b0 + 1) * pe->rows_per_batch;
      gate_row(b0, gA);
      if (yb < y0 + rows_valid) {
        rb = (uint32_t)(yb - y0);
        gate_row(b0 + 1, gB);
      }
    }
    typedef unsigned int mxm_st4 __attribute__((__vector_size__(16)));
    uint32_t brow[32] = {};   // the bias along the rows: all of it in front of the stores, which a load behind them would wait for
    if (EPI == WAN_EPI_TRANSPOSED && pe->bias != nullptr) {
#pragma unroll
      for (int r = 0; r < 32; ++r) brow[r] = pe->bias[min(y0 + row_lane + r, pe->M - 1)];
    }
    uint32_t ro[4];   // rows 8 i + a of the current a
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ro[i] = lane_off + (uint32_t)(8 * i) * ldo2;
      asm volatile("" : "+v"(ro[i]));
    }
    auto rload = [&](int ahead, int i) -> uint4 {
      return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rdesc, (int)(ro[i] + (uint32_t)ahead * ldo2), 0, 0));
    };
    uint4 rq[3][4] = {};   // residual rows of the next two y tiles are in flight while one is converted
    if (EPI == WAN_EPI_GATE_RES) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { rq[0][i] = rload(0, i); rq[1][i] = rload(1, i); }
    }
#pragma unroll
    for (int a = 0; a < 8; ++a) {
#pragma unroll
      for (int t = 0; t < 8; ++t) asm volatile("" : "+a"(acc[a][t]));   // (read here, not all 256 in front of the rows)
      if (EPI == WAN_EPI_GATE_RES && a + 2 < 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) rq[(a + 2) % 3][i] = rload(2, i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t rit = (uint32_t)(8 * i + a);
        float v[8], rv[8];
        if (EPI == WAN_EPI_GATE_RES) unpack8(rq[a % 3][i], rv);
        const bool second = row_lane + rit >= rb;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          float o = acc[a][t][i];
          if (EPI == WAN_EPI_TRANSPOSED) o += __uint_as_float(brow[rit] << 16);
          if (EPI == WAN_EPI_GELU_TANH) o = mx_gelu_tanh(o);
          if (EPI == WAN_EPI_GATE_RES) o = __builtin_fmaf(o, second ? gB[t] : gA[t], rv[t]);
          v[t] = o;
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(mxm_st4, pack8(v)), odesc, (int)ro[i], 0, 2);
        ro[i] += ldo2;
        asm volatile("" : "+v"(ro[i]));
        if (EPI == WAN_EPI_GELU_TANH) __builtin_amdgcn_sched_barrier(0);  // 8 GELUs' temporaries at a time
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (tile >= end) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // trailing DMA (the LDS is released at the end)
}

}  // namespace

// -1: the problem does not fit this kernel (gemm_mxfp4.hip's takes it)
int wan_gemm_mxfp4m_try(const MxGemm& p, int epilogue, hipStream_t st) {
  // A lane stores 8 columns or none; what the transposed form would store past the tokens lies in the caller's padding, which stays as it was.  So tokens that are no multiple of
  // 8 take the 128-row tiles: V^T of 75,600 and 75,597 tokens x 5,120 x 5,120 945 and 1,950 us, of 32,760 and 32,757 x 1,536 x 1,536 50 and 131.
  if (p.N % 8 != 0 || p.ldc % 8 != 0) return -1;
  if (((uintptr_t)p.C | (uintptr_t)p.R | (uintptr_t)p.mod | (uintptr_t)p.e) & 15) return -1;
  if (epilogue != WAN_EPI_TRANSPOSED && ((uintptr_t)p.bias & 15)) return -1;
  if (epilogue == WAN_EPI_GATE_RES && p.gate_idx >= 0 && p.rows_per_batch < MXM_BM) return -1;
  if (256 * (int64_t)(p.K / 2) + 256 >= ((int64_t)1 << 31) || 256 * p.ldc * 2 + 512 >= ((int64_t)1 << 31)) return -1;   // 32-bit offsets inside a tile
  const int64_t ty = (p.M + MXM_BM - 1) / MXM_BM, tx = (p.N + MXM_BN - 1) / MXM_BN;
  if (ty * tx >= ((int64_t)1 << 31)) return -1;
  const dim3 grid((unsigned)min(ty * tx, (int64_t)256)), wg(256);   // one workgroup a CU
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
