// Block-sparse attention for gfx950: blocks of 128 queries, each with a list of blocks of 64 keys (wan_select_blocks).
//   O_i = sum_j softmax_j(q_i k_j / sqrt(128)) v_j over the keys j of the listed blocks that lie below the batch's length
// bf16 in / out, fp32 statistics and accumulators, head dimension 128, V transposed as wan_attention takes it.
//
// Layout (lane: n = lane & 15, g = lane >> 4), on v_mfma_f32_16x16x32_bf16 as attention_w16n.hip:
//   S^T = K Q^T     register i of tile (kt, qt) = the score of q row 16 qt + n against LDS row 16 kt + 4 g + i of the K image
//   O^T = V^T P^T   register i of tile (dt, qt) = O[16 qt + n][16 dt + 4 g + i]
// LDS row 16 kt + m of the K image holds key 32 (kt >> 1) + 8 (m >> 2) + 4 (kt & 1) + (m & 3), so that a lane's scores of two S tiles are the 8
// consecutive keys it has to supply as the P^T operand: P never moves between lanes.
#include "attn_w64_shared.h"

namespace {

constexpr int Q_BLOCK = 128, FEW = 16;
constexpr float LAZY = 32.f;   // how far above its reference (log2) a row's scores may lie
constexpr float SPARSE_SCALE_LOG2E = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)

// ---- 2 waves x 64 queries ----------------------------------------------------------------------------------------------------------------------
// One wave per SIMD with the whole register file, its instruction stream laid out by hand as attention_w16n.hip's: 128 MFMAs of 16 cycles a tile
// (A 0 .. 31: S_a, B 32 .. 63: PV_b of the tile before, C 64 .. 95: S_b, D 96 .. 127: PV_a; a, b: the wave's q tiles 0, 1 and 2, 3), one gap of up
// to four issue slots behind each.  What is different here:
//   * two waves to a list, so that a block of 128 queries has a list of its own, and two such workgroups to a CU: 80 KB of LDS each, K in a ring of
//     two images and V^T in one of three (K(t) is in registers by the time K(t + 2) is fetched, V^T(t) is read in the middle of tile t);
//   * the tiles' addresses come from the list, one scalar load a tile ahead of its use;
//   * the softmax needs no bound on the scores: a half's maximum is taken (v_max3) between its last S tile and its first exp2, and only a score 2^LAZY
//     above the row's reference, the first tile and tiles that end inside leave the straight path (sp_cold).
//   * q is not scaled in front: rounded with the scale in it every score would be off by 2^-9 of its terms (outputs 0.0028 from the exact ones where now it is
//     0.0023, and the rounding of the outputs alone 0.0017).  The multiplication per score costs 4 % of a large call.
//   * the weights are rounded to bf16 (2^-8 each), which is what the product with V takes, and summed so rounded.  Two terms, the second what the first leaves, would
//     bring the outputs to their own rounding for half as many MFMAs again, and make NaN of an infinity in V (times a second term of 0 or less) where one term keeps it.
// Bound inside the CU: 75,600 tokens of 40 heads with 148 of 1,182 blocks each in 11.8 to 13.1 ms by the card, 1.12 to 1.24 PFLOP/s, the matrix pipe busy for 64 % of the cycles (1.77 GHz in
// the counters' run).  32,760 tokens of 12 heads, 64 blocks: 682 to 738 us, 59 %.  (The queries' sixteen loads one behind the other in front of the first tile cost
// 1 % of the one and 2 % of the other.)
// Gap plan (even gaps: one exp2 each): exp2 of a's score k behind MFMA 52 + 2 k, of b's behind 116 + 2 k, running into the next tile (k = 6 behind its
// MFMA 0); a score is multiplied in the odd gap in front of its exp2, a pair packed in the odd gap behind its second, fragments summed by one MFMA more behind
// the last product of each; maxima of a in the odd gaps 29 .. 51, of b 93 .. 115; DMA of tile
// t + 2 in every eighth gap, K from 3, V^T from 65 (the m0 of each in the gap in front of it): 64 pieces of 1 KB a CU and tile keep the path into the LDS
// busy for 1,024 cycles, and issued in a row they hold up the waves; V^T(t) fragments 41 .. 71, K(t + 1) fragments 67 .. 97; the
// addresses of tile t + 3 in the even gaps 112 .. 124.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct SHalf {
  f32x4 accO[8][2];   // O^T tiles [d tile][q tile]
  f32x4 s[4][2];      // S^T - m [kv tile][q tile]
  u32x4 pk[4];        // P^T fragments, f = 2 c + q tile
  float t;            // the score whose exp2 is next
  float p0, p1;       // the exp2 pair whose pack is pending
  f32x4 l[2];         // the row sums (all four registers the same), on the matrix pipe: a row of ones as one more row of V^T
  float top[2];       // maxima of the current tile
};
__device__ __forceinline__ void sp_qk0(f32x4& d, const mfma_bf16x8& k, const mfma_bf16x8& q, const f32x4& c) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %3" : "=&v"(d) : "v"(k), "a"(q), "v"(c));
}
__device__ __forceinline__ void sp_qk(f32x4& d, const mfma_bf16x8& k, const mfma_bf16x8& q) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(k), "a"(q));
}
__device__ __forceinline__ void sp_pv(f32x4& acc, const mfma_bf16x8& v, const mfma_bf16x8& p) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "a"(v), "v"(p));
}
// MFMA i = 0 .. 31 of an S phase: k-step i >> 3, kv tile (i >> 1) & 3, q tile i & 1; of a PV phase: fragment f = i >> 3, d tile i & 7
__device__ __forceinline__ void sp_s_step(SHalf& x, const mfma_bf16x8 (&kf)[4][4], const mfma_bf16x8 (&qf)[4][4], const f32x4 (&negm)[4], int qt0, int i) {
  const int ks = i >> 3, kt = (i >> 1) & 3, qt = i & 1;
  if (ks == 0) sp_qk0(x.s[kt][qt], kf[kt][0], qf[qt0 + qt][0], negm[qt0 + qt]);
  else sp_qk(x.s[kt][qt], kf[kt][ks], qf[qt0 + qt][ks]);
}
__device__ __forceinline__ void sp_pv_step(SHalf& x, const mfma_bf16x8 (&vf)[8][2], int i) {
  const int f = i >> 3, dt = i & 7;
  sp_pv(x.accO[dt][f & 1], vf[dt][f >> 1], __builtin_bit_cast(mfma_bf16x8, x.pk[f]));
}
// score k = 0 .. 31 of a half in the order its fragments are needed: f = k >> 3, then kv tile parity, then register
__device__ __forceinline__ float sp_score(const SHalf& x, int k) {
  const int f = k >> 3;
  return x.s[2 * (f >> 1) + ((k >> 2) & 1)][f & 1][k & 3];
}
__device__ __forceinline__ void sp_scale(SHalf& x, int k, float scale) {
  x.t = sp_score(x, k) * scale;
  asm volatile("" : "+v"(x.t));
}
__device__ __forceinline__ void sp_exp(SHalf& x, int k) {
  float& p = (k & 1) ? x.p1 : x.p0;
  p = __builtin_amdgcn_exp2f(x.t);
  asm volatile("" : "+v"(p));
}
__device__ __forceinline__ void sp_pack(SHalf& x, int k) {   // behind the odd score k
  const int j = k >> 1;
  x.pk[j >> 2][j & 3] = cvt_pk(x.p0, x.p1);
  asm volatile("" : "+v"(x.pk[j >> 2]));
}
// fragment f's weights into their rows' sums.  (An addition per score costs 256 issue cycles a tile, these eight MFMAs 64; v_dot2_f32_bf16 over the packed pairs is as few
// instructions as half the additions and cost 400 cycles a tile more.)
__device__ __forceinline__ void sp_sum_step(SHalf& x, const mfma_bf16x8& ones, int f) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(x.l[f & 1]) : "v"(ones), "v"(__builtin_bit_cast(mfma_bf16x8, x.pk[f])));
}
// step j = 0 .. 7 of the maximum over a q tile's 16 scores, in the order the S tiles are finished
template <int J>
__device__ __forceinline__ void sp_max(SHalf& x, int qt) {
  // (asm: fmaxf of values that hipcc has not seen computed comes with a v_max x, x in front)
  if constexpr (J == 0) asm volatile("v_max3_f32 %0, %1, %2, %3" : "=v"(x.top[qt]) : "v"(x.s[0][qt][0]), "v"(x.s[0][qt][1]), "v"(x.s[0][qt][2]));
  else if constexpr (J < 7) {
    constexpr int A = 2 * J + 1, B = 2 * J + 2;
    asm volatile("v_max3_f32 %0, %0, %1, %2" : "+v"(x.top[qt]) : "v"(x.s[A >> 2][qt][A & 3]), "v"(x.s[B >> 2][qt][B & 3]));
  } else asm volatile("v_max_f32 %0, %0, %1" : "+v"(x.top[qt]) : "v"(x.s[3][qt][3]));
}
// The lane's number, opaque: what the rare paths and the epilogue derive from it is not computed ahead of the tile loop and kept in registers
__device__ __forceinline__ uint32_t sp_lane() {
  uint32_t lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}
// step T = 0 .. 11 of both q tiles' maxima: one operation a gap while tiles are being finished, two from the ninth on
template <int T>
__device__ __forceinline__ void sp_maxes(SHalf& x) {
  if constexpr (T < 8) sp_max<T / 2>(x, T & 1);
  else {
    sp_max<T - 4>(x, 0);
    sp_max<T - 4>(x, 1);
  }
}
// What leaves the straight path: the scores of a tile's keys past the end become -inf, and a row's reference moves to its maximum -- for the first
// time (the row sum is 0: until a key has a finite score the reference is 0 and waits), or because a score lies more than 2^LAZY above it.
// Returns whether a row still waits.
__device__ __forceinline__ int sp_cold(SHalf& x, f32x4* negm, int rem, float scale, float lazy) {
  bool open = false;
  const int lim = rem - 8 * (int)(sp_lane() >> 4);
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    float t = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.s[kt][qt][i] = 32 * (kt >> 1) + 4 * (kt & 1) + i >= lim ? -INFINITY : x.s[kt][qt][i];
        asm volatile("" : "+v"(x.s[kt][qt][i]));
        t = fmaxf(t, x.s[kt][qt][i]);
      }
    t = fmaxf(t, __shfl_xor(t, 16, 64));
    t = fmaxf(t, __shfl_xor(t, 32, 64));
    const bool first = x.l[qt][0] == 0.f, none = t == -INFINITY;
    open |= first && none;
    if (none || (!first && t <= lazy)) t = 0.f;
    const float a = __builtin_amdgcn_exp2f(-fmaxf(t, 0.f) * scale);   // (a first reference below 0: there is nothing to scale yet)
    x.l[qt] *= a;
#pragma unroll
    for (int i = 0; i < 4; ++i) negm[qt][i] -= t;
    asm volatile("" : "+v"(negm[qt]), "+v"(x.l[qt]));
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      x.s[kt][qt] -= t;
      asm volatile("" : "+v"(x.s[kt][qt]));
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {   // one tile at a time, in the accumulator file before and after
      asm volatile("" : "+a"(x.accO[dt][qt]));
      x.accO[dt][qt] *= a;
      asm volatile("" : "+a"(x.accO[dt][qt]));
    }
  }
  return __any(open) ? 1 : 0;
}

// the tiles of a list: addresses of the one to fetch next, and how many keys the tiles in flight hold.  All of it is the same for the whole wave and has to
// live in scalar registers (`uni`, and the list behind a constant-address-space pointer: scalar loads)
struct SpList {
  const __attribute__((address_space(4))) int* p;
  int pos, last;                                   // the entry to load, the list's last one (loaded again behind it)
  int nxt;                                         // the entry loaded last
  const char *kb, *vb;
  uint32_t rs2;
  int len, nvalid;
  const char *ka, *va;                             // of the tile that is fetched next
  uint32_t krec, vrec;
  int rem0, rem1, rem2, rem3;                      // keys of tiles t, t + 1, ..
  int blk;
};
// nxt -> addresses, in steps that fit the gaps of the tile before; an entry that names no block: no keys, and nothing is read.  (The empty asm statements keep
// each step's result in scalar registers and in its gap: hipcc would otherwise do all of it, on the vector ALU, in front of the first use.)
__device__ __forceinline__ void sp_apply_block(SpList& d) {
  const bool ok = (uint32_t)d.nxt < (uint32_t)d.nvalid;
  d.blk = ok ? d.nxt : 0;
  d.rem3 = ok ? d.len - d.nxt * KVBLK : 0;      // (0 or more than 0: also what says whether the entry names a block)
  asm volatile("" : "+s"(d.blk), "+s"(d.rem3));
}
__device__ __forceinline__ void sp_apply_k(SpList& d) {
  d.ka = d.kb + (uint64_t)(uint32_t)d.blk * (uint64_t)(KVBLK * d.rs2);
  asm volatile("" : "+s"(d.ka));
}
__device__ __forceinline__ void sp_apply_rows(SpList& d) {
  const int rows = d.rem3 < KVBLK ? d.rem3 : KVBLK;
  d.krec = d.rem3 > 0 ? (uint32_t)(rows - 1) * d.rs2 + 256u : 0u;   // rows past the last key read as zeros
  asm volatile("" : "+s"(d.krec));
}
__device__ __forceinline__ void sp_apply_v(SpList& d) {
  d.va = d.vb + (uint64_t)(uint32_t)d.blk * (KVBLK * 2);
  d.vrec = d.rem3 > 0 ? 0xfffffff0u : 0u;   // (all ones and 0 would be a sign extension of the condition, which hipcc makes in vector registers)
  asm volatile("" : "+s"(d.va), "+s"(d.vrec));
}
__device__ __forceinline__ void sp_apply(SpList& d) { sp_apply_block(d); sp_apply_k(d); sp_apply_rows(d); sp_apply_v(d); }
__device__ __forceinline__ void sp_load(SpList& d) {
  d.nxt = d.p[d.pos < d.last ? d.pos : d.last];
  d.pos += 1;
  asm volatile("" : "+s"(d.pos));
}

// The 16 DMA pieces of a wave for one tile, K and V^T in turn: 4 LDS rows of K (source rows permuted), 8 of V^T.  A piece of V^T is a
// lane offset and a scalar one; those of K, whose rows past the last key have to fail the range check, are lane offsets as a whole
struct SpDma {
  uint32_t kofs[8], vofs, lds0, ldv2;
  float scale, lazy;   // of the scores, in front of exp2; LAZY in their unit
};
// Two statements: the LDS address goes into m0 a gap ahead (nothing that hipcc emits in a tile touches m0; together they need an s_nop between them).  The
// sum is made on the way into m0: forty of them kept in scalar registers did not fit.
template <int KS, int VS, int I>
__device__ __forceinline__ void sp_m0(const SpDma& m) {
  constexpr int q = I >> 1, AT = (I & 1) == 0 ? KS * IMG + q * 2048 : (2 + VS) * IMG + q * 2048;   // K: LDS rows 8 q .. 8 q + 7 (both waves); V^T: rows 16 q .. 16 q + 15
  asm volatile("s_add_u32 m0, %0, %1" ::"s"(m.lds0), "n"(AT) : "scc", "memory");
}
__device__ __forceinline__ void sp_dma(uint32_t voff, const char* base, uint32_t num_records, uint32_t soff) {
  const uint64_t b = (uint64_t)base;
  dma_u4 r;
  r[0] = (uint32_t)b;
  r[1] = (uint32_t)(b >> 32) & 0xffffu;  // stride 0
  r[2] = num_records;                    // bytes from base that may be read; beyond: zeros
  r[3] = 0x00020000u;
  asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff) : "memory");
}
template <int I>
__device__ __forceinline__ void sp_piece(const SpDma& m, const SpList& d) {
  constexpr int q = I >> 1;
  if constexpr ((I & 1) == 0) sp_dma(m.kofs[q], d.ka, d.krec, 0u);
  else sp_dma(m.vofs, d.va, d.vrec, (uint32_t)(16 * q) * m.ldv2);
}
template <int KS, int VS, int I = 0>
__device__ __forceinline__ void sp_fetch(const SpDma& m, const SpList& d) {
  if constexpr (I < 16) {
    sp_m0<KS, VS, I>(m);
    asm volatile("s_nop 0");
    sp_piece<I>(m, d);
    sp_fetch<KS, VS, I + 1>(m, d);
  }
}

// the keys of a tile past the end: their V may hold anything, and 0 * anything has to be 0 (a tile without keys was filled with zeros)
__device__ __forceinline__ void sp_clean(char* img, int rem, int wave) {
  const int tid = wave * 64 + (int)sp_lane();
#pragma unroll 1
  for (int i = tid; i < 1024; i += 128) {
    const int row = i >> 3, lim = rem - (((i & 7) ^ ((row >> 1) & 7)) * 8);   // keys of this 16-byte chunk that stay
    u32x4* v = reinterpret_cast<u32x4*>(img + i * 16);
    u32x4 w = *v;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = lim >= 2 * j + 2 ? w[j] : lim == 2 * j + 1 ? w[j] & 0xffffu : 0u;
    *v = w;
  }
  __syncthreads();
}

// the MFMA of gap G and what sits behind it; KS, VS: the images of tile t (K read already, V^T read here)
template <int KS, int VS, int G>
__device__ __forceinline__ void sp_slot(lds_cchar* lds, const int (&kaddr)[4], const int (&vaddr)[2], const mfma_bf16x8 (&qf)[4][4], f32x4 (&negm)[4], mfma_bf16x8 (&kf)[4][4],
                                        mfma_bf16x8 (&vf)[8][2], const mfma_bf16x8& ones, SHalf& a, SHalf& b, const SpDma& m, SpList& d, int& force_a, int& force_b) {
  constexpr int KN = (KS ^ 1) * IMG, VB = (2 + VS) * IMG;
  if constexpr (G < 32) sp_s_step(a, kf, qf, negm, 0, G);
  else if constexpr (G < 64) sp_pv_step(b, vf, G - 32);
  else if constexpr (G < 96) sp_s_step(b, kf, qf, negm, 2, G - 64);
  else sp_pv_step(a, vf, G - 96);
  if constexpr (G >= 32 && G < 64 && (G & 7) == 7) sp_sum_step(b, ones, (G - 32) >> 3);
  if constexpr (G >= 96 && (G & 7) == 7) sp_sum_step(a, ones, (G - 96) >> 3);
  SB();
  if constexpr ((G & 1) == 0) {
    if constexpr (G <= 50) sp_exp(b, 6 + G / 2);
    else if constexpr (G <= 114) sp_exp(a, (G - 52) / 2);
    else sp_exp(b, (G - 116) / 2);
    if constexpr (G <= 58 && G % 8 == 2) sp_m0<KS, (VS + 2) % 3, G / 8 * 2>(m);
    if constexpr (G >= 64 && G % 8 == 0) sp_m0<KS, (VS + 2) % 3, (G - 64) / 8 * 2 + 1>(m);
    if constexpr (G == 34) sp_load(d);
    if constexpr (G == 112) sp_apply_block(d);
    if constexpr (G == 116) sp_apply_k(d);
    if constexpr (G == 118) sp_apply_rows(d);
    if constexpr (G == 124) sp_apply_v(d);
  } else {
    // behind an odd score its pair's pack
    constexpr int K = G <= 51 ? 6 + G / 2 : G <= 115 ? (G - 53) / 2 : (G - 117) / 2;
    SHalf& x = G > 51 && G <= 115 ? a : b;
    // the score whose exp2 is next: in front of the pack, a compiler's instruction there is the wait state that hipcc would otherwise fill with an s_nop (it does not count
    // the asm MFMA); where a tile may leave the straight path, behind that
    if constexpr (G <= 49) sp_scale(b, 6 + (G + 1) / 2, m.scale);
    else if constexpr (G == 127) sp_scale(b, 6, m.scale);
    else if constexpr (G > 51 && G <= 113) sp_scale(a, (G - 51) / 2, m.scale);
    else if constexpr (G > 115) sp_scale(b, (G - 115) / 2, m.scale);
    if constexpr ((K & 1) == 1) sp_pack(x, K);
    if constexpr (G >= 41 && G <= 55) vf[(G - 41) / 2][0] = *(lds_frag*)(lds + (VB + (G - 41) / 2 * 2048) + vaddr[0]);
    if constexpr (G >= 57 && G <= 71) vf[(G - 57) / 2][1] = *(lds_frag*)(lds + (VB + (G - 57) / 2 * 2048) + vaddr[1]);
    if constexpr (G >= 67 && G <= 97) {
      constexpr int R = (G - 67) / 2;
      kf[R & 3][R >> 2] = *(lds_frag*)(lds + (KN + (R & 3) * 4096) + kaddr[R >> 2]);
    }
    if constexpr (G <= 59 && G % 8 == 3) sp_piece<G / 8 * 2>(m, d);
    if constexpr (G >= 65 && G % 8 == 1) sp_piece<(G - 65) / 8 * 2 + 1>(m, d);
    if constexpr (G >= 29 && G <= 51) sp_maxes<(G - 29) / 2>(a);
    if constexpr (G >= 93 && G <= 115) sp_maxes<(G - 93) / 2>(b);
    if constexpr (G == 51) {
      const uint64_t need = __ballot(fmaxf(a.top[0], a.top[1]) > m.lazy) | (uint64_t)(force_a | (d.rem0 < KVBLK));
      if (__builtin_expect(need != 0, 0)) {
        asm volatile("" ::: "memory");
        force_a = sp_cold(a, &negm[0], d.rem0, m.scale, m.lazy);
      }
    }
    if constexpr (G == 115) {
      const uint64_t need = __ballot(fmaxf(b.top[0], b.top[1]) > m.lazy) | (uint64_t)(force_b | (d.rem0 < KVBLK));
      if (__builtin_expect(need != 0, 0)) {
        asm volatile("" ::: "memory");
        force_b = sp_cold(b, &negm[2], d.rem0, m.scale, m.lazy);
      }
    }
    if constexpr (G == 51) sp_scale(a, 0, m.scale);
    if constexpr (G == 115) sp_scale(b, 0, m.scale);
  }
  SB();
  if constexpr (G < 127) sp_slot<KS, VS, G + 1>(lds, kaddr, vaddr, qf, negm, kf, vf, ones, a, b, m, d, force_a, force_b);
}

struct SparseArgs {
  const bf16_t *q, *k, *vt;
  bf16_t* o;
  int64_t q_row, q_batch, k_row, k_batch, ldv, Lq, Lk;
  const int *index, *count, *k_lens;
  int B, Bk, H, Hk, nq, keep;
  int q_prescaled;
  int parts;
  int whole;      // the first lists of a launch in parts that are not cut
  int rows;       // of a list in part
  float* part;    // parts > 1: [cut list][part][rows][128] sums, behind them [cut list][part][rows] {reference, row sum}
};

// PARTS: the lists from `whole` on are cut into `parts` workgroups' shares, which leave unnormalised sums for sparse_join_kernel
template <bool PARTS>
__global__ __launch_bounds__(128, 1) void attn_sparse_kernel(SparseArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[5 * IMG];   // K 0, 1, V^T 0, 1, 2
  lds_cchar* lds = (lds_cchar*)smem;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // an XCD gets runs of neighbouring blocks of queries of a head: their lists have much in common
  const bool cut = PARTS && (int)blockIdx.x >= p.whole;
  const int wg = uni(PARTS ? (cut ? xcd_remap(blockIdx.x - p.whole, gridDim.x - p.whole) : xcd_remap(blockIdx.x, p.whole)) : xcd_remap(blockIdx.x, gridDim.x));
  const int own = cut ? uni(wg / p.parts) : wg, id = cut ? uni(p.whole + own) : wg, pt = cut ? wg - own * p.parts : 0;
  const int bh = uni(id / p.nq), qb = id - bh * p.nq, b = uni(bh / p.H), h = bh - b * p.H;
  const int bk = uni(b % p.Bk), hk = uni(h / (p.H / p.Hk));

  typedef const __attribute__((address_space(4))) int const_int;
  // what the prologue reads is on its way together: the count and the length, the queries, then the first entries of the list
  int entries = p.keep, len = (int)p.Lk;
  if (p.count != nullptr) entries = ((const_int*)p.count)[id];
  if (p.k_lens != nullptr) len = ((const_int*)p.k_lens)[bk];
  const int64_t q0 = (int64_t)qb * Q_BLOCK + wave * 64;
  mfma_bf16x8 qf[4][4];
#pragma unroll
  for (int qt = 0; qt < 4; ++qt) {
    const int64_t r = min(q0 + 16 * qt + n, p.Lq - 1);
    const bf16_t* qp = p.q + (int64_t)b * p.q_batch + r * p.q_row + (int64_t)h * 128 + g * 8;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[qt][ks] = *reinterpret_cast<const mfma_bf16x8*>(qp + 32 * ks);
  }
  SB();
  entries = min(p.keep, max(entries, 0));
  len = min((int)p.Lk, max(len, 0));
  SpList d;
  d.len = uni(len);
  d.nvalid = uni((len + KVBLK - 1) / KVBLK);
  int e0 = 0, e1 = entries;
  if (cut) {
    e0 = uni((int)((int64_t)entries * pt / p.parts));
    e1 = uni((int)((int64_t)entries * (pt + 1) / p.parts));
  }
  const int nt = d.nvalid > 0 ? uni(e1 - e0) : 0;

  SHalf x[2];
  f32x4 negm[4];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      negm[2 * c + qt] = f32x4{0.f, 0.f, 0.f, 0.f};
      x[c].l[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
      x[c].top[qt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        x[c].accO[dt][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
        asm volatile("" : "+a"(x[c].accO[dt][qt]));
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) x[c].s[kt][qt] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // (b's weights "of the tile before" the first: zeros)
    }
    x[c].p0 = x[c].p1 = 0.f;
    x[c].t = -INFINITY;
#pragma unroll
    for (int f = 0; f < 4; ++f) x[c].pk[f] = u32x4{0u, 0u, 0u, 0u};
  }
  if (nt > 0) {
    d.p = (const_int*)(p.index + (int64_t)id * p.keep + e0);
    d.last = nt - 1;
    d.pos = 0;
    d.rs2 = uni((uint32_t)(p.k_row * 2));
    d.kb = uni(reinterpret_cast<const char*>(p.k + (int64_t)bk * p.k_batch + (int64_t)hk * 128));
    d.vb = uni(reinterpret_cast<const char*>(p.vt + ((int64_t)bk * p.Hk + hk) * 128 * p.ldv));
    SpDma m;
    m.lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 1024;
    m.ldv2 = uni((uint32_t)(p.ldv * 2));
    m.scale = __uint_as_float(uni(__float_as_uint(p.q_prescaled ? 1.f : SPARSE_SCALE_LOG2E)));
    m.lazy = __uint_as_float(uni(__float_as_uint(p.q_prescaled ? LAZY : LAZY / SPARSE_SCALE_LOG2E)));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t r = 8u * (i & 1) + ((uint32_t)tid >> 4), kt = i >> 1;   // LDS row 16 kt + r
      m.kofs[i] = (32u * (kt >> 1) + 8u * (r >> 2) + 4u * (kt & 1) + (r & 3u)) * d.rs2 + (((uint32_t)tid & 15u) ^ r) * 16u;
    }
    m.vofs = ((uint32_t)tid >> 3) * m.ldv2 + ((((uint32_t)tid & 7u) ^ (((uint32_t)tid >> 4) & 7u)) << 4);
    const int first[3] = {d.p[0], d.p[min(1, d.last)], d.p[min(2, d.last)]};
    d.pos = 3;
    d.nxt = uni(first[0]); sp_apply(d);
    d.rem0 = d.rem3;
    sp_fetch<0, 0>(m, d);
    d.nxt = uni(first[1]); sp_apply(d);
    d.rem1 = d.rem3;
    sp_fetch<1, 1>(m, d);
    d.nxt = uni(first[2]); sp_apply(d);
    d.rem2 = d.rem3;

    mfma_bf16x8 kf[4][4], vf[8][2];
#pragma unroll
    for (int qt = 0; qt < 4; ++qt)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) asm volatile("" : "+a"(qf[qt][ks]));
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        vf[dt][c] = __builtin_bit_cast(mfma_bf16x8, make_uint4(0u, 0u, 0u, 0u));
        asm volatile("" : "+a"(vf[dt][c]));
      }
    int kaddr[4], vaddr[2];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) kaddr[ks] = n * 256 + (((4 * ks + g) ^ n) << 4);
#pragma unroll
    for (int c = 0; c < 2; ++c) vaddr[c] = n * 128 + (((4 * c + g) ^ ((n >> 1) & 7)) << 4);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < 16; ++r) kf[r & 3][r >> 2] = *(lds_frag*)(lds + (r & 3) * 4096 + kaddr[r >> 2]);

    mfma_bf16x8 ones = __builtin_bit_cast(mfma_bf16x8, make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
    asm volatile("" : "+v"(ones));
    int force_a = 1, force_b = 1;   // a row without a reference is left
#define SP_TILE(J)                                                                                                               \
    if (t + (J) >= nt) break;                                                                                                    \
    d.krec = uni(d.krec);                                         /* (carried around the loop hipcc puts them into vector registers) */ \
    d.rem0 = uni(d.rem0);                                                                                                        \
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");   /* V^T(t), K(t + 1) have landed, V^T(t + 1) may fly; tile t - 1 is read */ \
    __builtin_amdgcn_s_barrier();                                                                                                \
    asm volatile("" ::: "memory");                                                                                               \
    if (__builtin_expect(d.rem0 < KVBLK, 0)) sp_clean(smem + (2 + (J) % 3) * IMG, d.rem0, wave);                                  \
    sp_slot<(J) & 1, (J) % 3, 0>(lds, kaddr, vaddr, qf, negm, kf, vf, ones, x[0], x[1], m, d, force_a, force_b);                        \
    d.rem0 = d.rem1;                                                                                                             \
    d.rem1 = d.rem2;                                                                                                             \
    d.rem2 = d.rem3;
    for (int t = 0;; t += 6) {
      SP_TILE(0)
      SP_TILE(1)
      SP_TILE(2)
      SP_TILE(3)
      SP_TILE(4)
      SP_TILE(5)
    }
#undef SP_TILE
    // b's last weights and products
#pragma unroll
    for (int k = 6; k < 32; ++k) {
      if (k > 6) sp_scale(x[1], k, m.scale);
      sp_exp(x[1], k);
      asm volatile("s_nop 1");   // (no MFMA between the exp2 and its use here)
      if (k & 1) sp_pack(x[1], k);
    }
    asm volatile("s_nop 7" ::: "memory");
    SB();
#pragma unroll
    for (int i = 0; i < 32; ++i) { sp_pv_step(x[1], vf, i); SB(); }
#pragma unroll
    for (int f = 0; f < 4; ++f) { sp_sum_step(x[1], ones, f); SB(); }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");   // trailing DMA (the LDS is released at the end); the last MFMAs -> accumulator reads
  }
  const int lane_e = (int)sp_lane(), ne = lane_e & 15, ge = lane_e >> 4;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      const int row = wave * 64 + 32 * c + 16 * qt + ne;
      const float l = x[c].l[qt][0];
      if (cut) {
        if ((int64_t)qb * Q_BLOCK + row >= p.Lq) continue;   // (one query of a block: its row alone, not 64 KB of sums)
        float* o = p.part + ((int64_t)wg * Q_BLOCK + row) * 128 + 4 * ge;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<float4*>(o + 16 * dt) = make_float4(x[c].accO[dt][qt][0], x[c].accO[dt][qt][1], x[c].accO[dt][qt][2], x[c].accO[dt][qt][3]);
        if (ge == 0) {
          float2* st = reinterpret_cast<float2*>(p.part + (int64_t)(gridDim.x - p.whole) * Q_BLOCK * 128) + (int64_t)wg * Q_BLOCK + row;
          *st = make_float2(l == 0.f ? -INFINITY : -negm[2 * c + qt][0] * (p.q_prescaled ? 1.f : SPARSE_SCALE_LOG2E), l);
        }
        continue;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;   // a row without keys: zeros
      if ((int64_t)qb * Q_BLOCK + row < p.Lq) {
        bf16_t* op = p.o + ((int64_t)b * p.Lq + (int64_t)qb * Q_BLOCK + row) * p.H * 128 + (int64_t)h * 128 + 4 * ge;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          uint2 w;
          w.x = cvt_pk(x[c].accO[dt][qt][0] * inv, x[c].accO[dt][qt][1] * inv);
          w.y = cvt_pk(x[c].accO[dt][qt][2] * inv, x[c].accO[dt][qt][3] * inv);
          *reinterpret_cast<uint2*>(op + 16 * dt) = w;
        }
      }
    }
}

// ---- up to 16 queries ------------------------------------------------------------------------------------------------------------------------
// A token, or a handful: the cache's bytes and the latency are all there is.  A wave takes a block of 64 keys by itself, K and V^T straight from memory in
// the operands' layouts (the permuted key order of above: 16 rows x 64 bytes a load of K, 16 x 64 of V^T), all 32 KB of it in flight at once, and a
// workgroup's four waves join their sums in the LDS.  A list is cut into as many workgroups as leave a wave one block, up to 1,024 in all, then
// sparse_join_kernel as above.
// Bound by latency and by the way the bytes lie (rows of 256 bytes, of V^T 128): a token of 40 heads (8 of the cache) against 32 blocks each, 42 MB, in 12.6 us and 4
// for the join, the kernel above 18 and 5.  16 queries there: 17.7 and 23.5 us; 12 heads, 148 blocks each: 25.9 and 31.6; 1 head, 1,182: 38.8 and 67.0; 40 heads of their own
// caches, 148: 49.0 and 45.2; one query of 40 heads, 590: 112 and 114.
__global__ __launch_bounds__(256) void attn_sparse_few_kernel(SparseArgs p) {
  __shared__ __attribute__((aligned(16))) float sum[4][FEW][132];
  __shared__ float2 stat[4][FEW];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = blockIdx.x, id = wg / p.parts, pt = wg - id * p.parts;
  const int b = id / p.H, h = id - b * p.H, bk = b % p.Bk, hk = h / (p.H / p.Hk);
  // (the first entry is read with the count and the length, not behind them)
  const int* list = p.index + (int64_t)id * p.keep;
  int e = pt * 4 + wave, next = list[min(e, p.keep - 1)];
  int entries = p.keep;
  if (p.count != nullptr) entries = min(entries, max(p.count[id], 0));
  int len = (int)p.Lk;
  if (p.k_lens != nullptr) len = min(len, max(p.k_lens[bk], 0));
  const int nvalid = (len + KVBLK - 1) / KVBLK;

  mfma_bf16x8 qf[4];
  const bf16_t* qp = p.q + (int64_t)b * p.q_batch + (int64_t)min(n, (int)p.Lq - 1) * p.q_row + (int64_t)h * 128 + 8 * g;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) qf[ks] = *reinterpret_cast<const mfma_bf16x8*>(qp + 32 * ks);
  const float scale = p.q_prescaled ? 1.f : SPARSE_SCALE_LOG2E;
  const bf16_t* kb = p.k + (int64_t)bk * p.k_batch + (int64_t)hk * 128 + 8 * g;
  const bf16_t* vb = p.vt + (((int64_t)bk * p.Hk + hk) * 128 + n) * p.ldv + 8 * g;
  f32x4 acc[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, ref = 0.f, l = 0.f;   // the row's maximum so far, what its weights are relative to (0 until there is a maximum), this lane's share of its sum
  for (; e < entries; e += 4 * p.parts) {
    const int blk = __builtin_amdgcn_readfirstlane(next);
    next = list[min(e + 4 * p.parts, p.keep - 1)];
    if ((uint32_t)blk >= (uint32_t)nvalid) continue;
    const int rem = len - blk * KVBLK;   // keys from here on
    mfma_bf16x8 kf[4][4], vf[8][2];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const int key = min(32 * (kt >> 1) + 8 * (n >> 2) + 4 * (kt & 1) + (n & 3), rem - 1);   // (past the end: the last key again, masked below)
      const bf16_t* kr = kb + ((int64_t)blk * KVBLK + key) * p.k_row;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) kf[kt][ks] = *reinterpret_cast<const mfma_bf16x8*>(kr + 32 * ks);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int c = 0; c < 2; ++c) vf[dt][c] = *reinterpret_cast<const mfma_bf16x8*>(vb + (int64_t)(16 * dt) * p.ldv + blk * (int64_t)KVBLK + 32 * c);
    f32x4 s[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt][ks], qf[ks], s[kt], 0, 0, 0);
      s[kt] *= scale;
    }
    if (rem < KVBLK) {   // scores of keys past the end, and their V, which may hold anything: 0 * anything has to be 0
      const int lim = rem - 8 * g;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (32 * (kt >> 1) + 4 * (kt & 1) + i >= lim) s[kt][i] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          u32x4 w = __builtin_bit_cast(u32x4, vf[dt][c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int left = lim - 32 * c - 2 * j;
            const uint32_t x = w[j];
            w[j] = left >= 2 ? x : left == 1 ? x & 0xffffu : 0u;
          }
          vf[dt][c] = __builtin_bit_cast(mfma_bf16x8, w);
        }
    }
    float t = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) t = fmaxf(t, s[kt][i]);
    t = fmaxf(t, __shfl_xor(t, 16, 64));
    t = fmaxf(t, __shfl_xor(t, 32, 64));
    const float up = fmaxf(top, t);
    ref = up == -INFINITY ? 0.f : up;
    const float a = __builtin_amdgcn_exp2f(top - ref);
    top = up;
    l *= a;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt] *= a;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(s[2 * c + (j >> 2)][j & 3] - ref);
        l += w[j];
      }
      const mfma_bf16x8 pk = __builtin_bit_cast(mfma_bf16x8, pack8(w));   // (one bf16 term as above; the row sum takes the weights as they are)
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[dt][c], pk, acc[dt], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(&sum[wave][n][16 * dt + 4 * g]) = acc[dt];
  if (g == 0) stat[wave][n] = make_float2(l == 0.f ? -INFINITY : ref, l);
  __syncthreads();
  const int row = tid >> 4, col = (tid & 15) * 8;
  if (row >= p.Lq) return;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, stat[w][row].x);
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 ml = stat[w][row];
    const float a = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
    l += ml.y * a;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] += sum[w][row][col + j] * a;
  }
  if (p.parts > 1) {
    float* d = p.part + ((int64_t)wg * p.rows + row) * 128 + col;
    *reinterpret_cast<float4*>(d) = make_float4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<float4*>(d + 4) = make_float4(o[4], o[5], o[6], o[7]);
    if (col == 0) reinterpret_cast<float2*>(p.part + (int64_t)gridDim.x * p.rows * 128)[(int64_t)wg * p.rows + row] = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;   // a row without keys: zeros
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] *= inv;
  *reinterpret_cast<uint4*>(p.o + ((int64_t)b * p.Lq + row) * p.H * 128 + (int64_t)h * 128 + col) = pack8(o);
}

// o = sum of the parts' sums, each scaled from its own reference to the largest, over the row sums likewise: one wave per row, two columns a lane
__global__ __launch_bounds__(256) void sparse_join_kernel(SparseArgs p, int wgs) {
  const int id = blockIdx.x, row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;   // id: of the lists that were cut
  const int bh = (p.whole + id) / p.nq, qb = p.whole + id - bh * p.nq, b = bh / p.H, h = bh - b * p.H;
  const int64_t r = (int64_t)qb * Q_BLOCK + row;
  if (r >= p.Lq) return;
  const float2* st = reinterpret_cast<const float2*>(p.part + (int64_t)wgs * p.rows * 128) + (int64_t)id * p.parts * p.rows + row;
  const float2 ml = lane < p.parts ? st[lane * p.rows] : make_float2(-INFINITY, 0.f);   // (at most 64 parts)
  const float top = wave_max(ml.x);
  const float a = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
  const float l = wave_sum(ml.y * a);
  const float* o = p.part + ((int64_t)id * p.parts * p.rows + row) * 128 + 2 * lane;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll 8
  for (int k = 0; k < p.parts; ++k) {
    const float2 v = *reinterpret_cast<const float2*>(o + (int64_t)k * p.rows * 128);
    const float ak = __shfl(a, k, 64);
    s0 += v.x * ak;
    s1 += v.y * ak;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;   // a row without keys: zeros
  *reinterpret_cast<uint32_t*>(p.o + ((int64_t)b * p.Lq + r) * p.H * 128 + (int64_t)h * 128 + 2 * lane) = cvt_pk(s0 * inv, s1 * inv);
}

// How a launch's lists are cut.  Up to 16 queries: one workgroup for every four blocks of a list, up to 1,024 in all.  Else 512 workgroups run at a time, and what is left
// of the lists behind whole rounds of 512 is cut into the number of shares that takes the least time: what was measured is 1.4 us a block, and for shares 7 us for the join and
// 0.28 ns for each of a list's rows and shares (its partial sums are written and read), while all of them run at a time.  Lists x blocks, in us whole and in shares:
// 12 x 100 (64 queries each) 148, in 16 shares 30.4; 64 x 140 205, in 8 58.1, in 4 70.4; 96 x 32 57.3, in 4 38.1; 96 x 8 22.9, in 2 28.1; 36 x 4 14.4, in 2 16.4;
// 220 x 48 79.4, in 2 65.2, in 3 86.7; 516 x 64 with the last four in shares 138, at an earlier state 150 where it took 221 uncut; 756 x 64 191, then 206 and 225.
struct SparsePlan {
  int64_t whole, cut;
  int parts;
};
SparsePlan sparse_plan(int64_t Lq, int64_t lists, int keep) {
  const bool few = Lq <= FEW;
  const int64_t whole = few ? 0 : lists / 512 * 512, cut = lists - whole;
  int64_t n = 1;
  if (few) {
    n = 1024 / cut;
    if (n > (keep + 3) / 4) n = (keep + 3) / 4;
    if (n > 64) n = 64;
  } else if (cut > 0) {
    const double rows = (double)(cut * (Lq < Q_BLOCK ? Lq : Q_BLOCK));
    double best = 1.4 * keep;
    for (int k = 2; k <= 32 && k <= keep && k * cut <= 512; ++k) {
      const double t = 1.4 * ((keep + k - 1) / k) + 7.0 + 0.00028 * rows * k;
      if (t < best) { best = t; n = k; }
    }
  }
  if (n < 2) return {lists, 0, 1};
  return {whole, cut, (int)n};
}

}  // namespace

static bool sp_shares(const wan_bf16* o, int64_t o_elements, const wan_bf16* t, int64_t t_elements) {
  const uintptr_t a = (uintptr_t)o, b = (uintptr_t)t;
  return a < b + t_elements * 2 && b < a + o_elements * 2;
}

extern "C" int64_t wan_sparse_attention_scratch_bytes(int B, int64_t Lq, int H, int keep) {
  if (B < 1 || Lq < 1 || H < 1 || keep < 1) return 0;
  const int64_t lists = (Lq + Q_BLOCK - 1) / Q_BLOCK * H * B;
  const SparsePlan pl = sparse_plan(Lq, lists, keep);
  return pl.cut * pl.parts * (Lq <= FEW ? FEW : Q_BLOCK) * (128 + 2) * 4;
}

extern "C" int wan_sparse_attention(const wan_bf16* q, int64_t q_row, int64_t q_batch, const wan_bf16* k, int64_t k_row, int64_t k_batch, const wan_bf16* vt, wan_bf16* o,
                                    const int* index, const int* count, const int* k_lens, int B, int Bk, int64_t Lq, int64_t Lk, int64_t ldv, int H, int Hk, int keep,
                                    int q_prescaled, void* scratch, int64_t scratch_bytes, void* stream) {
  WAN_REQUIRE(q && k && vt && o && index, "wan_sparse_attention: null pointer");
  WAN_REQUIRE(B >= 1 && Bk >= 1 && B % Bk == 0, "wan_sparse_attention: Bk must divide B (B=%d Bk=%d)", B, Bk);
  WAN_REQUIRE(H >= 1 && Hk >= 1 && H % Hk == 0, "wan_sparse_attention: the heads of k must divide the heads of q (H=%d Hk=%d)", H, Hk);
  WAN_REQUIRE(Lq >= 1 && Lk >= 1 && keep >= 1, "wan_sparse_attention: empty problem (Lq=%lld Lk=%lld keep=%d)", (long long)Lq, (long long)Lk, keep);
  WAN_REQUIRE(ldv % KVBLK == 0 && ldv >= Lk, "wan_sparse_attention: ldv=%lld must be a multiple of 64 and >= Lk", (long long)ldv);
  WAN_REQUIRE(q_row >= (int64_t)H * 128 && k_row >= (int64_t)Hk * 128 && q_row % 8 == 0 && k_row % 8 == 0 && q_batch % 8 == 0 && k_batch % 8 == 0,
              "wan_sparse_attention: strides must be multiples of 8 elements, a row's at least its heads * 128");
  WAN_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)vt | (uintptr_t)o) & 15) == 0, "wan_sparse_attention: pointers must be 16-byte aligned");
  // a tile's 64 key rows and its 128 rows of V^T are addressed with 32-bit offsets from the tile's own 64-bit base
  WAN_REQUIRE(k_row < ((int64_t)1 << 24) && ldv < ((int64_t)1 << 23), "wan_sparse_attention: a row of k of %lld elements or %lld keys exceed the kernel's offsets", (long long)k_row, (long long)ldv);
  const int64_t nq = (Lq + Q_BLOCK - 1) / Q_BLOCK;
  WAN_REQUIRE(nq * H * B < ((int64_t)1 << 31) - 1024, "wan_sparse_attention: grid too large");
  const int64_t lists = nq * H * B;
  const SparsePlan pl = sparse_plan(Lq, lists, keep);
  const int64_t need = wan_sparse_attention_scratch_bytes(B, Lq, H, keep);
  WAN_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0), "wan_sparse_attention: needs 16-byte aligned scratch of %lld bytes", (long long)need);
  // one workgroup's output would be another's input (q itself is read by the workgroup alone that writes its place)
  const int64_t on = (int64_t)B * Lq * H * 128;
  WAN_REQUIRE(!sp_shares(o, on, k, (Bk - 1) * k_batch + (Lk - 1) * k_row + Hk * 128) && !sp_shares(o, on, vt, (int64_t)Bk * Hk * 128 * ldv),
              "wan_sparse_attention: the output must not overlap k or vt");
  WAN_REQUIRE(!sp_shares(o, on, q, (B - 1) * q_batch + (Lq - 1) * q_row + H * 128) || (o == q && (Lq == 1 || q_row == (int64_t)H * 128) && (B == 1 || q_batch == Lq * H * 128)),
              "wan_sparse_attention: an output that overlaps q must be q, contiguous");
  hipStream_t st = as_stream(stream);
  const SparseArgs a = {q, k, vt, o, q_row, q_batch, k_row, k_batch, ldv, Lq, Lk, index, count, k_lens, B, Bk, H, Hk, (int)nq, keep, q_prescaled, pl.parts, (int)pl.whole, Lq <= FEW ? FEW : Q_BLOCK, reinterpret_cast<float*>(scratch)};
  const unsigned wgs = (unsigned)(pl.whole + pl.cut * pl.parts);
  if (Lq <= FEW) {
    hipLaunchKernelGGL(attn_sparse_few_kernel, dim3(wgs), dim3(256), 0, st, a);
  } else if (pl.cut == 0) {
    hipLaunchKernelGGL(attn_sparse_kernel<false>, dim3(wgs), dim3(128), 0, st, a);
  } else {
    hipLaunchKernelGGL(attn_sparse_kernel<true>, dim3(wgs), dim3(128), 0, st, a);
  }
  if (pl.cut > 0) {
    WAN_LAUNCH_CHECK();
    const int64_t rows = Lq < Q_BLOCK ? Lq : Q_BLOCK;
    hipLaunchKernelGGL(sparse_join_kernel, dim3((unsigned)pl.cut, (unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, (int)(pl.cut * pl.parts));
  }
  WAN_LAUNCH_CHECK();
  return 0;
}
