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

constexpr int Q_BLOCK = 128;
constexpr float LAZY = 32.f;   // how far above its reference (log2) a row's scores may lie
constexpr float SPARSE_SCALE_LOG2E = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)

struct SparseArgs {
  const bf16_t *q, *k, *vt;
  bf16_t* o;
  int64_t q_row, q_batch, k_row, k_batch, ldv, Lq, Lk;
  const int *index, *count, *k_lens;
  int B, Bk, H, Hk, nq, keep;
  int q_prescaled;
};

__device__ __forceinline__ f32x4 mfma16(const mfma_bf16x8& a, const mfma_bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 4 waves x 32 queries, one list entry at a time, two stages of K / V^T in LDS
__global__ __launch_bounds__(256, 2) void attn_sparse_kernel(SparseArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[4 * IMG];   // K stage 0, 1, V^T stage 0, 1
  lds_cchar* lds = (lds_cchar*)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int bh = id / p.nq, qb = id - bh * p.nq, b = bh / p.H, h = bh - b * p.H;
  const int bk = b % p.Bk, hk = h / (p.H / p.Hk);
  const int* list = p.index + (int64_t)id * p.keep;
  int entries = p.keep;
  if (p.count != nullptr) entries = min(entries, max(p.count[id], 0));
  int len = (int)p.Lk;
  if (p.k_lens != nullptr) len = min(len, max(p.k_lens[bk], 0));
  const int nvalid = (len + KVBLK - 1) / KVBLK;
  const char* kb = reinterpret_cast<const char*>(p.k + (int64_t)bk * p.k_batch + (int64_t)hk * 128);
  const char* vb = reinterpret_cast<const char*>(p.vt + ((int64_t)bk * p.Hk + hk) * 128 * p.ldv);
  const uint32_t rs2 = (uint32_t)(p.k_row * 2), ldv2 = (uint32_t)(p.ldv * 2);

  uint32_t kofs[4], vofs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = (uint32_t)tid >> 4;
    kofs[i] = (32u * (i >> 1) + 8u * (m >> 2) + 4u * (i & 1) + (m & 3u)) * rs2 + (((uint32_t)tid & 15u) ^ m) * 16u;
    vofs[i] = (32u * i + ((uint32_t)tid >> 3)) * ldv2 + ((((uint32_t)tid & 7u) ^ (((uint32_t)tid >> 4) & 7u)) << 4);
  }
  auto fetch = [&](int blk, int st) {
    blk = __builtin_amdgcn_readfirstlane(blk);
    const int rows = min(KVBLK, len - blk * KVBLK);
    const char* ka = uni(kb + (int64_t)blk * KVBLK * rs2);
    const char* va = uni(vb + (int64_t)blk * KVBLK * 2);
    const uint32_t klen = uni((uint32_t)(rows - 1) * rs2 + 256u);     // rows past the last key read as zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      dma_issue(kofs[i], ka, klen, lds0 + st * IMG + wave * 1024 + i * 4096);
      dma_issue(vofs[i], va, 0xffffffffu, lds0 + (2 + st) * IMG + wave * 1024 + i * 4096);
    }
  };
  // the next entry that names a block with keys, from position e on
  auto next = [&](int e) {
    while (e < entries && (unsigned)list[e] >= (unsigned)nvalid) ++e;
    return e;
  };

  const int64_t q0 = (int64_t)qb * Q_BLOCK + wave * 32;
  mfma_bf16x8 qf[2][4];
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    const int64_t r = min(q0 + 16 * qt + n, p.Lq - 1);
    const bf16_t* qp = p.q + (int64_t)b * p.q_batch + r * p.q_row + (int64_t)h * 128 + g * 8;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint4 w = *reinterpret_cast<const uint4*>(qp + 32 * ks);
      if (!p.q_prescaled) {   // the scale folded into q and rounded with it (as the dense kernels do): no multiplication per score
        float f[8];
        unpack8(w, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= SPARSE_SCALE_LOG2E;
        w = pack8(f);
      }
      qf[qt][ks] = __builtin_bit_cast(mfma_bf16x8, w);
    }
  }
  const uint4 one_bits = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  const mfma_bf16x8 ones = __builtin_bit_cast(mfma_bf16x8, one_bits);
  f32x4 acc[8][2], l[2], negm[2];
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    l[qt] = negm[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool unset[2] = {true, true};   // the row has no reference yet

  int e = next(0), st = 0;
  if (e < entries) fetch(list[e], 0);
  bool force = true;
  while (e < entries) {
    const int blk = __builtin_amdgcn_readfirstlane(list[e]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    e = next(e + 1);
    if (e < entries) fetch(list[e], st ^ 1);
    const int rem = len - blk * KVBLK;
    if (rem < KVBLK) {   // the keys past the end: their V may hold anything, 0 * anything has to be 0
      for (int i = tid; i < 1024; i += 256) {
        const int row = i >> 3, lim = rem - (((i & 7) ^ ((row >> 1) & 7)) * 8);
        bf16_t* v = reinterpret_cast<bf16_t*>(smem + (2 + st) * IMG + i * 16);
        for (int j = max(lim, 0); j < 8; ++j) v[j] = 0;
      }
      __syncthreads();
    }
    // S - m: the reference enters as the C operand of each tile's first product
    f32x4 s[4][2];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const mfma_bf16x8 kf = *(lds_frag*)(lds + st * IMG + (16 * kt + n) * 256 + (((4 * ks + g) ^ n) << 4));
        s[kt][0] = mfma16(kf, qf[0][ks], ks == 0 ? negm[0] : s[kt][0]);
        s[kt][1] = mfma16(kf, qf[1][ks], ks == 0 ? negm[1] : s[kt][1]);
      }
    if (rem < KVBLK) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (32 * (kt >> 1) + 8 * g + 4 * (kt & 1) + i >= rem) s[kt][qt][i] = -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      top[qt] = fmaxf(s[0][qt][0], s[0][qt][1]);
#pragma unroll
      for (int k = 2; k < 16; k += 2) top[qt] = fmaxf(top[qt], fmaxf(s[k >> 2][qt][k & 3], s[(k + 1) >> 2][qt][(k + 1) & 3]));
    }
    // The reference m of a row follows its maximum only when a score lies more than 2^LAZY above it: until then the weights 2^(s - m) are merely
    // large numbers, which bf16 and fp32 carry with the same relative precision.  The first block sets it.
    if (force || __any(fmaxf(top[0], top[1]) > LAZY)) {
      bool open = false;
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        float t = top[qt];
        t = fmaxf(t, __shfl_xor(t, 16, 64));
        t = fmaxf(t, __shfl_xor(t, 32, 64));
        const bool none = t == -INFINITY;      // (every product so far is -inf: the row waits for a block with another)
        if (none || (!unset[qt] && t <= LAZY)) t = 0.f;
        unset[qt] = unset[qt] && none;
        open |= unset[qt];
        const float a = __builtin_amdgcn_exp2f(-t);
#pragma unroll
        for (int i = 0; i < 4; ++i) { negm[qt][i] -= t; l[qt][i] *= a; }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[dt][qt] *= a;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kt][qt][i] -= t;
      }
      force = __any(open);
    }
    mfma_bf16x8 pf[2][2];
#pragma unroll
    for (int qt = 0; qt < 2; ++qt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint4 w;
        w.x = cvt_pk(__builtin_amdgcn_exp2f(s[2 * c][qt][0]), __builtin_amdgcn_exp2f(s[2 * c][qt][1]));
        w.y = cvt_pk(__builtin_amdgcn_exp2f(s[2 * c][qt][2]), __builtin_amdgcn_exp2f(s[2 * c][qt][3]));
        w.z = cvt_pk(__builtin_amdgcn_exp2f(s[2 * c + 1][qt][0]), __builtin_amdgcn_exp2f(s[2 * c + 1][qt][1]));
        w.w = cvt_pk(__builtin_amdgcn_exp2f(s[2 * c + 1][qt][2]), __builtin_amdgcn_exp2f(s[2 * c + 1][qt][3]));
        pf[qt][c] = __builtin_bit_cast(mfma_bf16x8, w);
      }
    // the row sums are one more tile of the product, over a V of ones: of the rounded weights, as the numerator's, and already over all lanes
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[0] = mfma16(ones, pf[0][c], l[0]);
      l[1] = mfma16(ones, pf[1][c], l[1]);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = 16 * dt + n;
        const mfma_bf16x8 vf = *(lds_frag*)(lds + (2 + st) * IMG + row * 128 + (((4 * c + g) ^ ((row >> 1) & 7)) << 4));
        acc[dt][0] = mfma16(vf, pf[0][c], acc[dt][0]);
        acc[dt][1] = mfma16(vf, pf[1][c], acc[dt][1]);
      }
    st ^= 1;
  }
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    const float t = l[qt][0];
    const float inv = t == 0.f ? 0.f : 1.f / t;   // a row without keys: zeros
    const int64_t r = q0 + 16 * qt + n;
    if (r < p.Lq) {
      bf16_t* op = p.o + ((int64_t)b * p.Lq + r) * p.H * 128 + (int64_t)h * 128 + 4 * g;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        uint2 w;
        w.x = cvt_pk(acc[dt][qt][0] * inv, acc[dt][qt][1] * inv);
        w.y = cvt_pk(acc[dt][qt][2] * inv, acc[dt][qt][3] * inv);
        *reinterpret_cast<uint2*>(op + 16 * dt) = w;
      }
    }
  }
}

}  // namespace

extern "C" int64_t wan_sparse_attention_scratch_bytes(int B, int64_t Lq, int H, int keep) {
  return 0;
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
  WAN_REQUIRE(nq * H * B < ((int64_t)1 << 31), "wan_sparse_attention: grid too large");
  SparseArgs a = {q, k, vt, o, q_row, q_batch, k_row, k_batch, ldv, Lq, Lk, index, count, k_lens, B, Bk, H, Hk, (int)nq, keep, q_prescaled};
  hipLaunchKernelGGL(attn_sparse_kernel, dim3((unsigned)(nq * H * B)), dim3(256), 0, as_stream(stream), a);
  WAN_LAUNCH_CHECK();
  return 0;
}
