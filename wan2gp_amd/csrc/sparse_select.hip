// The choice of key blocks for block-sparse attention (attention_sparse.hip), gfx950.
//   wan_block_mean     mean of each block of `block` tokens of x [B, L, H, 128], per head, in fp32
//   wan_select_blocks  for each block of queries the `keep` blocks of keys whose mean key has the largest product with the block's mean query
//
// Everything between the bf16 rows and the list is summed in 64 bits.  The lists are whole numbers: two blocks whose scores differ by less
// than a sum's rounding error would swap with the order of that sum, and a swapped block is another output.  In fp32 a 720p step (23,640 lists
// out of 1,182 blocks) holds some dozens of such pairs, in fp64 none: the products of two fp32 numbers are exact there, and two sums in
// different orders agree to 2^-50.
#include "common.h"

namespace {

constexpr int KEY_BLOCK = 64;

// ---- block means -----------------------------------------------------------------------------------------------------------------------
// One workgroup per (block of tokens, 128-column head group, batch): a thread owns 8 columns (16-byte loads) and every fourth row.
__global__ __launch_bounds__(256) void block_mean_kernel(const bf16_t* __restrict__ x, int64_t row_stride, int64_t batch_stride, const int* __restrict__ lens,
                                                        float* __restrict__ out, int64_t L, int H, int block, int nblk) {
  __shared__ double part[3][64][8];
  const int n = blockIdx.x, b = blockIdx.z;
  const int col8 = blockIdx.y * 64 + (threadIdx.x & 63), rg = threadIdx.x >> 6;   // four heads of 16 chunks per workgroup
  int64_t end = L;
  if (lens != nullptr) end = min(max((int64_t)lens[b], (int64_t)0), L);
  const int64_t r0 = (int64_t)n * block;
  const int rows = (int)min((int64_t)block, max(end - r0, (int64_t)0));
  double s[8] = {0., 0., 0., 0., 0., 0., 0., 0.};
  const bool live = col8 < H * 16;
  if (live) {
    const bf16_t* p = x + (int64_t)b * batch_stride + r0 * row_stride + (int64_t)col8 * 8;
#pragma unroll 8
    for (int r = rg; r < rows; r += 4) {
      float f[8];
      unpack8(*reinterpret_cast<const uint4*>(p + (int64_t)r * row_stride), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += (double)f[j];
    }
  }
  if (rg > 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[rg - 1][threadIdx.x & 63][j] = s[j];
  }
  __syncthreads();
  if (rg == 0 && live) {
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double t = s[j] + part[0][threadIdx.x][j] + part[1][threadIdx.x][j] + part[2][threadIdx.x][j];
      m[j] = rows > 0 ? (float)(t / (double)rows) : 0.f;
    }
    float* o = out + (((int64_t)b * H + (col8 >> 4)) * nblk + n) * 128 + (col8 & 15) * 8;
    *reinterpret_cast<float4*>(o) = make_float4(m[0], m[1], m[2], m[3]);
    *reinterpret_cast<float4*>(o + 4) = make_float4(m[4], m[5], m[6], m[7]);
  }
}

// ---- scores ----------------------------------------------------------------------------------------------------------------------------
// An fp64 score as an unsigned number that sorts the same way: NaN above +inf (a NaN in a block has to show in the output, not to vanish with
// the block), -0 equal to +0.
__device__ __forceinline__ uint64_t order_key(double s) {
  if (s != s) return ~0ull;
  if (s == 0.) s = 0.;
  const uint64_t u = (uint64_t)__double_as_longlong(s);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// keys[row][j] for 64 query blocks x 64 key blocks of one (batch, head)
__global__ __launch_bounds__(256) void block_score_kernel(const float* __restrict__ qm, const float* __restrict__ km, uint64_t* __restrict__ keys, int H, int Hk,
                                                         int Bk, int nq, int nk) {
  __shared__ float qs[64][33], ks[64][33];
  const int bh = blockIdx.z, b = bh / H, h = bh - b * H;
  const float* qp = qm + (int64_t)bh * nq * 128;
  const float* kp = km + ((int64_t)(b % Bk) * Hk + h / (H / Hk)) * nk * 128;
  const int q0 = blockIdx.y * 64, k0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  double acc[4][4] = {};
  for (int d0 = 0; d0 < 128; d0 += 32) {
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i >> 5, c = i & 31;
      qs[r][c] = q0 + r < nq ? qp[(int64_t)(q0 + r) * 128 + d0 + c] : 0.f;
      ks[r][c] = k0 + r < nk ? kp[(int64_t)(k0 + r) * 128 + d0 + c] : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < 32; ++c) {
      double a[4], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = (double)qs[ty + 16 * i][c]; w[i] = (double)ks[tx + 16 * i][c]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_fma(a[i], w[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = q0 + ty + 16 * i, k = k0 + tx + 16 * j;
      if (q < nq && k < nk) keys[((int64_t)bh * nq + q) * nk + k] = order_key(acc[i][j]);
    }
}

// ---- the `keep` largest of a row ---------------------------------------------------------------------------------------------------------
// One workgroup per row, the row's keys in LDS: the keep-th largest key bit by bit from the top, then one pass that emits what is above it and the
// first of what equals it, in ascending order.
__global__ __launch_bounds__(256) void block_select_kernel(const uint64_t* __restrict__ keys, const int* __restrict__ k_lens, int* __restrict__ index,
                                                          int* __restrict__ count, int H, int Bk, int nq, int nk, int keep) {
  extern __shared__ uint64_t row[];
  __shared__ int wsum[2][4];
  const int64_t r = blockIdx.x;
  const int b = (int)(r / ((int64_t)H * nq));
  int n = nk;
  if (k_lens != nullptr) n = min(nk, max(0, (int)(((int64_t)k_lens[b % Bk] + KEY_BLOCK - 1) / KEY_BLOCK)));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* idx = index + r * keep;
  const int want = min(keep, n);
  if (tid == 0) count[r] = want;
  for (int i = want + tid; i < keep; i += 256) idx[i] = -1;
  if (want == n) {
    for (int i = tid; i < n; i += 256) idx[i] = i;
    return;
  }
  for (int i = tid; i < n; i += 256) row[i] = keys[r * nk + i];
  __syncthreads();
  uint64_t t = 0;      // the largest value that at least `want` keys reach
  int ge = n;          // how many reach it
  for (int bit = 63; bit >= 0 && ge != want; --bit) {
    const uint64_t c = t | (1ull << bit);
    int m = 0;
    for (int i = tid; i < n; i += 256) m += row[i] >= c;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
    if (lane == 0) wsum[bit & 1][wave] = m;
    __syncthreads();
    m = wsum[bit & 1][0] + wsum[bit & 1][1] + wsum[bit & 1][2] + wsum[bit & 1][3];
    if (m >= want) { t = c; ge = m; }
  }
  // more than `want` keys reach t only if the smallest of them equal t: the first of those are taken
  int above = 0;
  for (int i = tid; i < n; i += 256) above += row[i] > t;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) above += __shfl_xor(above, o, 64);
  __syncthreads();
  if (lane == 0) wsum[0][wave] = above;
  __syncthreads();
  above = wsum[0][0] + wsum[0][1] + wsum[0][2] + wsum[0][3];
  if (wave != 0) return;
  int room = ge == want ? n : want - above, out = 0;   // room: how many of the keys that equal t are still taken
  for (int i0 = 0; i0 < n; i0 += 64) {
    const uint64_t k = i0 + lane < n ? row[i0 + lane] : 0ull;
    const bool in = i0 + lane < n;
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t eq = __ballot(in && k == t);
    const bool take = in && (k > t || (k == t && __popcll(eq & below) < room));
    const uint64_t tk = __ballot(take);
    if (take) idx[out + __popcll(tk & below)] = i0 + lane;
    out += __popcll(tk);
    room -= min(room, (int)__popcll(eq));
  }
}

}  // namespace

extern "C" int wan_block_mean(const wan_bf16* x, int64_t row_stride, int64_t batch_stride, const int* lens, float* out, int B, int64_t L, int H, int block, void* stream) {
  WAN_REQUIRE(x && out, "wan_block_mean: null pointer");
  WAN_REQUIRE(B >= 1 && L >= 1 && H >= 1 && block >= 1, "wan_block_mean: empty problem (B=%d L=%lld H=%d block=%d)", B, (long long)L, H, block);
  WAN_REQUIRE(row_stride % 8 == 0 && batch_stride % 8 == 0 && row_stride >= (int64_t)H * 128, "wan_block_mean: strides must be multiples of 8 elements, a row's at least H * 128");
  WAN_REQUIRE((((uintptr_t)x | (uintptr_t)out) & 15) == 0, "wan_block_mean: pointers must be 16-byte aligned");
  const int64_t nblk = (L + block - 1) / block;
  WAN_REQUIRE(nblk < ((int64_t)1 << 31) && B < 65536 && H <= 4 * 65535, "wan_block_mean: grid too large");
  hipLaunchKernelGGL(block_mean_kernel, dim3((unsigned)nblk, (unsigned)((H * 16 + 63) / 64), (unsigned)B), dim3(256), 0, as_stream(stream), x, row_stride, batch_stride, lens, out,
                     L, H, block, (int)nblk);
  WAN_LAUNCH_CHECK();
  return 0;
}

extern "C" int64_t wan_select_blocks_scratch_bytes(int B, int H, int64_t nq, int64_t nk) {
  if (B < 1 || H < 1 || nq < 1 || nk < 1) return 0;
  return (int64_t)B * H * nq * nk * 8;
}

extern "C" int wan_select_blocks(const float* q_mean, const float* k_mean, const int* k_lens, int* index, int* count, int B, int Bk, int H, int Hk, int64_t nq, int64_t nk,
                                 int keep, void* scratch, int64_t scratch_bytes, void* stream) {
  WAN_REQUIRE(q_mean && k_mean && index && count, "wan_select_blocks: null pointer");
  WAN_REQUIRE(B >= 1 && Bk >= 1 && B % Bk == 0, "wan_select_blocks: Bk must divide B (B=%d Bk=%d)", B, Bk);
  WAN_REQUIRE(H >= 1 && Hk >= 1 && H % Hk == 0, "wan_select_blocks: the heads of k must divide the heads of q (H=%d Hk=%d)", H, Hk);
  WAN_REQUIRE(nq >= 1 && nk >= 1 && keep >= 1, "wan_select_blocks: empty problem (nq=%lld nk=%lld keep=%d)", (long long)nq, (long long)nk, keep);
  WAN_REQUIRE(nk <= 20000, "wan_select_blocks: %lld blocks of keys (at most 20,000: a row of scores has to fit the LDS)", (long long)nk);
  WAN_REQUIRE((int64_t)B * H < 65536 && (int64_t)B * H * nq < ((int64_t)1 << 31) && (nq + 63) / 64 < 65536, "wan_select_blocks: grid too large");
  WAN_REQUIRE(scratch && scratch_bytes >= wan_select_blocks_scratch_bytes(B, H, nq, nk) && ((uintptr_t)scratch & 15) == 0,
              "wan_select_blocks: needs 16-byte aligned scratch of %lld bytes", (long long)wan_select_blocks_scratch_bytes(B, H, nq, nk));
  WAN_REQUIRE((((uintptr_t)q_mean | (uintptr_t)k_mean) & 15) == 0, "wan_select_blocks: the means must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  uint64_t* keys = reinterpret_cast<uint64_t*>(scratch);
  hipLaunchKernelGGL(block_score_kernel, dim3((unsigned)((nk + 63) / 64), (unsigned)((nq + 63) / 64), (unsigned)(B * H)), dim3(256), 0, st, q_mean, k_mean, keys, H, Hk, Bk, (int)nq, (int)nk);
  WAN_LAUNCH_CHECK();
  hipLaunchKernelGGL(block_select_kernel, dim3((unsigned)(B * H * nq)), dim3(256), (unsigned)(nk * 8), st, keys, k_lens, index, count, H, Bk, (int)nq, (int)nk, keep);
  WAN_LAUNCH_CHECK();
  return 0;
}
