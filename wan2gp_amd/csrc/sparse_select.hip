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
// One workgroup per (block of tokens, two heads, batch): a thread owns 8 columns (16-byte loads) and every eighth row, eight loads in flight.  Bound by
// the rows' bytes: 75,600 rows of 40 heads in 145 us, 5.3 TB/s.
__global__ __launch_bounds__(256) void block_mean_kernel(const bf16_t* __restrict__ x, int64_t row_stride, int64_t batch_stride, const int* __restrict__ lens,
                                                        float* __restrict__ out, int64_t L, int H, int block, int nblk) {
  __shared__ double part[8][32][9];   // (a pitch of 9: the sums below read along the second index)
  const int n = blockIdx.x, b = blockIdx.z;
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const int col8 = blockIdx.y * 32 + c;
  int64_t end = L;
  if (lens != nullptr) end = min(max((int64_t)lens[b], (int64_t)0), L);
  const int64_t r0 = (int64_t)n * block;
  const int rows = (int)min((int64_t)block, max(end - r0, (int64_t)0));
  double s[8] = {0., 0., 0., 0., 0., 0., 0., 0.};
  if (col8 < H * 16) {
    const bf16_t* p = x + (int64_t)b * batch_stride + r0 * row_stride + (int64_t)col8 * 8;
    int r = rg;
    for (; r + 56 < rows; r += 64) {
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const uint4*>(p + (int64_t)(r + 8 * u) * row_stride);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float f[8];
        unpack8(v[u], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += (double)f[j];
      }
    }
    for (; r < rows; r += 8) {
      float f[8];
      unpack8(*reinterpret_cast<const uint4*>(p + (int64_t)r * row_stride), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += (double)f[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) part[rg][c][j] = s[j];
  __syncthreads();
  const int col = threadIdx.x, h = blockIdx.y * 2 + (col >> 7);   // a column a thread
  if (h < H) {
    double t = 0.;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += part[k][col >> 3][col & 7];
    out[(((int64_t)b * H + h) * nblk + n) * 128 + (col & 127)] = rows > 0 ? (float)(t / (double)rows) : 0.f;
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

// Scores on v_mfma_f64_16x16x4_f64: lane (n, g) supplies A[n][g] (query block n) and B[g][n] (key block n) of a step; register i holds D[4 i + g][n].  A
// sum's order is free, so step 4 s + e takes column 16 s + 4 g + e: a load of four floats a lane is 64 consecutive bytes of each row (32 consecutive floats a
// lane read every line of the L2 four times).  Two tiles of 16 key blocks at a time: two independent chains of products, and twice the loads in flight.
typedef double f64x4 __attribute__((ext_vector_type(4)));
struct QueryMeans {
  double a[32];
};
__device__ __forceinline__ QueryMeans load_queries(const float* qp) {   // (of the lane's row, from its column 4 g on)
  QueryMeans q;
#pragma unroll
  for (int s = 0; s < 32; s += 4) {
    const float4 v = *reinterpret_cast<const float4*>(qp + 4 * s);
    q.a[s] = v.x; q.a[s + 1] = v.y; q.a[s + 2] = v.z; q.a[s + 3] = v.w;
  }
  return q;
}
__device__ __forceinline__ void score_pair(const QueryMeans& q, const float* kp, int k0, int n, int nk, f64x4 (&acc)[2]) {
  float4 v[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const float* r = kp + (int64_t)min(k0 + 16 * u + n, nk - 1) * 128;
#pragma unroll
    for (int s = 0; s < 8; ++s) v[u][s] = *reinterpret_cast<const float4*>(r + 16 * s);
  }
  acc[0] = acc[1] = f64x4{0., 0., 0., 0.};
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const float f[2][4] = {{v[0][s].x, v[0][s].y, v[0][s].z, v[0][s].w}, {v[1][s].x, v[1][s].y, v[1][s].z, v[1][s].w}};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[0] = __builtin_amdgcn_mfma_f64_16x16x4f64(q.a[4 * s + e], (double)f[0][e], acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_f64_16x16x4f64(q.a[4 * s + e], (double)f[1][e], acc[1], 0, 0, 0);
    }
  }
}

// More than 256 blocks of keys: the scores go to memory, keys[row][j].  One wave per 16 query blocks x `tiles` tiles of key blocks (even: eight, down to two where that leaves
// fewer than 2,048 waves: 24 heads x 13 x 512 take 5.0 us with two, 14.1 with eight); the four waves of a workgroup read the same keys.  Bound by the fp64 matrix rate (a step
// 64 cycles) and the conversions in front of it: 40 heads x 591 x 1,182 in 173 us, 41 TFLOP/s and 223 MB of scores written.
__global__ __launch_bounds__(256) void block_score_kernel(const float* __restrict__ qm, const float* __restrict__ km, uint64_t* __restrict__ keys, int H, int Hk,
                                                         int Bk, int nq, int nk, int tiles) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int bh = blockIdx.z, b = bh / H, h = bh - b * H;
  const int q0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * 16, k0 = blockIdx.x * (16 * tiles);
  if (q0 >= nq) return;
  const QueryMeans qs = load_queries(qm + ((int64_t)bh * nq + min(q0 + n, nq - 1)) * 128 + 4 * g);
  const float* kp = km + ((int64_t)(b % Bk) * Hk + h / (H / Hk)) * nk * 128 + 4 * g;
  for (int t = 0; t < tiles && k0 + 16 * t < nk; t += 2) {
    f64x4 acc[2];
    score_pair(qs, kp, k0 + 16 * t, n, nk, acc);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = q0 + 4 * i + g, k = k0 + 16 * (t + u) + n;
        if (q < nq && k < nk) keys[((int64_t)bh * nq + q) * nk + k] = order_key(acc[u][i]);
      }
  }
}

// ---- the `keep` largest of a row ---------------------------------------------------------------------------------------------------------
// Both kernels find the keep-th largest key bit by bit from the top (t: the largest value that at least `want` keys reach; they stop as soon as exactly that
// many do), then emit what is above it and the first of what equals it, in ascending order.  A key 0 is none.

// A wave, N keys a lane in registers, first over the keys' upper halves -- 20 of the mantissa's bits decide nearly every row.
template <int N, class F>
__device__ __forceinline__ void select_row(F&& key, int n, int want, int* idx) {
  const int lane = threadIdx.x & 63;
  uint32_t hi[N], lo[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = j * 64 + lane;
    const uint64_t k = i < n ? key(i) : 0ull;
    hi[j] = (uint32_t)(k >> 32);
    lo[j] = (uint32_t)k;
  }
  uint32_t th = 0, tl = 0;
  int ge = n;
  for (int bit = 31; bit >= 0 && ge != want; --bit) {
    const uint32_t c = th | (1u << bit);
    int m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m += __popcll(__ballot(hi[j] >= c));
    if (m >= want) { th = c; ge = m; }
  }
  if (ge != want) {
    for (int bit = 31; bit >= 0 && ge != want; --bit) {
      const uint32_t c = tl | (1u << bit);
      int m = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) m += __popcll(__ballot(hi[j] > th || (hi[j] == th && lo[j] >= c)));
      if (m >= want) { tl = c; ge = m; }
    }
  }
  int room = n;          // how many of the keys that equal t are taken
  if (ge != want) {
    int above = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) above += __popcll(__ballot(hi[j] > th || (hi[j] == th && lo[j] > tl)));
    room = want - above;
  }
  int out = 0;
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool eq = hi[j] == th && lo[j] == tl;
    const uint64_t eqs = __ballot(eq);
    const bool take = hi[j] > th || (hi[j] == th && lo[j] > tl) || (eq && __popcll(eqs & below) < room);
    const uint64_t tk = __ballot(take);
    if (take) idx[out + __popcll(tk & below)] = j * 64 + lane;
    out += __popcll(tk);
    room -= min(room, (int)__popcll(eqs));
  }
}

// count and what of the list does not depend on scores; true: the list is complete
__device__ __forceinline__ bool open_row(int* idx, int* count, int n, int want, int keep) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) *count = want;
  for (int i = want + lane; i < keep; i += 64) idx[i] = -1;
  if (want < n) return false;
  for (int i = lane; i < n; i += 64) idx[i] = i;
  return true;
}
__device__ __forceinline__ int candidates(const int* k_lens, int b, int nk) {
  return k_lens == nullptr ? nk : min(nk, max(0, (int)(((int64_t)k_lens[b] + KEY_BLOCK - 1) / KEY_BLOCK)));
}

// Up to 256 blocks of keys: scores and choice in one launch, the scores never leave the LDS.  Eight waves take the key tiles of 16 query blocks in turn, then two of their rows
// each.  40 heads x 128 x 256: 22 us, in two launches 34.  (With more keys the two phases one behind the other leave too much idle: 13 x 1,182 takes 44 us so and 28 in two launches,
// 591 x 1,182 271 and 235.)
constexpr int CHOOSE_KEYS = 256;
__global__ __launch_bounds__(512) void block_choose_kernel(const float* __restrict__ qm, const float* __restrict__ km, const int* __restrict__ k_lens, int* __restrict__ index,
                                                          int* __restrict__ count, int H, int Hk, int Bk, int nq, int nk, int keep) {
  __shared__ uint64_t row[16 * CHOOSE_KEYS];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = blockIdx.y, b = bh / H, h = bh - b * H, q0 = blockIdx.x * 16;
  const int have = candidates(k_lens, b % Bk, nk), want = min(keep, have);
  if (want < have) {
    const QueryMeans qs = load_queries(qm + ((int64_t)bh * nq + min(q0 + n, nq - 1)) * 128 + 4 * g);
    const float* kp = km + ((int64_t)(b % Bk) * Hk + h / (H / Hk)) * nk * 128 + 4 * g;
    const int k0 = wave * 32;
    if (k0 < have) {
      f64x4 acc[2];
      score_pair(qs, kp, k0, n, nk, acc);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          row[(4 * i + g) * CHOOSE_KEYS + k0 + 16 * u + n] = order_key(acc[u][i]);   // (k0 + 31 < 256)
    }
  }
  __syncthreads();
  for (int r = wave; r < 16 && q0 + r < nq; r += 8) {
    const int64_t at = (int64_t)bh * nq + q0 + r;
    if (open_row(index + at * keep, count + at, have, want, keep)) continue;
    const uint64_t* keys = row + r * CHOOSE_KEYS;
    select_row<CHOOSE_KEYS / 64>([&](int i) { return keys[i]; }, have, want, index + at * keep);
  }
}

// Up to 2,048: one wave per row, its keys from memory.  Bound by the ballots and the scores' bytes: 23,640 rows of 1,182 in 62 us.  The whole choice took 237 us so and 390 us with
// the search by a workgroup below; 609 against 937 us at 1,024 x 2,048.  N, the keys a lane holds, goes by the blocks of keys in steps of four: a step is 8 to 15 us of
// 40 x 591 rows (the whole choice out of 1,400 blocks 258 us with 24 keys a lane, 288 with 32; out of 800 152 with 16, 158 with 19; out of 1,216 216 with 20, 213 with 19).
template <int N>
__global__ __launch_bounds__(256) void block_select_wave_kernel(const uint64_t* __restrict__ keys, const int* __restrict__ k_lens, int* __restrict__ index,
                                                               int* __restrict__ count, int H, int Bk, int nq, int nk, int keep, int64_t rows) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int n = candidates(k_lens, (int)(r / ((int64_t)H * nq)) % Bk, nk), want = min(keep, n);
  if (open_row(index + r * keep, count + r, n, want, keep)) return;
  select_row<N>([&](int i) { return keys[r * nk + i]; }, n, want, index + r * keep);
}

// More than 2,048 blocks: one workgroup per row, the row's keys in LDS.  16 waves where the LDS has room for two rows or fewer (128 x 20,000 of 40 heads: 2.49 ms,
// with 4 waves 4.35), else 4, more workgroups side by side (512 x 4,096: 1.31 ms, with 16 waves 1.67).
template <int WG_WAVES>
__global__ __launch_bounds__(64 * WG_WAVES) void block_select_kernel(const uint64_t* __restrict__ keys, const int* __restrict__ k_lens, int* __restrict__ index,
                                                          int* __restrict__ count, int H, int Bk, int nq, int nk, int keep) {
  extern __shared__ uint64_t row[];
  __shared__ int wsum[2][WG_WAVES];
  const int64_t r = blockIdx.x;
  const int b = (int)(r / ((int64_t)H * nq));
  int n = nk;
  if (k_lens != nullptr) n = min(nk, max(0, (int)(((int64_t)k_lens[b % Bk] + KEY_BLOCK - 1) / KEY_BLOCK)));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* idx = index + r * keep;
  const int want = min(keep, n);
  if (tid == 0) count[r] = want;
  for (int i = want + tid; i < keep; i += 64 * WG_WAVES) idx[i] = -1;
  if (want == n) {
    for (int i = tid; i < n; i += 64 * WG_WAVES) idx[i] = i;
    return;
  }
  for (int i = tid; i < n; i += 64 * WG_WAVES) row[i] = keys[r * nk + i];
  __syncthreads();
  uint64_t t = 0;
  int ge = n;
  for (int bit = 63; bit >= 0 && ge != want; --bit) {
    const uint64_t c = t | (1ull << bit);
    int m = 0;
    for (int i = tid; i < n; i += 64 * WG_WAVES) m += row[i] >= c;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
    if (lane == 0) wsum[bit & 1][wave] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < WG_WAVES; ++w) m += wsum[bit & 1][w];
    if (m >= want) { t = c; ge = m; }
  }
  int above = 0;
  for (int i = tid; i < n; i += 64 * WG_WAVES) above += row[i] > t;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) above += __shfl_xor(above, o, 64);
  __syncthreads();
  if (lane == 0) wsum[0][wave] = above;
  __syncthreads();
  above = 0;
#pragma unroll
  for (int w = 0; w < WG_WAVES; ++w) above += wsum[0][w];
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
  WAN_REQUIRE(nblk < ((int64_t)1 << 31) && B < 65536 && H <= 2 * 65535, "wan_block_mean: grid too large");
  hipLaunchKernelGGL(block_mean_kernel, dim3((unsigned)nblk, (unsigned)((H + 1) / 2), (unsigned)B), dim3(256), 0, as_stream(stream), x, row_stride, batch_stride, lens, out,
                     L, H, block, (int)nblk);
  WAN_LAUNCH_CHECK();
  return 0;
}

extern "C" int64_t wan_select_blocks_scratch_bytes(int B, int H, int64_t nq, int64_t nk) {
  if (B < 1 || H < 1 || nq < 1 || nk <= CHOOSE_KEYS) return 0;   // (the scores stay in the LDS)
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
  const int64_t need = wan_select_blocks_scratch_bytes(B, H, nq, nk);
  WAN_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0), "wan_select_blocks: needs 16-byte aligned scratch of %lld bytes", (long long)need);
  WAN_REQUIRE((((uintptr_t)q_mean | (uintptr_t)k_mean) & 15) == 0, "wan_select_blocks: the means must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  if (nk <= CHOOSE_KEYS) {
    hipLaunchKernelGGL(block_choose_kernel, dim3((unsigned)((nq + 15) / 16), (unsigned)(B * H)), dim3(512), 0, st, q_mean, k_mean, k_lens, index, count, H, Hk, Bk, (int)nq, (int)nk, keep);
    WAN_LAUNCH_CHECK();
    return 0;
  }
  uint64_t* keys = reinterpret_cast<uint64_t*>(scratch);
  int tiles = 8;
  while (tiles > 2 && (nk + 16 * tiles - 1) / (16 * tiles) * ((nq + 15) / 16) * B * H < 2048) tiles /= 2;
  hipLaunchKernelGGL(block_score_kernel, dim3((unsigned)((nk + 16 * tiles - 1) / (16 * tiles)), (unsigned)((nq + 63) / 64), (unsigned)(B * H)), dim3(256), 0, st, q_mean, k_mean, keys, H,
                     Hk, Bk, (int)nq, (int)nk, tiles);
  WAN_LAUNCH_CHECK();
  const int64_t rows = (int64_t)B * H * nq;
  const dim3 grid((unsigned)((rows + 3) / 4)), wg(256);
#define SELECT(N) hipLaunchKernelGGL(block_select_wave_kernel<N>, grid, wg, 0, st, keys, k_lens, index, count, H, Bk, (int)nq, (int)nk, keep, rows)
  switch (nk <= 2048 ? (nk + 255) / 256 : 0) {
    case 2: SELECT(8); break;
    case 3: SELECT(12); break;
    case 4: SELECT(16); break;
    case 5: SELECT(20); break;
    case 6: SELECT(24); break;
    case 7: SELECT(28); break;
    case 8: SELECT(32); break;
#undef SELECT
    default:
      if (nk <= 6800) hipLaunchKernelGGL(block_select_kernel<4>, dim3((unsigned)rows), wg, (unsigned)(nk * 8), st, keys, k_lens, index, count, H, Bk, (int)nq, (int)nk, keep);
      else hipLaunchKernelGGL(block_select_kernel<16>, dim3((unsigned)rows), dim3(1024), (unsigned)(nk * 8), st, keys, k_lens, index, count, H, Bk, (int)nq, (int)nk, keep);
  }
  WAN_LAUNCH_CHECK();
  return 0;
}
