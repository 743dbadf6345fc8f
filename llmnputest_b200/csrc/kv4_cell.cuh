// The 4-bit paged KV cache: its storage unit and the helpers its kernels share.
//
// A page holds `page` tokens (a multiple of 16) of every kv head.  Per kv head it is
// [page / 16][D / 64] cells of 1152 bytes; a cell is 16 tokens x 64 dims of K and of V:
//
//   0..511     K codes  [t % 8][c][t / 8][8 bytes]: dims 16 c .. 16 c + 15 of token t,
//              nibble k of a 32-bit word is the word's k-th dim
//   512..1023  V codes  [g][c][p][quad][e][2 bytes]: dims 8 g + 4 quad .. + 3 of token
//              8 p + 2 c + e
//   1024..1087 K (d, m) [t % 8][t / 8] bf16 pairs;  1088..1151 V (d, m), the same
//
// A value is code * d + m.  The order is the one in which mma.sync m16n8k16 wants its A
// operand: lane (g = lane / 4, c = lane % 4) takes 16 consecutive bytes of K codes (its
// 16 dims of tokens g and g + 8) and 16 of V codes (its 4 tokens, 8 dims), a warp 512
// consecutive bytes of each, and no byte holds two tokens, so that a new token is written
// without reading what is beside it.
#pragma once

#include <cuda_fp16.h>

#include "b2_common.cuh"

namespace b2 {

constexpr int kKv4CellBytes = 1152;
constexpr int kKv4Tile = 16;    // tokens of a cell
constexpr int kKv4Group = 64;   // dims of a cell: the values that share a (d, m)
constexpr int kKv4VCodes = 512, kKv4KMeta = 1024, kKv4VMeta = 1088;
constexpr float kKv4MinStep = 9.094947017729282e-13f;  // 2^-40, the least d
constexpr int kKv4MaxHalfDim = 128;                    // head_dim <= 256
constexpr int kDevBadPosition = 5;  // a position or page outside its table, pool or planned length

// theta^(-2i/D) / (2 pi) for pair i: an angle is pos * turn[i] whole turns, so that its
// fraction is exact to 2^-53 of the whole at any position (fp32 angles lose 2^-24 of it)
struct Kv4Rope {
  double turn[kKv4MaxHalfDim];
  int on;
};

// A kernel parameter's table entry by a lane's own index: through its generic address, as the
// constant port would take the 32 lanes' indices one by one.
__device__ __forceinline__ double kv4_turn(const Kv4Rope& rope, int i) {
  double t;
  asm("ld.f64 %0, [%1];" : "=d"(t) : "l"(rope.turn + i));
  return t;
}

// cos and sin of u turns in fp64: to the nearest quarter turn, then the Taylor series of an
// angle of pi/4 at most (the first term left out is below 3e-18).  Without branches, so that
// several angles are evaluated side by side.
__device__ __forceinline__ void kv4_cos_sin(double u, double& cs, double& sn) {
  const double quarter = rint(4.0 * u);
  const double x = fma(quarter, -0.25, u) * 6.283185307179586476925287, y = x * x;
  double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;  // 1 / 17!, 1 / 16!
  s = fma(s, y, -1.0 / 1307674368000.0);
  c = fma(c, y, -1.0 / 87178291200.0);
  s = fma(s, y, 1.0 / 6227020800.0);
  c = fma(c, y, 1.0 / 479001600.0);
  s = fma(s, y, -1.0 / 39916800.0);
  c = fma(c, y, -1.0 / 3628800.0);
  s = fma(s, y, 1.0 / 362880.0);
  c = fma(c, y, 1.0 / 40320.0);
  s = fma(s, y, -1.0 / 5040.0);
  c = fma(c, y, -1.0 / 720.0);
  s = fma(s, y, 1.0 / 120.0);
  c = fma(c, y, 1.0 / 24.0);
  s = fma(s, y, -1.0 / 6.0);
  c = fma(c, y, -0.5);
  s = fma(s * y, x, x);
  c = fma(c, y, 1.0);
  const int k = static_cast<int>(static_cast<long long>(quarter)) & 3;
  cs = k & 1 ? s : c;
  sn = k & 1 ? c : s;
  if (k == 1 || k == 2) cs = -cs;
  if (k >= 2) sn = -sn;
}

// byte of K code word w (8 dims) of token t: dims 8 w .. 8 w + 7 of the cell's 64
__host__ __device__ constexpr int kv4_k_word(int t, int w) {
  return (t % 8) * 64 + (w / 2) * 16 + (t / 8) * 8 + (w % 2) * 4;
}
// byte of the V code half-word of token t's dims 4 x .. 4 x + 3
__host__ __device__ constexpr int kv4_v_half(int t, int x) {
  return kKv4VCodes + (x / 2) * 64 + (t % 8 / 2) * 16 + (t / 8) * 8 + (x % 2) * 4 + (t % 2) * 2;
}
// byte of token t's (d, m) pair in its 64-byte block
__host__ __device__ constexpr int kv4_meta(int t) { return (t % 8) * 8 + (t / 8) * 4; }

// Sequence b's rows [lo, hi) of a ragged batch (cu null: row b alone), kept inside 0..rows.
__device__ __forceinline__ void kv4_rows(const int* cu, int rows, int b, int& lo, int& hi) {
  if (!cu) {
    lo = b;
    hi = b + 1;
    return;
  }
  lo = min(max(cu[b], 0), rows);
  hi = min(max(cu[b + 1], lo), rows);
}

// The job-th (sequence, page) that a ragged batch touches, for a warp: returns the
// sequence, or -1 behind the last; pg = the page's index in its sequence.
__device__ __forceinline__ int kv4_find_job(const int* cu, const int* pos, int rows, int batch, int page, int job,
                                            int& pg) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int b = b0 + lane;
    int n = 0, first = 0;
    if (b < batch) {
      int lo, hi;
      kv4_rows(cu, rows, b, lo, hi);
      const long long p0 = pos[b];
      if (hi > lo && p0 >= 0) {
        first = static_cast<int>(p0 / page);
        n = static_cast<int>((p0 + (hi - lo) - 1) / page) - first + 1;
      } else if (hi > lo && p0 < -1) {
        n = 1;  // reported by its job
      }
    }
    int end = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, job < end);
    if (hit) {
      const int l = __ffs(hit) - 1;
      pg = __shfl_sync(0xffffffffu, first, l) + job - (__shfl_sync(0xffffffffu, end, l) - __shfl_sync(0xffffffffu, n, l));
      return b0 + l;
    }
    job -= __shfl_sync(0xffffffffu, end, 31);
  }
  return -1;
}

// The page of the pool that holds page pg of sequence b, or -1.
__device__ __forceinline__ int kv4_page_id(const int* table, int max_pages, int n_pages, int b, int pg) {
  if (pg < 0 || pg >= max_pages) return -1;
  const int id = table[static_cast<size_t>(b) * max_pages + pg];
  return id >= 0 && id < n_pages ? id : -1;
}

// Sum of v over the threads below this one; total = over all (blockDim.x threads, 32 warps at most).
__device__ __forceinline__ int kv4_block_before(int v, int* warps, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += x;
  }
  __syncthreads();  // the array's last use is over
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  int x = lane < nw ? warps[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  const int before = __shfl_sync(0xffffffffu, x, max(warp - 1, 0));
  return s - v + (warp ? before : 0);
}

}  // namespace b2
