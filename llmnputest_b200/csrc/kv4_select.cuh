// Choosing the pages that a query attends to in a long cache, by a bound on their scores.
//
//   bound(page) = max over the kv head's q heads of sum_d max(q_d lo_d, q_d hi_d),
//
// lo and hi the page's key summary (per dim, over its tokens): no token of the page scores
// higher with any of the heads.  Per (sequence, kv head) the n_sel pages with the largest
// bounds are listed, in ascending order of the page; the page of the query's own position
// is always among them, and of two equal bounds the lower page goes first.
//
// Which page is the n_sel-th turns on the last bit of two bounds, so q is turned and the
// sums are taken in fp64; the summaries are bf16, so that every product is exact.
//
// A cluster per (sequence, kv head): its CTAs take every further group of pages, a warp
// 256 / D pages at a time (D / 8 lanes a page, 8 dims each), and push the bounds, as integers
// of the same order, into the first CTA's shared memory, which finds the n_sel-th by 8-bit
// digits from the highest bit in which they differ, until a digit settles it (two or three
// rounds of eight), and writes the pages in order.  One launch and no workspace; with the
// bounds in a kernel of their own, a warp per page, and eight rounds, 512 pages of 8 kv heads
// measured 21 us and 16 sequences of up to 1024 pages 41 us.
#pragma once

#include "kv4_cell.cuh"
#include "kv4_decode.cuh"

namespace b2 {

struct Kv4SelectParams {
  const float* q;  // [batch][ld_q]
  long long ld_q;
  const __nv_bfloat16* summary;  // [n_pages][hkv][2][D]
  const int* table;
  const int* pos;
  int* sel;  // [batch][hkv][n_sel]
  int batch, hq, hkv, page, max_pages, n_pages, n_sel;
  int key_pages;  // pages planned for (max_len)
  int ctas;       // of a cluster
};

// a double as an unsigned integer of the same order, 1 or more; NaN and -inf are 1
__device__ __forceinline__ unsigned long long kv4_key(double x) {
  if (!(x > -INFINITY)) return 1;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ void st_dsmem_u64(uint32_t local_addr, uint32_t rank, unsigned long long v) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(local_addr), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ra), "l"(v) : "memory");
}

constexpr int kKv4SelectThreads = 256;

template <int D>
__global__ void __launch_bounds__(kKv4SelectThreads) kv4_select_kernel(const Kv4SelectParams p,
                                                                      const __grid_constant__ Kv4Rope rope) {
  constexpr int LR = D / 8, RW = 32 / LR, W = kKv4SelectThreads / 32;
  extern __shared__ unsigned long long keys[];  // the first CTA's are used
  __shared__ __align__(16) double q[kKv4MaxGroup][D];
  __shared__ double turn_s[2][D / 2];
  __shared__ int hist[256], scan[W], sh_digit, sh_above, sh_count;
  __shared__ unsigned long long sh_diff;
  const int rank = blockIdx.x % p.ctas, kvh = blockIdx.x / p.ctas, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = p.hq / p.hkv;
  if (p.ctas > 1) cluster_arrive_relaxed();  // waited for before anything is pushed
  pdl_wait();
  pdl_launch_dependents();
  int* sel = p.sel + (static_cast<size_t>(b) * p.hkv + kvh) * p.n_sel;
  const int pos = p.pos[b];
  if (pos < 0 || pos >= static_cast<long long>(p.max_pages) * p.page || pos / p.page >= p.key_pages) {
    if (rank == 0) {
      if (pos != -1 && tid == 0) record_error(kDevBadPosition);
      for (int i = tid; i < p.n_sel; i += kKv4SelectThreads) sel[i] = -1;
    }
    if (p.ctas > 1) cluster_wait_acquire();
    return;  // the whole cluster
  }
  const int n = pos / p.page + 1;  // pages; the last is chosen without a bound
  const int need = p.n_sel - 1;    // of the n - 1 others
  if (need < n - 1 && need > 0) {
    // ---- q turned to pos
    if (rope.on) {
      for (int i = tid; i < D / 2; i += kKv4SelectThreads) {
        double u = static_cast<double>(pos) * kv4_turn(rope, i);
        u -= rint(u);
        kv4_cos_sin(u, turn_s[0][i], turn_s[1][i]);
      }
      __syncthreads();
    }
    for (int e = tid; e < grp * (D / 2); e += kKv4SelectThreads) {
      const int j = e / (D / 2), i = e % (D / 2);
      const float* src = p.q + static_cast<size_t>(b) * p.ld_q + static_cast<size_t>(kvh * grp + j) * D;
      const double a = src[i], z = src[i + D / 2];
      const double c = rope.on ? turn_s[0][i] : 1.0, s = rope.on ? turn_s[1][i] : 0.0;
      q[j][i] = a * c - z * s;
      q[j][i + D / 2] = z * c + a * s;
    }
    __syncthreads();
    if (p.ctas > 1) cluster_wait_acquire();
    // ---- the bounds
    const uint32_t keys_s = smem_u32(keys);
    const int l = lane % LR, sub = lane / LR;
    for (int pg0 = (rank * W + warp) * RW; pg0 < n - 1; pg0 += p.ctas * W * RW) {
      const int pg = pg0 + sub;
      const bool in = pg < n - 1;
      const int id = in ? kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg) : -1;
      double lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.0;
      if (id >= 0) {
        const __nv_bfloat16* sm = p.summary + (static_cast<size_t>(id) * p.hkv + kvh) * 2 * D + 8 * l;
        const uint4 a = *reinterpret_cast<const uint4*>(sm), z = *reinterpret_cast<const uint4*>(sm + D);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[2 * i] = bf16lo_to_f32(aw[i]);
          lo[2 * i + 1] = bf16hi_to_f32(aw[i]);
          hi[2 * i] = bf16lo_to_f32(zw[i]);
          hi[2 * i + 1] = bf16hi_to_f32(zw[i]);
        }
      }
      double best = -INFINITY;
      for (int j = 0; j < grp; ++j) {
        const double2* x2 = reinterpret_cast<const double2*>(&q[j][8 * l]);
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double2 x = x2[i];
          s = fma(x.x, x.x > 0.0 ? hi[2 * i] : lo[2 * i], s);
          s = fma(x.y, x.y > 0.0 ? hi[2 * i + 1] : lo[2 * i + 1], s);
        }
#pragma unroll
        for (int o = LR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        best = fmax(best, s);
      }
      if (in && l == 0) {
        if (id < 0) record_error(kDevBadPosition);
        const unsigned long long k = id < 0 ? 0ull : kv4_key(best);
        if (p.ctas > 1) st_dsmem_u64(keys_s + pg * 8, 0, k);
        else keys[pg] = k;
      }
    }
    if (p.ctas > 1) cluster_sync_all();
  } else if (p.ctas > 1) {
    cluster_wait_acquire();
  }
  if (rank != 0) return;  // nothing reads this CTA's shared memory
  if (need >= n - 1) {    // every page
    for (int i = tid; i < p.n_sel; i += kKv4SelectThreads) {
      if (i < n && kv4_page_id(p.table, p.max_pages, p.n_pages, b, i) < 0) record_error(kDevBadPosition);
      sel[i] = i < n ? i : -1;
    }
    return;
  }
  if (tid == 0) {
    if (kv4_page_id(p.table, p.max_pages, p.n_pages, b, n - 1) < 0) record_error(kDevBadPosition);
    sel[need] = n - 1;
    sh_diff = 0;
  }
  if (need == 0) return;
  __syncthreads();
  // ---- the highest bit in which two bounds differ
  {
    unsigned long long d = 0;
    const unsigned long long k0 = keys[0];
    for (int i = tid; i < n - 1; i += kKv4SelectThreads) d |= keys[i] ^ k0;
    const unsigned hi = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(d >> 32));
    const unsigned lo = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(d));
    if (lane == 0 && (hi | lo)) atomicOr(&sh_diff, static_cast<unsigned long long>(hi) << 32 | lo);
  }
  __syncthreads();
  // ---- the need-th largest: of the keys that begin as `at` does down to bit `shift`, `left` are
  // to be taken, the larger ones all
  unsigned long long at = keys[0];
  int shift = sh_diff ? 64 - __clzll(sh_diff) : 0, left = need;
  at = shift < 64 ? at >> shift : 0;  // the common beginning
  while (shift > 0) {
    const int bits = min(8, shift);
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n - 1; i += kKv4SelectThreads) {
      const unsigned long long k = keys[i];
      if ((shift < 64 ? k >> shift : 0) == at) atomicAdd(&hist[k >> (shift - bits) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // digits from the top: the one at which the count from above reaches `left`
    const int mine = hist[255 - tid];
    int s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    if (lane == 31) scan[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; ++w) s += scan[w];
    if (s >= left && s - mine < left) {
      sh_digit = 255 - tid;
      sh_above = s - mine;
      sh_count = mine;
    }
    __syncthreads();
    shift -= bits;
    at = at << bits | static_cast<unsigned>(sh_digit);
    left -= sh_above;
    if (sh_count == left) break;  // every key that begins so is taken
  }
  // ---- in order: every thread a run of pages; above `at` all, at it the first `left`
  const int per = (n - 1 + kKv4SelectThreads - 1) / kKv4SelectThreads;
  const int i0 = min(n - 1, tid * per), i1 = min(n - 1, i0 + per);
  int above = 0, equal = 0;
  for (int i = i0; i < i1; ++i) {
    const unsigned long long k = shift < 64 ? keys[i] >> shift : 0;
    above += k > at;
    equal += k == at;
  }
  int both = above | (equal << 16), s = both;  // 16 bits each (n <= 16384)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += v;
  }
  __syncthreads();
  if (lane == 31) scan[warp] = s;
  __syncthreads();
  for (int w = 0; w < warp; ++w) s += scan[w];
  s -= both;
  int gt = s & 0xFFFF, eq = s >> 16;
  for (int i = i0; i < i1; ++i) {
    const unsigned long long k = shift < 64 ? keys[i] >> shift : 0;
    if (k > at || (k == at && eq < left)) sel[gt + min(eq, left)] = i;
    gt += k > at;
    eq += k == at;
  }
}

}  // namespace b2
