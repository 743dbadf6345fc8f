// Choosing the pages that a query attends to in a long cache, by a bound on their scores.
//
//   bound(page) = max over the kv head's q heads of sum_d max(q_d lo_d, q_d hi_d),
//
// lo and hi the page's key summary (per dim, over its tokens): no token of the page scores
// higher with any of the heads.  Per (sequence, kv head) the n_sel pages with the largest
// bounds are listed, in ascending order of the page; the page of the query's own position
// is always among them, and of two equal bounds the lower page goes first.
//
// Which page is the n_sel-th turns on the last bit of two bounds, so q is rotated and the
// sums are taken in fp64; the summaries are bf16, so that every product is exact.
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
  int* sel;        // [batch][hkv][n_sel]
  unsigned long long* key;  // [batch][hkv][key_pages]: bounds as rising integers
  int batch, hq, hkv, page, max_pages, n_pages, n_sel, key_pages;
};

// a double as an unsigned integer of the same order; NaN, -inf and pages that do not count are 0
__device__ __forceinline__ unsigned long long kv4_key(double x) {
  if (!(x > -INFINITY)) return 0;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int kKv4ScoreThreads = 128;
constexpr int kKv4ScorePages = 32;  // pages per CTA of the bounds' kernel

template <int D>
__global__ void __launch_bounds__(kKv4ScoreThreads) kv4_score_kernel(const Kv4SelectParams p,
                                                                    const __grid_constant__ Kv4Rope rope) {
  constexpr int J = D / 32, W = kKv4ScoreThreads / 32;
  __shared__ double q[kKv4MaxGroup][D];
  const int kvh = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = p.hq / p.hkv;
  pdl_wait();
  pdl_launch_dependents();
  const int pos = p.pos[b];
  if (pos < 0 || pos >= static_cast<long long>(p.max_pages) * p.page) return;  // the next kernel reports it
  const int last = min(pos / p.page, p.key_pages - 1);
  const int pg0 = blockIdx.x * kKv4ScorePages;
  if (pg0 > last) return;
  for (int e = threadIdx.x; e < grp * (D / 2); e += kKv4ScoreThreads) {
    const int j = e / (D / 2), i = e % (D / 2);
    const float* src = p.q + static_cast<size_t>(b) * p.ld_q + static_cast<size_t>(kvh * grp + j) * D;
    const double a = src[i], z = src[i + D / 2];
    double sn = 0.0, cs = 1.0;
    if (rope.on) {
      double u = static_cast<double>(pos) * rope.turn[i];
      u -= rint(u);
      sincospi(2.0 * u, &sn, &cs);
    }
    q[j][i] = a * cs - z * sn;
    q[j][i + D / 2] = z * cs + a * sn;
  }
  __syncthreads();
  unsigned long long* key = p.key + (static_cast<size_t>(b) * p.hkv + kvh) * p.key_pages;
  for (int pg = pg0 + warp; pg <= last && pg < pg0 + kKv4ScorePages; pg += W) {
    const int id = kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg);
    if (id < 0) {
      if (lane == 0) {
        record_error(kDevBadPosition);
        key[pg] = 0;
      }
      continue;
    }
    const __nv_bfloat16* sm = p.summary + (static_cast<size_t>(id) * p.hkv + kvh) * 2 * D + lane;
    double lo[J], hi[J];
#pragma unroll
    for (int i = 0; i < J; ++i) {
      lo[i] = __bfloat162float(sm[32 * i]);
      hi[i] = __bfloat162float(sm[D + 32 * i]);
    }
    double best = -INFINITY;
    for (int j = 0; j < grp; ++j) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < J; ++i) {
        const double x = q[j][lane + 32 * i];
        s = fma(x, x > 0.0 ? hi[i] : lo[i], s);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      best = fmax(best, s);
    }
    if (lane == 0) key[pg] = pg == last ? ~0ull : max(kv4_key(best), 1ull);
  }
}

constexpr int kKv4PickThreads = 256;

// One CTA per (sequence, kv head): the n_sel-th largest key by 8-bit digits, then the pages
// above it and the first of those at it, written in order.
__global__ void __launch_bounds__(kKv4PickThreads) kv4_pick_kernel(const Kv4SelectParams p) {
  extern __shared__ unsigned long long keys[];
  __shared__ int hist[256], scan[kKv4PickThreads / 32 + 1];
  __shared__ unsigned long long sh_prefix;
  __shared__ int sh_need;
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  int* sel = p.sel + (static_cast<size_t>(b) * p.hkv + kvh) * p.n_sel;
  const int pos = p.pos[b];
  if (pos < 0 || pos >= static_cast<long long>(p.max_pages) * p.page || pos / p.page >= p.key_pages) {
    if (pos != -1 && tid == 0) record_error(kDevBadPosition);
    for (int i = tid; i < p.n_sel; i += kKv4PickThreads) sel[i] = -1;
    return;
  }
  const int n = pos / p.page + 1;
  const unsigned long long* key = p.key + (static_cast<size_t>(b) * p.hkv + kvh) * p.key_pages;
  for (int i = tid; i < n; i += kKv4PickThreads) keys[i] = key[i];
  unsigned long long at = 0;  // the n_sel-th largest key; ties at it taken: `need`
  int need = p.n_sel;
  __syncthreads();
  if (n > p.n_sel) {
    for (int shift = 56; shift >= 0; shift -= 8) {
      hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kKv4PickThreads) {
        const unsigned long long k = keys[i];
        if (shift == 56 || (k >> (shift + 8)) == (at >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      // digits from the top: the one at which the count from above reaches need
      const int mine = hist[255 - tid];
      int s = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
      }
      if (lane == 31) scan[warp] = s;
      __syncthreads();
      int before = 0;
      for (int w = 0; w < warp; ++w) before += scan[w];
      s += before;
      if (s >= need && s - mine < need) {
        sh_prefix = at | (static_cast<unsigned long long>(255 - tid) << shift);
        sh_need = need - (s - mine);
      }
      __syncthreads();
      at = sh_prefix;
      need = sh_need;
    }
  }
  // in order: every thread takes a run of pages
  const int per = (n + kKv4PickThreads - 1) / kKv4PickThreads;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int above = 0, equal = 0;
  for (int i = i0; i < i1; ++i) {
    above += keys[i] > at;
    equal += keys[i] == at;
  }
  // exclusive sums of both over the threads, 16 bits each (n <= 16384)
  int both = above | (equal << 16), s = both;
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
    const bool up = keys[i] > at, tie = keys[i] == at;
    if (up || (tie && eq < need)) sel[gt + min(eq, need)] = i;
    gt += up;
    eq += tie;
  }
  for (int i = n + tid; i < p.n_sel; i += kKv4PickThreads) sel[i] = -1;
}

}  // namespace b2
