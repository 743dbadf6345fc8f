// Choosing the pages that a query attends to in a long cache, by a bound on their scores.
//
//   bound(page) = max over the kv head's q heads of sum_d max(q_d lo_d, q_d hi_d),
//
// lo and hi the page's key summary (per dim, over its tokens): but for the roundings of the
// summary to bf16 and of the keys to 4 bits no token of the page scores higher with any of
// the heads.  Per (sequence, kv head) the n_sel pages with the largest bounds are listed, in
// ascending order of the page; the page of the query's own position is always among them, and
// of two equal bounds the lower page goes first.
//
// The bounds are products of a pages x 2 D matrix, the summaries as they lie in memory, with the
// heads' min(q, 0) and max(q, 0), so the tensor cores take them: mma.sync m16n8k16 of bf16, q in
// three parts that sum to its 24 bits, 16 pages x 8 heads a warp at a time (16 sequences x 8 kv
// heads of up to 1024 pages: 14.0 us, where fp32 FMAs took 22.6).  Two CTAs per SM spill 44 and 80 bytes
// at head_dim 128 and 256; one (162 and 224 registers) makes select and decode of 16 sequences of
// 1 to 32768 51.3 us instead of 46.5, and 48.9 instead of 44.1.
//
// Which page is the n_sel-th may turn on the last bit of two bounds.  With E, a bound on what the
// fp32 sums are off, the choice is the exact one where the last page taken and the first left out
// are further apart than 2 E.  Where not (rarely with random keys; always with equal bounds), the
// pages within 2 E of the border are summed again in fp64, with q turned in fp64 and the
// summaries bf16, every product exact, and chosen by that.  (In fp64 throughout: 45 us.)
//
// A cluster per (sequence, kv head): its CTAs take every further group of pages and push the
// bounds into the first CTA's shared memory, which finds the n_sel-th by 8-bit digits from the
// highest bit in which they differ, until a digit settles it (two or three rounds), and writes
// the pages in order.  That tail is what bounds a small call, about 3.5 us of 7.0 for one sequence
// of 512 pages; the bytes of the summaries would take 2.6 of the 14.0 us.
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
  int max_len;    // tokens planned for
  int key_pages;  // in pages
  int ctas;       // of a cluster
};

// Numbers as unsigned integers of the same order, 1 or more; NaN and -inf are 1.
__device__ __forceinline__ unsigned kv4_key(float x) {
  if (!(x > -INFINITY)) return 1;
  const unsigned u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long kv4_key(double x) {
  if (!(x > -INFINITY)) return 1;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int kKv4SelectThreads = 256;

// The need-th largest of n keys (0 < need < n): on return those whose bits from `shift` up are
// above `at` are `need` - `left`, and of those at it the first `left` belong to them; `whole`
// if those at it are `left`.
struct Kv4Nth {
  unsigned long long at;
  int shift, left;
  bool whole;
};
struct Kv4NthShared {
  int hist[256], scan[kKv4SelectThreads / 32], digit, above, count;
  unsigned long long diff;
};
template <typename F>
__device__ __forceinline__ Kv4Nth kv4_nth(const F& key, int n, int need, Kv4NthShared& sh) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) sh.diff = 0;
  __syncthreads();
  const unsigned long long k0 = key(0);
  unsigned long long d = 0;
  for (int i = tid; i < n; i += kKv4SelectThreads) d |= key(i) ^ k0;
  const unsigned hi = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(d >> 32));
  const unsigned lo = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(d));
  if (lane == 0 && (hi | lo)) atomicOr(&sh.diff, static_cast<unsigned long long>(hi) << 32 | lo);
  __syncthreads();
  Kv4Nth r;
  r.shift = sh.diff ? 64 - __clzll(sh.diff) : 0;
  r.at = r.shift < 64 ? k0 >> r.shift : 0;  // the common beginning
  r.left = need;
  r.whole = false;
  while (r.shift > 0 && !r.whole) {
    const int bits = min(8, r.shift);
    sh.hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kKv4SelectThreads) {
      const unsigned long long k = key(i);
      if ((r.shift < 64 ? k >> r.shift : 0) == r.at) atomicAdd(&sh.hist[k >> (r.shift - bits) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // digits from the top: the one at which the count from above reaches `left`
    const int mine = sh.hist[255 - tid];
    int s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    if (lane == 31) sh.scan[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; ++w) s += sh.scan[w];
    if (s >= r.left && s - mine < r.left) {
      sh.digit = 255 - tid;
      sh.above = s - mine;
      sh.count = mine;
    }
    __syncthreads();
    r.shift -= bits;
    r.at = r.at << bits | static_cast<unsigned>(sh.digit);
    r.left -= sh.above;
    r.whole = sh.count == r.left;
  }
  return r;
}

__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 64 dims of 16 pages' summaries as a warp holds them: of pages gl and gl + 8 (gl = lane / 4),
// lo and hi, the 8 dims from 8 c and from 32 + 8 c on (c = lane % 4), bf16 as they are stored
struct Kv4Near {
  uint4 v[2][2][2];
};

template <int D>
__global__ void __launch_bounds__(kKv4SelectThreads, 2) kv4_select_kernel(const Kv4SelectParams p,
                                                                      const __grid_constant__ Kv4Rope rope) {
  constexpr int G = D / 64, W = kKv4SelectThreads / 32;
  extern __shared__ __align__(16) unsigned long long exact[];  // [key_pages], then the fp32 bounds (the first CTA's)
  float* const bound = reinterpret_cast<float*>(exact + p.key_pages);
  __shared__ uint2 qb[G][8][3][32];  // B operands: 64 dims; lo or hi, 16 dims; a bf16 part of q; lane
  __shared__ double turn_s[2][D / 2];
  __shared__ float size[W];
  __shared__ unsigned most;  // the largest sum_d qa |lo or hi| of a page, its bits (the first CTA's)
  __shared__ int n_close;
  __shared__ float in_least[W], out_most[W];
  __shared__ Kv4NthShared nth_s;
  const int rank = blockIdx.x % p.ctas, kvh = blockIdx.x / p.ctas, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = p.hq / p.hkv;
  if (tid == 0) most = 0;
  if (p.ctas > 1) {
    __syncthreads();
    cluster_arrive_release();  // waited for before anything is pushed
  }
  pdl_wait();
  pdl_launch_dependents();
  int* sel = p.sel + (static_cast<size_t>(b) * p.hkv + kvh) * p.n_sel;
  const int pos = p.pos[b];
  if (pos < 0 || pos >= static_cast<long long>(p.max_pages) * p.page || pos >= p.max_len) {
    if (rank == 0) {
      if (pos != -1 && tid == 0) record_error(kDevBadPosition);
      for (int i = tid; i < p.n_sel; i += kKv4SelectThreads) sel[i] = -1;
    }
    if (p.ctas > 1) cluster_wait_acquire();
    return;  // the whole cluster
  }
  const int n = pos / p.page + 1;  // pages; the last is chosen without a bound
  const int need = p.n_sel - 1;    // of the n - 1 others
  if (need >= n - 1 || need == 0) {
    if (rank == 0)
      for (int i = tid; i < p.n_sel; i += kKv4SelectThreads) {
        const int pg = need == 0 ? n - 1 : i;
        if (pg < n && kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg) < 0) record_error(kDevBadPosition);
        sel[i] = pg < n ? pg : -1;
      }
    if (p.ctas > 1) cluster_wait_acquire();
    return;
  }
  const int gl = lane >> 2, c = lane & 3;
  auto find = [&](int pg) { return pg < n - 1 ? kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg) : -1; };
  auto load = [&](const int (&id)[2], int g, Kv4Near& x) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const __nv_bfloat16* sm = p.summary + (static_cast<size_t>(max(id[r], 0)) * p.hkv + kvh) * 2 * D + 64 * g + 8 * c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x.v[r][e >> 1][e & 1] = id[r] < 0 ? make_uint4(0, 0, 0, 0)
                                          : *reinterpret_cast<const uint4*>(sm + (e >> 1) * D + 32 * (e & 1));
    }
  };
  // ---- the first pages' summaries set out; q turned to pos
  const int step = p.ctas * W * 16;
  int pg = (rank * W + warp) * 16 + gl;  // and pg + 8
  Kv4Near x;
  int id[2] = {find(pg), find(pg + 8)}, id_next[2] = {find(pg + step), find(pg + step + 8)};
  load(id, 0, x);
  if (rope.on) {
    for (int i = tid; i < D / 2; i += kKv4SelectThreads) {
      double u = static_cast<double>(pos) * kv4_turn(rope, i);
      u -= rint(u);
      kv4_cos_sin(u, turn_s[0][i], turn_s[1][i]);
    }
    __syncthreads();
  }
  // value i or i + D / 2 of head j, turned
  auto turned = [&](int j, int i, bool second) -> double {
    const float* src = p.q + static_cast<size_t>(b) * p.ld_q + static_cast<size_t>(kvh * grp + j) * D;
    const double a = src[i], z = src[i + D / 2];
    if (!rope.on) return second ? z : a;
    const double c = turn_s[0][i], s = turn_s[1][i];
    return second ? z * c + a * s : a * c - z * s;
  };
  // the B operands: below zero for lo, above for hi, three bf16 that sum to q's 24 bits
  float top = 0.f;
  for (int e = tid; e < kKv4MaxGroup * (D / 4); e += kKv4SelectThreads) {
    const int j = e % kKv4MaxGroup, d0 = e / kKv4MaxGroup * 4;
    uint32_t w[2][3][2] = {};
    if (j < grp) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + i;
        float v = static_cast<float>(turned(j, d % (D / 2), d >= D / 2));
        if (v != 0.f && fabsf(v) < 7.9e-31f) top = INFINITY;  // too small for the parts: all in fp64
        const int side = v > 0.f;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const __nv_bfloat16 h = __float2bfloat16_rn(v);
          v -= __bfloat162float(h);
          w[0][k][i >> 1] |= side ? 0u : static_cast<uint32_t>(__bfloat16_as_ushort(h)) << (16 * (i & 1));
          w[1][k][i >> 1] |= side ? static_cast<uint32_t>(__bfloat16_as_ushort(h)) << (16 * (i & 1)) : 0u;
        }
      }
    }
    const int at = d0 % 64, chunk = at / 8;  // chunk 4 i + c, its first or second half
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int side = 0; side < 2; ++side)
        qb[d0 / 64][side * 4 + chunk / 4 * 2 + at / 4 % 2][k][j * 4 + chunk % 4] = make_uint2(w[side][k][0], w[side][k][1]);
  }
  __syncthreads();
  if (p.ctas > 1) cluster_wait_acquire();
  // ---- the bounds in fp32: 16 pages x 8 heads a warp at a time
  const uint32_t bound_s = smem_u32(bound);
  while (pg - gl < n - 1) {
    float s[4] = {}, low[4] = {}, all[4] = {};  // sums of q's first part, of the others, of the products' sizes
    int id_after[2] = {find(pg + 2 * step), find(pg + 2 * step + 8)};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      Kv4Near y;
      if (g + 1 < G) load(id, g + 1, y);
      else load(id_next, 0, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 u = x.v[0][k >> 2][k >> 1 & 1], v = x.v[1][k >> 2][k >> 1 & 1];
        const uint32_t a0 = k & 1 ? u.z : u.x, a1 = k & 1 ? v.z : v.x, a2 = k & 1 ? u.w : u.y, a3 = k & 1 ? v.w : v.y;
        const uint2 b0 = qb[g][k][0][lane], b1 = qb[g][k][1][lane], b2 = qb[g][k][2][lane];
        constexpr uint32_t kAbs = 0x7FFF7FFFu;
        float first[4];  // summed outside: 16 products each stay near enough for E
        mma_bf16_first(first, a0, a1, a2, a3, b0.x, b0.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += first[e];
        mma_bf16_m16n8k16(low[0], low[1], low[2], low[3], a0, a1, a2, a3, b1.x, b1.y);
        mma_bf16_m16n8k16(low[0], low[1], low[2], low[3], a0, a1, a2, a3, b2.x, b2.y);
        mma_bf16_m16n8k16(all[0], all[1], all[2], all[3], a0 & kAbs, a1 & kAbs, a2 & kAbs, a3 & kAbs, b0.x & kAbs,
                          b0.y & kAbs);
      }
      x = y;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float best = -INFINITY;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (2 * c + e < grp) {
          const float size = all[2 * r + e];
          best = fmaxf(best, s[2 * r + e] + low[2 * r + e]);
          top = size <= top ? top : size < INFINITY ? size : INFINITY;  // NaN too: nothing is then decided in fp32
        }
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
      const int at = pg + 8 * r;
      if (at < n - 1 && c == 0) {
        if (id[r] < 0) {
          record_error(kDevBadPosition);
          best = -INFINITY;
        }
        if (p.ctas > 1) st_dsmem_f32(bound_s + at * 4, 0, best);
        else bound[at] = best;
      }
      id[r] = id_next[r];
      id_next[r] = id_after[r];
    }
    pg += step;
  }
  top = warp_max(top);
  if (lane == 0) size[warp] = top;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, size[w]);
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(&most)));
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(to), "r"(__float_as_uint(top)) : "memory");
  }
  if (p.ctas > 1) cluster_sync_all();
  else __syncthreads();
  if (rank != 0) return;  // nothing reads this CTA's shared memory

  // ---- the need largest bounds
  if (tid == 0) {
    if (kv4_page_id(p.table, p.max_pages, p.n_pages, b, n - 1) < 0) record_error(kDevBadPosition);
    sel[need] = n - 1;
  }
  auto key = [&](int i) { return static_cast<unsigned long long>(kv4_key(bound[i])); };
  Kv4Nth t = kv4_nth(key, n - 1, need, nth_s);
  // E: of 16 exact products, summed to single precision, each sum is off by 2^-23 of their sizes'
  // sum at most; then D / 8 fp32 sums, half as much each.  The sizes' own sum is that of the first
  // parts, within 1%; q's rounding, its other parts (4 D sums, 2^-9 as large) and the last sum are
  // below 4 such roundings.
  const float off = __uint_as_float(most) * ((16 + D / 16 + 4) * 1.02f * 1.1920929e-7f);
  float least = INFINITY, first_out = -INFINITY;  // of those taken, of those left out
  for (int i = tid; i < n - 1; i += kKv4SelectThreads) {
    if ((key(i) >> t.shift) >= t.at) least = fminf(least, bound[i]);
    else first_out = fmaxf(first_out, bound[i]);
  }
  least = -warp_max(-least);
  first_out = warp_max(first_out);
  if (lane == 0) {
    in_least[warp] = least;
    out_most[warp] = first_out;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    least = fminf(least, in_least[w]);
    first_out = fmaxf(first_out, out_most[w]);
  }
  const bool sure = t.whole && least - first_out > 2.f * off;  // false where off is not finite
  if (!sure) {
    // ---- again for those within 2 E of the border, in fp64: a warp a page
    if (tid == 0) n_close = 0;
    __syncthreads();
    int* const close = reinterpret_cast<int*>(bound);  // their list takes the bounds' place, from below
    int n_in = 0;
    for (int i0 = 0; i0 < n - 1; i0 += kKv4SelectThreads) {
      const int i = i0 + tid;
      const float v = i < n - 1 ? bound[i] : 0.f;
      const bool in = v > least + 2.f * off, out = v < least - 2.f * off;
      if (i < n - 1) exact[i] = in ? ~0ull : 0ull;
      n_in += __syncthreads_count(i < n - 1 && in);  // and these bounds have been read
      if (i < n - 1 && !in && !out) close[atomicAdd(&n_close, 1)] = i;
      __syncthreads();
    }
    for (int c = warp; c < n_close; c += W) {
      const int i = close[c], page = kv4_page_id(p.table, p.max_pages, p.n_pages, b, i);
      unsigned long long k = 1;
      if (page >= 0) {
        const __nv_bfloat16* sm = p.summary + (static_cast<size_t>(page) * p.hkv + kvh) * 2 * D;
        double best = -INFINITY;
        for (int j = 0; j < grp; ++j) {
          double s = 0.0;
          for (int d = lane; d < D / 2; d += 32)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const double v = turned(j, d, e);
              s = fma(v, static_cast<double>(__bfloat162float(sm[(v > 0.0 ? D : 0) + d + e * (D / 2)])), s);
            }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          best = fmax(best, s);
        }
        k = min(kv4_key(best), ~0ull - 1);
      }
      if (lane == 0) exact[i] = k;
    }
    __syncthreads();
    if (n_close <= kKv4SelectThreads) {  // each against the others: of those at hand need - n_in are taken
      const int i = tid < n_close ? close[tid] : 0;
      const unsigned long long k = exact[i];
      int ahead = 0;
      for (int c = 0; c < n_close; ++c) {
        const unsigned long long o = exact[close[c]];
        ahead += o > k || (o == k && close[c] < i);
      }
      __syncthreads();
      if (tid < n_close) exact[i] = ahead < need - n_in ? ~0ull : 0ull;
      __syncthreads();
      t.at = ~0ull;
      t.shift = 0;
      t.left = need;
    } else {
      t = kv4_nth([&](int i) { return exact[i]; }, n - 1, need, nth_s);
    }
  }
  // ---- in order: every thread a run of pages; above `at` all, at it the first `left`
  const int per = (n - 1 + kKv4SelectThreads - 1) / kKv4SelectThreads;
  const int i0 = min(n - 1, tid * per), i1 = min(n - 1, i0 + per);
  auto place = [&](int i) {
    const unsigned long long k = sure ? key(i) : exact[i];
    return t.shift < 64 ? k >> t.shift : 0ull;
  };
  int above = 0, equal = 0;
  for (int i = i0; i < i1; ++i) {
    above += place(i) > t.at;
    equal += place(i) == t.at;
  }
  int both = above | (equal << 16), s = both;  // 16 bits each (n <= 16384)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += v;
  }
  __syncthreads();
  if (lane == 31) nth_s.scan[warp] = s;
  __syncthreads();
  for (int w = 0; w < warp; ++w) s += nth_s.scan[w];
  s -= both;
  int gt = s & 0xFFFF, eq = s >> 16;
  for (int i = i0; i < i1; ++i) {
    const unsigned long long k = place(i);
    if (k > t.at || (k == t.at && eq < t.left)) sel[gt + min(eq, t.left)] = i;
    gt += k > t.at;
    eq += k == t.at;
  }
}

}  // namespace b2
