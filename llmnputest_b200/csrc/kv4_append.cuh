// Appending rows to the 4-bit paged KV cache, and reading rows back.
//
//   append  k of every new row is rotated to its position (half-split RoPE, in fp64), then
//           per (token, kv head, 64 dims) of k and of v
//             m = bf16(min x), d = max(bf16((max x - m) / 15), 2^-40),
//             code = clamp(floor((x - m) / d + 1/2), 0, 15)
//           and the page's key summary (min and max per dim, bf16) takes the new keys in.
//   gather  code * d + m of the rows asked for.
//
// The codes are whole numbers that turn on the last bit of x at a border between two of
// them, and are to be the same whatever the order of evaluation.  So keys are turned in fp64: a
// lane's first token by its own sine and cosine, every further one by a complex multiplication
// with the turn of the positions between the two (16 at head_dim 64, 8 at 128, 4 at 256), whose
// sine and cosine are evaluated once a page.  Every choice is made in fp32 with a bound on its
// error; the few that lie within the bound of a border (1 in 10^4 or less) are made again in
// fp64.
//
// One CTA per (page of a sequence, kv head), so that the page's summary needs no second pass.
// D / 8 lanes have a token, each two quads of dims (4 l and D / 2 + 4 l: the pairs that turn
// together), so that what is done once per 64 values is done for 32 / (D / 8) tokens at a
// time: 168 instructions a token and head of 64 dims, where a warp per token executed 282.  The
// codes are put together in shared memory as the cell's bytes.
//
// What bounds it: those instructions and their latency (2 x 64 values turned, compared and
// divided; under half of the issue slots are used), in two rounds of CTAs, four per SM.  8192
// tokens of 8 heads of 64 in four prompts, appended and read back, take 27.7 us, 9.2 by the
// bytes; one token for each of 64 sequences 8.4 us, two launches and their chains of loads.
// Five CTAs per SM spill registers (24 to 60 bytes): 28.6 us, and 36.6 against 32.8 for 4096
// tokens of 8 heads of 128; six and eight measured no less than five.
#pragma once

#include "kv4_cell.cuh"

namespace b2 {

constexpr int kKv4AppendThreads = 128;

struct Kv4RowsParams {
  const void* k;  // [rows][ld]: kv head h at h * D (append: in, gather: out)
  const void* v;
  long long ld_k, ld_v;
  uint8_t* pool;  // [n_pages][hkv][page / 16][D / 64][1152]
  const int* table;  // [batch][max_pages]
  const int* pos;    // [batch] position of the first row of each sequence; -1: none
  const int* cu;     // [batch + 1] row offsets, or null: one row per sequence
  __nv_bfloat16* summary;  // [n_pages][hkv][2][D] min, max of the page's keys, or null
  int rows, batch, hkv, page, max_pages, n_pages;
  int is_f32;  // k and v are fp32 (else bf16)
  int wide;    // append: four values of a row can be loaded at once
};

__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// The choices that fp32 cannot make, out of line: a few in 10^4.
template <int RL>
__device__ __noinline__ float kv4_step_fp64(double top, float m) {
#pragma unroll
  for (int o = RL / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
  return static_cast<float>((top - m) / 15.0);
}
__device__ __noinline__ uint32_t kv4_code_fp64(double x, float m, float d) {
  return static_cast<uint32_t>(fmin(fmax(floor((x - m) / d + 0.5), 0.0), 15.0));
}

// Two fp32 as bf16, hi in the upper half.
__device__ __forceinline__ uint32_t bf16x2_of(float hi, float lo) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The codes of 64 values, NV in each of RL lanes in a row (x(i) in fp64; f their fp32
// roundings), 4 bits each from the lowest, and (d, m).  The whole warp takes part.
template <int RL, int NV, typename X>
__device__ __forceinline__ uint32_t kv4_quantise(const X& x, const float (&f)[NV], uint32_t& meta) {
  float mn = f[0], mx = f[0], odd = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    mn = fminf(mn, f[i]);
    mx = fmaxf(mx, f[i]);
    odd = fmaf(f[i], 0.f, odd);  // NaN if a value is not finite
  }
#pragma unroll
  for (int o = RL / 2; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const unsigned bad = __ballot_sync(0xffffffffu, isnan(odd));
  const uint32_t mb = bf16x2_of(mn, mn) & 0xFFFF0000u;  // the rounding is monotone: that of the least x itself
  const float m = __uint_as_float(mb);
  // (max x - m) / 15: fp32 is off by 2^-22 of it, or of max x, at most; where bf16's rounding
  // could see that, in fp64
  const float q = (mx - m) * (1.f / 15.f);
  const float reach = fmaxf(fabsf(mx), fabsf(mn)) + fabsf(m), slack = reach * 2.4e-7f;
  const uint32_t both = bf16x2_of(q + slack, q - slack);
  float d = __uint_as_float(both & 0xFFFF0000u);
  const bool unsure = both >> 16 != (both & 0xFFFFu);
  if (__any_sync(0xffffffffu, unsure)) {
    double top = x(0);
#pragma unroll
    for (int i = 1; i < NV; ++i) top = fmax(top, x(i));
    const float sure = round_bf16(kv4_step_fp64<RL>(top, m));
    if (unsure) d = sure;
  }
  d = fmaxf(d, kKv4MinStep);
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(d));
  // (x - m) / d in fifteenths, off by 2^-21 of what enters it at most, clamped to 0..1 in the same
  // instruction; 15 of it to the nearest whole number in the low bits of 3 * 2^22 + it.  Nearer
  // than that to half a step between two, in fp64 (as where 1 / 15 d would be subnormal).
  const float part = inv * (1.f / 15.f), nm = -m * part;
  const float near = part > 1e-37f ? 0.5f - fmaf(reach * inv, 4.8e-7f, 1e-5f) : 0.f;
  float off = 0.f, sum[NV / 4];  // sum: four codes, 2^23 + c0 + 16 c1 + ...
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float z = __saturatef(fmaf(f[i], part, nm)), t = fmaf(z, 15.f, 12582912.f) - 12582912.f;
    off = fmaxf(off, fabsf(fmaf(z, 15.f, -t)));
    sum[i / 4] = fmaf(t, static_cast<float>(1 << 4 * (i % 4)), i % 4 ? sum[i / 4] : 8388608.f);
  }
  uint32_t code = NV == 8 ? prmt(__float_as_uint(sum[0]), __float_as_uint(sum[NV / 4 - 1]), 0x5410u)
                          : __float_as_uint(sum[0]) & 0xFFFFu;
  const bool border = !(off < near);
  if (__any_sync(0xffffffffu, border)) {
    if (border) {
      code = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) code |= kv4_code_fp64(x(i), m, d) << (4 * i);
    }
  }
  meta = (__float_as_uint(d) >> 16) | mb;
  // a value that is not finite makes its 64 NaN: 4 bits have no such value
  const int lane = threadIdx.x & 31;
  if (bad >> (lane & ~(RL - 1)) & ((RL == 32 ? 0u : 1u << RL) - 1u)) {
    code = 0;
    meta = 0x7FC00000u | (__float_as_uint(kKv4MinStep) >> 16);
  }
  return code;
}

// Four values of a row, fp32 or bf16 (16 or 8 bytes where the rows are aligned so).
__device__ __forceinline__ void kv4_load4(const char* src, bool f32, bool wide, float (&x)[4]) {
  if (f32) {
    const float* v = reinterpret_cast<const float*>(src);
    if (wide) {
      const float4 w = *reinterpret_cast<const float4*>(v);
      x[0] = w.x;
      x[1] = w.y;
      x[2] = w.z;
      x[3] = w.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = v[i];
    }
  } else {
    const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(src);
    if (wide) {
      const uint2 w = *reinterpret_cast<const uint2*>(v);
      x[0] = bf16lo_to_f32(w.x);
      x[1] = bf16hi_to_f32(w.x);
      x[2] = bf16lo_to_f32(w.y);
      x[3] = bf16hi_to_f32(w.y);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(v[i]);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kKv4AppendThreads, 4) kv4_append_kernel(const Kv4RowsParams p,
                                                                          const __grid_constant__ Kv4Rope rope) {
  constexpr int G = D / kKv4Group, W = kKv4AppendThreads / 32;
  constexpr int LR = D / 8, RW = 32 / LR, STEP = W * RW;  // lanes of a token, tokens of a warp, of the CTA
  // a lane's 8 values are of one group of 64 (D = 64) or of two
  constexpr int RL = D == 64 ? 8 : 16, NV = D == 64 ? 8 : 4, U = 8 / NV;
  __shared__ __align__(16) uint8_t image[G * kKv4CellBytes];
  __shared__ double turn_s[2][D / 2];  // cos, sin of the turn of STEP positions
  __shared__ float low[W][D], high[W][D];
  __shared__ int job_seq, job_page;

  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = lane % LR, mine = warp * RW + lane / LR;  // this lane's place in its token; its token of STEP
  pdl_wait();
  pdl_launch_dependents();
  int b = blockIdx.x, pg = 0;
  if (p.cu) {
    if (warp == 0) {
      b = kv4_find_job(p.cu, p.pos, p.rows, p.batch, p.page, blockIdx.x, pg);
      if (lane == 0) {
        job_seq = b;
        job_page = pg;
      }
    }
    __syncthreads();
    b = job_seq;
    pg = job_page;
    if (b < 0) return;
  }
  int row0, row1;
  kv4_rows(p.cu, p.rows, b, row0, row1);
  const int pos = p.pos[b];
  if (!p.cu) pg = max(pos, 0) / p.page;
  if (pos == -1 || row1 <= row0) return;
  const int id = pos < 0 ? -1 : kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg);
  if (id < 0) {  // outside the table or the pool: record, write nothing
    if (threadIdx.x == 0) record_error(kDevBadPosition);
    return;
  }
  // this page's new tokens: offsets [t0, t1) of the page
  const long long base = static_cast<long long>(pg) * p.page;
  const int t0 = static_cast<int>(max(static_cast<long long>(pos), base) - base);
  const int t1 = static_cast<int>(min(static_cast<long long>(pos) + (row1 - row0), base + p.page) - base);
  const int first = t0 / kKv4Tile * kKv4Tile;
  uint8_t* cells = p.pool + (static_cast<size_t>(id) * p.hkv + h) * (static_cast<size_t>(p.page / kKv4Tile) * G * kKv4CellBytes);

  // the rows' bytes, from this lane's first token on; a token ahead of the work on it
  const long long esize = p.is_f32 ? 4 : 2, row = row0 + (base + first + mine - pos);
  const char* k_at = static_cast<const char*>(p.k) + (row * p.ld_k + static_cast<long long>(h) * D + 4 * l) * esize;
  const char* v_at = static_cast<const char*>(p.v) + (row * p.ld_v + static_cast<long long>(h) * D + 4 * l) * esize;
  const long long k_step = STEP * p.ld_k * esize, v_step = STEP * p.ld_v * esize, half = D / 2 * esize;
  float k_in[2][4], v_in[2][4];
  auto load = [&](int at) {
    if (at >= t0 && at < t1) {
      kv4_load4(k_at, p.is_f32, p.wide, k_in[0]);
      kv4_load4(k_at + half, p.is_f32, p.wide, k_in[1]);
      kv4_load4(v_at, p.is_f32, p.wide, v_in[0]);
      kv4_load4(v_at + half, p.is_f32, p.wide, v_in[1]);
    } else {  // its codes are not kept
#pragma unroll
      for (int i = 0; i < 8; ++i) k_in[i / 4][i % 4] = v_in[i / 4][i % 4] = 0.f;
    }
    k_at += k_step;
    v_at += v_step;
  };
  load(first + mine);

  // the turn of this lane's first token; that of the STEP positions to its next one
  const bool several = first + STEP < t1;
  double cs[4], sn[4];
  if (rope.on) {
    if (several && threadIdx.x < D / 2) {
      double u = STEP * kv4_turn(rope, threadIdx.x);
      u -= rint(u);
      kv4_cos_sin(u, turn_s[0][threadIdx.x], turn_s[1][threadIdx.x]);
    }
    const double at = static_cast<double>(base + first + mine);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      double u = at * kv4_turn(rope, 4 * l + i);
      u -= rint(u);
      kv4_cos_sin(u, cs[i], sn[i]);
    }
    if (several) __syncthreads();
  }
  // least and largest keys of the lane's dims, as bf16 pairs: the rounding is monotone
  __nv_bfloat162 lo_k[4], hi_k[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo_k[i] = __float2bfloat162_rn(INFINITY);
    hi_k[i] = __float2bfloat162_rn(-INFINITY);
  }

  for (int tile = first; tile < t1; tile += kKv4Tile) {
#pragma unroll 1
    for (int t = mine; t < kKv4Tile; t += STEP) {
      const int at = tile + t;
      const bool fresh = at >= t0 && at < t1;
      float k[8], f[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        k[i] = k_in[i / 4][i % 4];
        v[i] = v_in[i / 4][i % 4];
      }
      load(at + STEP);
      auto turned = [&](int i) -> double {  // value i of the lane's eight keys
        const int j = i & 3;
        const double a = k[j], c = k[4 + j];
        if (!rope.on) return i < 4 ? a : c;
        return i < 4 ? a * cs[j] - c * sn[j] : c * cs[j] + a * sn[j];
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(turned(i));
      if (fresh) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 r = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          lo_k[i] = __hmin2(lo_k[i], r);
          hi_k[i] = __hmax2(hi_k[i], r);
        }
      }
      // the codes of the lane's two quads, and the (d, m) of their groups, into the cells' bytes
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint32_t quad[2], dm[2];
        if (U == 1) {
          const uint32_t c = which ? kv4_quantise<RL, 8>([&](int i) { return static_cast<double>(v[i]); }, v, dm[0])
                                   : kv4_quantise<RL, 8>(turned, f, dm[0]);
          quad[0] = c & 0xFFFFu;
          quad[1] = c >> 16;
          dm[1] = dm[0];
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float fu[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fu[i] = which ? v[4 * u + i] : f[4 * u + i];
            quad[u] = which ? kv4_quantise<RL, 4>([&](int i) { return static_cast<double>(fu[i]); }, fu, dm[u])
                            : kv4_quantise<RL, 4>([&](int i) { return turned(4 * u + i); }, fu, dm[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int dim = 4 * l + u * (D / 2), g = dim / kKv4Group, in = dim % kKv4Group;
          uint8_t* cell = image + g * kKv4CellBytes;
          const int to = which ? kv4_v_half(t, in / 4) : kv4_k_word(t, in / 8) + (in / 4 % 2) * 2;
          *reinterpret_cast<uint16_t*>(cell + to) = static_cast<uint16_t>(quad[u]);
          if (in == 0) *reinterpret_cast<uint32_t*>(cell + (which ? kKv4VMeta : kKv4KMeta) + kv4_meta(t)) = dm[u];
        }
      }
      if (rope.on && several) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double c = cs[i], wc = turn_s[0][4 * l + i], ws = turn_s[1][4 * l + i];
          cs[i] = c * wc - sn[i] * ws;
          sn[i] = sn[i] * wc + c * ws;
        }
      }
    }
    __syncthreads();
    uint8_t* cell0 = cells + static_cast<size_t>(tile / kKv4Tile) * G * kKv4CellBytes;
    if (tile >= t0 && tile + kKv4Tile <= t1) {
      for (int e = threadIdx.x; e < G * kKv4CellBytes / 16; e += kKv4AppendThreads)
        reinterpret_cast<uint4*>(cell0)[e] = reinterpret_cast<const uint4*>(image)[e];
    } else {  // the tokens beside the new ones stay: 2 bytes of K or V codes have one token, (d, m) 4
      for (int e = threadIdx.x; e < G * kKv4CellBytes / 2; e += kKv4AppendThreads) {
        const int o = e % (kKv4CellBytes / 2) * 2;
        const int t = o < kKv4VCodes   ? o / 64 + o / 8 % 2 * 8
                      : o < kKv4KMeta ? (o / 8 % 2) * 8 + (o / 16 % 4) * 2 + o / 2 % 2
                                      : o % 64 / 8 + o / 4 % 2 * 8;
        if (tile + t >= t0 && tile + t < t1)
          reinterpret_cast<uint16_t*>(cell0)[e] = reinterpret_cast<const uint16_t*>(image)[e];
      }
    }
    __syncthreads();
  }
  if (!p.summary) return;
  // the warp's tokens, then the warps
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = LR; o < 32; o <<= 1) {
      lo_k[i] = __hmin2(lo_k[i], __shfl_xor_sync(0xffffffffu, lo_k[i], o));
      hi_k[i] = __hmax2(hi_k[i], __shfl_xor_sync(0xffffffffu, hi_k[i], o));
    }
    if (lane < LR) {
      const int dim = 4 * l + (i / 2) * (D / 2) + 2 * (i % 2);
      low[warp][dim] = __low2float(lo_k[i]);
      low[warp][dim + 1] = __high2float(lo_k[i]);
      high[warp][dim] = __low2float(hi_k[i]);
      high[warp][dim + 1] = __high2float(hi_k[i]);
    }
  }
  __syncthreads();
  __nv_bfloat16* sm = p.summary + (static_cast<size_t>(id) * p.hkv + h) * 2 * D;
  for (int i = threadIdx.x; i < D; i += kKv4AppendThreads) {
    float a = INFINITY, z = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a = fminf(a, low[w][i]);
      z = fmaxf(z, high[w][i]);
    }
    if (t0 > 0) {  // the page had tokens before
      a = fminf(a, __bfloat162float(sm[i]));
      z = fmaxf(z, __bfloat162float(sm[D + i]));
    }
    sm[i] = __float2bfloat16_rn(a);
    sm[D + i] = __float2bfloat16_rn(z);
  }
}

template <typename T>
__device__ __forceinline__ void kv4_store8(T* dst, const float (&x)[8]);
template <>
__device__ __forceinline__ void kv4_store8<float>(float* dst, const float (&x)[8]) {
  reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void kv4_store8<__nv_bfloat16>(__nv_bfloat16* dst, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One CTA per (page of a sequence, kv head).  128 threads have a word of K codes each (8 dims of
// a token of the cell), 64 a pair of words of V (8 dims of two tokens), for every cell of the
// page; 8 values are stored at once (rows 16-byte aligned).
constexpr int kKv4GatherThreads = 192;

template <int D, typename T>
__global__ void __launch_bounds__(kKv4GatherThreads) kv4_gather_kernel(const Kv4RowsParams p) {
  constexpr int G = D / kKv4Group;
  __shared__ int job_seq, job_page;
  const int h = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  int b = blockIdx.x, pg = 0;
  if (p.cu) {
    if (threadIdx.x < 32) {
      b = kv4_find_job(p.cu, p.pos, p.rows, p.batch, p.page, blockIdx.x, pg);
      if (threadIdx.x == 0) {
        job_seq = b;
        job_page = pg;
      }
    }
    __syncthreads();
    b = job_seq;
    pg = job_page;
    if (b < 0) return;
  }
  int row0, row1;
  kv4_rows(p.cu, p.rows, b, row0, row1);
  const int pos = p.pos[b];
  if (!p.cu) pg = max(pos, 0) / p.page;
  if (pos == -1 || row1 <= row0) return;
  const int id = pos < 0 ? -1 : kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg);
  if (id < 0) {
    if (threadIdx.x == 0) record_error(kDevBadPosition);
    return;
  }
  const long long base = static_cast<long long>(pg) * p.page;
  const int t0 = static_cast<int>(max(static_cast<long long>(pos), base) - base);
  const int t1 = static_cast<int>(min(static_cast<long long>(pos) + (row1 - row0), base + p.page) - base);
  const int tile0 = t0 / kKv4Tile, n_cells = ((t1 + kKv4Tile - 1) / kKv4Tile - tile0) * G;
  const uint8_t* cells = p.pool + ((static_cast<size_t>(id) * p.hkv + h) * (p.page / kKv4Tile) + tile0) *
                                      static_cast<size_t>(G * kKv4CellBytes);
  const long long to_row = row0 + (base - pos) + tile0 * kKv4Tile;  // of the first tile's first token
  const int lo = t0 - tile0 * kKv4Tile, hi = t1 - tile0 * kKv4Tile;
  auto value = [](uint32_t code, uint32_t dm) {
    return fmaf(static_cast<float>(code & 15u), bf16lo_to_f32(dm), bf16hi_to_f32(dm));
  };
  if (threadIdx.x < 128) {
    const int t = threadIdx.x / 8, c = threadIdx.x % 8;
    T* out = static_cast<T*>(const_cast<void*>(p.k)) + static_cast<size_t>(h) * D + 8 * c;
#pragma unroll 4
    for (int i = 0; i < n_cells; ++i) {
      const uint8_t* cell = cells + static_cast<size_t>(i) * kKv4CellBytes;
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(cell + kv4_k_word(t, c));
      const uint32_t dm = *reinterpret_cast<const uint32_t*>(cell + kKv4KMeta + kv4_meta(t));
      const int at = i / G * kKv4Tile + t;
      if (at < lo || at >= hi) continue;
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = value(bits >> (4 * k), dm);
      kv4_store8<T>(out + (to_row + at) * p.ld_k + 64 * (i % G), x);
    }
  } else {
    const int pr = (threadIdx.x - 128) / 8, c = threadIdx.x % 8;  // tokens 2 pr and 2 pr + 1
    T* out = static_cast<T*>(const_cast<void*>(p.v)) + static_cast<size_t>(h) * D + 8 * c;
#pragma unroll 2
    for (int i = 0; i < n_cells; ++i) {
      const uint8_t* cell = cells + static_cast<size_t>(i) * kKv4CellBytes;
      const uint2 bits = *reinterpret_cast<const uint2*>(cell + kv4_v_half(2 * pr, 2 * c));
      uint32_t dm[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) dm[s] = *reinterpret_cast<const uint32_t*>(cell + kKv4VMeta + kv4_meta(2 * pr + s));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int at = i / G * kKv4Tile + 2 * pr + s;
        if (at < lo || at >= hi) continue;
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = value(bits.x >> (16 * s + 4 * k), dm[s]);
          x[4 + k] = value(bits.y >> (16 * s + 4 * k), dm[s]);
        }
        kv4_store8<T>(out + (to_row + at) * p.ld_v + 64 * (i % G), x);
      }
    }
  }
}

}  // namespace b2
