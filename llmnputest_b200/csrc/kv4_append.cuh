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
// them, and are to be the same whatever the order of evaluation.  So keys are turned in fp64
// (as fast as integer work here: a complex multiplication a token by the angle of four
// positions, from one sincospi a page), and every choice is made in fp32 with a bound on its
// error; the few that lie within the bound of a border (1 in 10^4 or less) are made again in
// fp64.
//
// One CTA per (page of a sequence, kv head), a warp per token, lanes over the dims; the page's
// summary needs no second pass that way.  Codes go through shared memory into the cell's
// words.  Bound by instruction issue (about 115 a token and head of 64 dims).
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
};

// The least and the largest of a warp's values (sm_100a reduces them in one instruction).
__device__ __forceinline__ float warp_redux_min(float v) {
  float r;
  asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_redux_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// The codes of a warp's 64 values (lane: x0, x1; f0, f1 their fp32 roundings): d and m, by lane
// the two codes.  T is double where the values are not fp32 themselves.
template <typename T>
__device__ __forceinline__ void kv4_quantise(T x0, T x1, float f0, float f1, uint32_t& c0, uint32_t& c1,
                                             uint32_t& meta) {
  const float mn = warp_redux_min(fminf(f0, f1)), mx = warp_redux_max(fmaxf(f0, f1));
  // a value that is not finite makes its 64 NaN: 4 bits have no such value
  if (__any_sync(0xffffffffu, !(fabsf(f0) < INFINITY) || !(fabsf(f1) < INFINITY))) {
    c0 = c1 = 0;
    meta = 0x7FC00000u | (__float_as_uint(kKv4MinStep) >> 16);
    return;
  }
  const float m = round_bf16(mn);  // the rounding is monotone: that of the least x itself
  // (max x - m) / 15: f32 is off by 2^-22 of it, or of max x, at most; where bf16's rounding
  // could see that, in fp64
  float q = (mx - m) * (1.f / 15.f);
  const float slack = (fabsf(mx) + fabsf(m)) * 2.4e-7f;
  if (round_bf16(q - slack) != round_bf16(q + slack)) {
    double top = fmax(static_cast<double>(x0), static_cast<double>(x1));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    q = static_cast<float>((top - m) / 15.0);
  }
  const float d = fmaxf(round_bf16(q), kKv4MinStep), inv = __frcp_rn(d);
  // (x - m) / d + 1/2 is off by `tol` at most: 2^-21 of what enters it
  const float tol = fmaf((fmaxf(fabsf(mx), fabsf(mn)) + fabsf(m)) * inv, 4.8e-7f, 1e-5f);
  auto code = [&](T x, float f) -> uint32_t {
    const float y = fmaf(f - m, inv, 0.5f);
    const float lo = fminf(fmaxf(floorf(y - tol), 0.f), 15.f), hi = fminf(fmaxf(floorf(y + tol), 0.f), 15.f);
    if (lo == hi) return static_cast<uint32_t>(lo);
    return static_cast<uint32_t>(fmin(fmax(floor((static_cast<double>(x) - m) / d + 0.5), 0.0), 15.0));
  };
  c0 = code(x0, f0);
  c1 = code(x1, f1);
  meta = (__float_as_uint(d) >> 16) | (__float_as_uint(m) & 0xFFFF0000u);
}

// Four codes in four bytes as 16 bits of nibbles.
__device__ __forceinline__ uint32_t kv4_nibbles(uint32_t bytes) {
  const uint32_t y = (bytes | bytes >> 4) & 0x00FF00FFu;
  return (y | y >> 8) & 0xFFFFu;
}

template <int D>
__global__ void __launch_bounds__(kKv4AppendThreads) kv4_append_kernel(const Kv4RowsParams p,
                                                                      const __grid_constant__ Kv4Rope rope) {
  constexpr int G = D / kKv4Group, J = D / 32, W = kKv4AppendThreads / 32, T = kKv4Tile / W;
  __shared__ __align__(16) uint8_t codes[2][kKv4Tile][D];  // K, V
  __shared__ uint32_t meta[2][G][kKv4Tile];
  __shared__ float low[W][D], high[W][D];
  __shared__ int job_seq, job_page;

  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  uint8_t* cells = p.pool + (static_cast<size_t>(id) * p.hkv + h) * (static_cast<size_t>(p.page / kKv4Tile) * G * kKv4CellBytes);

  float lo_k[J], hi_k[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    lo_k[j] = INFINITY;
    hi_k[j] = -INFINITY;
  }
  // the turn of this warp's first token, and that of the W positions to its next one
  const int tile0 = t0 / kKv4Tile;
  double cs[J / 2], sn[J / 2], cs_w[J / 2], sn_w[J / 2];
  if (rope.on) {
    const bool several = t1 - t0 > 1;
    const double first = static_cast<double>(several ? base + tile0 * kKv4Tile + warp : base + t0);
#pragma unroll
    for (int j = 0; j < J / 2; ++j) {
      const double turn = kv4_turn(rope, lane + 32 * j);
      double u = first * turn;
      u -= rint(u);
      sincospi(2.0 * u, &sn[j], &cs[j]);
      cs_w[j] = 1.0;
      sn_w[j] = 0.0;
      if (several) {
        u = W * turn;
        u -= rint(u);
        sincospi(2.0 * u, &sn_w[j], &cs_w[j]);
      }
    }
  }
  for (int tile = tile0; tile * kKv4Tile < t1; ++tile) {
    float in[T][2][J];
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int at = tile * kKv4Tile + warp + i * W;
      if (at < t0 || at >= t1) continue;
      const size_t row = static_cast<size_t>(row0 + (base + at - pos));
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const size_t off = row * (which ? p.ld_v : p.ld_k) + static_cast<size_t>(h) * D + lane;
        const void* src = which ? p.v : p.k;
#pragma unroll
        for (int j = 0; j < J; ++j)
          in[i][which][j] = p.is_f32 ? static_cast<const float*>(src)[off + 32 * j]
                                     : __bfloat162float(static_cast<const __nv_bfloat16*>(src)[off + 32 * j]);
      }
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int t = warp + i * W, at = tile * kKv4Tile + t;
      if (at >= t0 && at < t1) {  // uniform in the warp
        double x[J];
        float f[J];
        if (rope.on) {
#pragma unroll
          for (int j = 0; j < J / 2; ++j) {
            const double a = in[i][0][j], c = in[i][0][j + J / 2];
            x[j] = a * cs[j] - c * sn[j];
            x[j + J / 2] = c * cs[j] + a * sn[j];
          }
#pragma unroll
          for (int j = 0; j < J; ++j) f[j] = static_cast<float>(x[j]);
        } else {
#pragma unroll
          for (int j = 0; j < J; ++j) f[j] = in[i][0][j];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float r = round_bf16(f[j]);
          lo_k[j] = fminf(lo_k[j], r);
          hi_k[j] = fmaxf(hi_k[j], r);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t c0, c1, dm;
          if (rope.on) kv4_quantise<double>(x[2 * g], x[2 * g + 1], f[2 * g], f[2 * g + 1], c0, c1, dm);
          else kv4_quantise<float>(f[2 * g], f[2 * g + 1], f[2 * g], f[2 * g + 1], c0, c1, dm);
          codes[0][t][64 * g + lane] = static_cast<uint8_t>(c0);
          codes[0][t][64 * g + 32 + lane] = static_cast<uint8_t>(c1);
          if (lane == 0) meta[0][g][t] = dm;
          const float v0 = in[i][1][2 * g], v1 = in[i][1][2 * g + 1];
          kv4_quantise<float>(v0, v1, v0, v1, c0, c1, dm);
          codes[1][t][64 * g + lane] = static_cast<uint8_t>(c0);
          codes[1][t][64 * g + 32 + lane] = static_cast<uint8_t>(c1);
          if (lane == 0) meta[1][g][t] = dm;
        }
      }
      if (rope.on) {
#pragma unroll
        for (int j = 0; j < J / 2; ++j) {
          const double c = cs[j];
          cs[j] = c * cs_w[j] - sn[j] * sn_w[j];
          sn[j] = sn[j] * cs_w[j] + c * sn_w[j];
        }
      }
    }
    __syncthreads();
    uint8_t* cell0 = cells + static_cast<size_t>(tile) * G * kKv4CellBytes;
    const int base_t = tile * kKv4Tile;
    auto fresh = [&](int t) { return base_t + t >= t0 && base_t + t < t1; };
    for (int e = threadIdx.x; e < G * 288; e += kKv4AppendThreads) {
      const int g = e / 288, w = e % 288;
      uint8_t* cell = cell0 + g * kKv4CellBytes;
      if (w < 128) {  // a word of K codes: 8 dims of one token
        const int t = w / 8, x = w % 8;
        if (!fresh(t)) continue;
        const uint2 bytes = *reinterpret_cast<const uint2*>(&codes[0][t][64 * g + 8 * x]);
        *reinterpret_cast<uint32_t*>(cell + kv4_k_word(t, x)) = kv4_nibbles(bytes.x) | kv4_nibbles(bytes.y) << 16;
      } else if (w < 256) {  // a word of V codes: 4 dims of two tokens
        const int pr = (w - 128) / 16, x = (w - 128) % 16, t = 2 * pr;
        const uint32_t a = kv4_nibbles(*reinterpret_cast<const uint32_t*>(&codes[1][t][64 * g + 4 * x]));
        const uint32_t z = kv4_nibbles(*reinterpret_cast<const uint32_t*>(&codes[1][t + 1][64 * g + 4 * x]));
        uint16_t* to = reinterpret_cast<uint16_t*>(cell + kv4_v_half(t, x));
        if (fresh(t) && fresh(t + 1)) {
          *reinterpret_cast<uint32_t*>(to) = a | z << 16;
        } else {
          if (fresh(t)) to[0] = static_cast<uint16_t>(a);
          if (fresh(t + 1)) to[1] = static_cast<uint16_t>(z);
        }
      } else {
        const int which = (w - 256) / 16, t = (w - 256) % 16;
        if (fresh(t))
          *reinterpret_cast<uint32_t*>(cell + (which ? kKv4VMeta : kKv4KMeta) + kv4_meta(t)) = meta[which][g][t];
      }
    }
    __syncthreads();
  }
  if (!p.summary) return;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    low[warp][lane + 32 * j] = lo_k[j];
    high[warp][lane + 32 * j] = hi_k[j];
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

// One CTA per (page of a sequence, kv head); a thread decodes 8 dims of one token of K and
// of two tokens of V at a time and stores 8 values at once (rows 16-byte aligned).
template <int D, typename T>
__global__ void __launch_bounds__(kKv4AppendThreads) kv4_gather_kernel(const Kv4RowsParams p) {
  constexpr int G = D / kKv4Group;
  __shared__ int job_seq, job_page;
  const int h = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < 32) {
    int pg = 0;
    const int b = kv4_find_job(p.cu, p.pos, p.rows, p.batch, p.page, blockIdx.x, pg);
    if (threadIdx.x == 0) {
      job_seq = b;
      job_page = pg;
    }
  }
  __syncthreads();
  const int b = job_seq, pg = job_page;
  if (b < 0) return;
  int row0, row1;
  kv4_rows(p.cu, p.rows, b, row0, row1);
  const int pos = p.pos[b];
  if (pos == -1 || row1 <= row0) return;
  const int id = pos < 0 ? -1 : kv4_page_id(p.table, p.max_pages, p.n_pages, b, pg);
  if (id < 0) {
    if (threadIdx.x == 0) record_error(kDevBadPosition);
    return;
  }
  const long long base = static_cast<long long>(pg) * p.page;
  const int t0 = static_cast<int>(max(static_cast<long long>(pos), base) - base);
  const int t1 = static_cast<int>(min(static_cast<long long>(pos) + (row1 - row0), base + p.page) - base);
  const uint8_t* cells = p.pool + (static_cast<size_t>(id) * p.hkv + h) * (static_cast<size_t>(p.page / kKv4Tile) * G * kKv4CellBytes);
  T* kout = static_cast<T*>(const_cast<void*>(p.k));
  T* vout = static_cast<T*>(const_cast<void*>(p.v));
  const long long to_row = row0 + (base - pos);
  const int tile0 = t0 / kKv4Tile, tiles = (t1 + kKv4Tile - 1) / kKv4Tile - tile0;
  // per cell: 16 x 8 words of K, then 8 x 8 word pairs of V
  for (int e = threadIdx.x; e < tiles * G * 192; e += kKv4AppendThreads) {
    const int w = e % 192, g = e / 192 % G, tile = tile0 + e / (192 * G);
    const uint8_t* cell = cells + (static_cast<size_t>(tile) * G + g) * kKv4CellBytes;
    float x[8];
    if (w < 128) {
      const int t = w / 8, c = w % 8, at = tile * kKv4Tile + t;
      if (at < t0 || at >= t1) continue;
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(cell + kv4_k_word(t, c));
      const uint32_t dm = *reinterpret_cast<const uint32_t*>(cell + kKv4KMeta + kv4_meta(t));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((bits >> (4 * i)) & 15u), bf16lo_to_f32(dm), bf16hi_to_f32(dm));
      kv4_store8<T>(kout + (to_row + at) * p.ld_k + static_cast<size_t>(h) * D + 64 * g + 8 * c, x);
    } else {
      const int pr = (w - 128) / 8, c = (w - 128) % 8;  // tokens 2 pr and 2 pr + 1, dims 8 c ..
      const uint2 bits = *reinterpret_cast<const uint2*>(cell + kv4_v_half(2 * pr, 2 * c));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int t = 2 * pr + s, at = tile * kKv4Tile + t;
        if (at < t0 || at >= t1) continue;
        const uint32_t dm = *reinterpret_cast<const uint32_t*>(cell + kKv4VMeta + kv4_meta(t));
        const uint32_t q0 = bits.x >> (16 * s), q1 = bits.y >> (16 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = fmaf(static_cast<float>((q0 >> (4 * i)) & 15u), bf16lo_to_f32(dm), bf16hi_to_f32(dm));
          x[4 + i] = fmaf(static_cast<float>((q1 >> (4 * i)) & 15u), bf16lo_to_f32(dm), bf16hi_to_f32(dm));
        }
        kv4_store8<T>(vout + (to_row + at) * p.ld_v + static_cast<size_t>(h) * D + 64 * g + 8 * c, x);
      }
    }
  }
}

}  // namespace b2
