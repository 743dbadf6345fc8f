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
// them, so the rotation, d and the quotient are evaluated in fp64: the same inputs give the
// same codes whatever the order of evaluation.
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

template <int D>
__global__ void __launch_bounds__(kKv4AppendThreads) kv4_append_kernel(const Kv4RowsParams p,
                                                                      const __grid_constant__ Kv4Rope rope) {
  constexpr int G = D / kKv4Group, J = D / 32, W = kKv4AppendThreads / 32;
  __shared__ __align__(16) uint8_t codes[2][kKv4Tile][D];  // K, V
  __shared__ uint32_t meta[2][G][kKv4Tile];
  __shared__ float low[W][D], high[W][D];
  __shared__ int job_seq, job_page;

  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {
    int pg = 0;
    const int b = kv4_find_job(p.cu, p.pos, p.rows, p.batch, p.page, blockIdx.x, pg);
    if (lane == 0) {
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
  for (int tile = t0 / kKv4Tile; tile * kKv4Tile < t1; ++tile) {
    for (int t = warp; t < kKv4Tile; t += W) {
      const int at = tile * kKv4Tile + t;
      if (at < t0 || at >= t1) continue;
      const long long position = base + at;
      const size_t row = static_cast<size_t>(row0 + (position - pos));
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        double x[J];
        const size_t off = row * (which ? p.ld_v : p.ld_k) + static_cast<size_t>(h) * D + lane;
        const void* src = which ? p.v : p.k;
#pragma unroll
        for (int j = 0; j < J; ++j)
          x[j] = p.is_f32 ? static_cast<const float*>(src)[off + 32 * j]
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(src)[off + 32 * j]);
        if (which == 0 && rope.on) {
#pragma unroll
          for (int j = 0; j < J / 2; ++j) {
            double u = static_cast<double>(position) * rope.turn[lane + 32 * j], sn, cs;
            u -= rint(u);
            sincospi(2.0 * u, &sn, &cs);
            const double a = x[j], c = x[j + J / 2];
            x[j] = a * cs - c * sn;
            x[j + J / 2] = c * cs + a * sn;
          }
        }
        if (which == 0) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const float r = __bfloat162float(__float2bfloat16_rn(static_cast<float>(x[j])));
            lo_k[j] = fminf(lo_k[j], r);
            hi_k[j] = fmaxf(hi_k[j], r);
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          double mn = fmin(x[2 * g], x[2 * g + 1]), mx = fmax(x[2 * g], x[2 * g + 1]);
          // a value that is not finite makes its 64 NaN: 4 bits have no such value
          bool bad = !isfinite(static_cast<float>(x[2 * g])) || !isfinite(static_cast<float>(x[2 * g + 1]));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            mn = fmin(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          }
          bad = __any_sync(0xffffffffu, bad);
          const float m = __bfloat162float(__float2bfloat16_rn(static_cast<float>(mn)));
          const float d = fmaxf(__bfloat162float(__float2bfloat16_rn(static_cast<float>((mx - m) / 15.0))), kKv4MinStep);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const double c = fmin(fmax(floor((x[2 * g + e] - m) / d + 0.5), 0.0), 15.0);
            codes[which][t][64 * g + 32 * e + lane] = bad ? 0 : static_cast<uint8_t>(c);
          }
          if (lane == 0) {
            const uint32_t mb = bad ? 0x7FC0u : (__float_as_uint(m) >> 16);
            meta[which][g][t] = (bad ? __float_as_uint(kKv4MinStep) >> 16 : __float_as_uint(d) >> 16) | (mb << 16);
          }
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
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits |= static_cast<uint32_t>(codes[0][t][64 * g + 8 * x + i]) << (4 * i);
        *reinterpret_cast<uint32_t*>(cell + kv4_k_word(t, x)) = bits;
      } else if (w < 256) {  // half words of V codes: 4 dims of two tokens
        const int pr = (w - 128) / 16, x = (w - 128) % 16;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int t = 2 * pr + s;
          if (!fresh(t)) continue;
          uint32_t bits = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) bits |= static_cast<uint32_t>(codes[1][t][64 * g + 4 * x + i]) << (4 * i);
          *reinterpret_cast<uint16_t*>(cell + kv4_v_half(t, x)) = static_cast<uint16_t>(bits);
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
