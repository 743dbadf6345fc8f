// C entry points of the 4-bit paged KV cache (b2_kv4_*): argument checks, launch plans.
// Part of the library's one translation unit; uses its device_info, fail and cuda_fail.
#pragma once

#include <atomic>
#include <cmath>

#include "kv4_append.cuh"
#include "kv4_decode.cuh"
#include "kv4_pages.cuh"
#include "kv4_select.cuh"

namespace {

constexpr int kKv4MaxSelectPages = 16384;  // 12 bytes of shared memory each: 192 KB

struct Kv4Shape {
  int batch, hkv, head_dim, page, max_pages, n_pages;
};

int kv4_check(const Kv4Shape& s) {
  if (s.head_dim != 64 && s.head_dim != 128 && s.head_dim != 256)
    return fail(B2_ERR_ARG, "head_dim %d: 64, 128 and 256 are built", s.head_dim);
  if (s.batch < 1 || s.batch > 65535) return fail(B2_ERR_ARG, "batch %d outside 1..65535", s.batch);
  if (s.hkv < 1 || s.hkv > 65535) return fail(B2_ERR_ARG, "n_kv_heads %d outside 1..65535", s.hkv);
  if (s.page < 16 || s.page % 16 || s.page > 4096)
    return fail(B2_ERR_ARG, "page %d: a multiple of 16, at most 4096, is needed", s.page);
  if (s.max_pages < 1 || s.n_pages < 1) return fail(B2_ERR_ARG, "empty page table or pool");
  if (static_cast<long long>(s.max_pages) * s.page > (1LL << 30))
    return fail(B2_ERR_ARG, "a page table over more than 2^30 tokens");
  return B2_OK;
}

int kv4_heads(int hq, int hkv) {
  if (hq < 1 || hq % hkv) return fail(B2_ERR_ARG, "bad head counts hq=%d hkv=%d", hq, hkv);
  if (hq / hkv > b2::kKv4MaxGroup) return fail(B2_ERR_ARG, "GQA group %d > 8 is not supported", hq / hkv);
  return B2_OK;
}

// the angles' table of (theta, head_dim), made once per thread for calls with the same two
const b2::Kv4Rope& kv4_rope(float theta, int head_dim, int flags) {
  static thread_local b2::Kv4Rope off = {}, on = {};
  static thread_local float on_theta = 0.f;
  static thread_local int on_dim = 0;
  if (flags & B2_KV4_NO_ROPE) return off;
  if (on_theta != theta || on_dim != head_dim) {
    for (int i = 0; i < head_dim / 2; ++i)
      on.turn[i] = std::pow(static_cast<double>(theta), -2.0 * i / head_dim) / 6.283185307179586476925287;
    on.on = 1;
    on_theta = theta;
    on_dim = head_dim;
  }
  return on;
}

struct Kv4Launch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  Kv4Launch(dim3 grid, int threads, void* stream, size_t smem = 0) {
    if (pdl_for(kPdlOther)) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
  }
  void cluster(int n) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = n;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
};

// head_dim as a template argument
template <typename F>
auto kv4_by_dim(int head_dim, F f) {
  return head_dim == 64    ? f(std::integral_constant<int, 64>())
         : head_dim == 128 ? f(std::integral_constant<int, 128>())
                           : f(std::integral_constant<int, 256>());
}

constexpr int kKv4DecodeWarps = 4;

struct Kv4DecodePlan {
  int tiles, splits, ctas;  // splits 0: tiles dealt over ctas
  size_t span_bytes, ws_bytes;
};

// A cluster per (sequence, kv head) while the clusters fit the GPU at once and no warp has more
// than 16 tiles (one sequence, 8 kv heads of 64: 11.3 us against 13.6 dealt at 16384 tokens,
// but two of 32768 22.4 against 18.5, and one of 32768 with 128 dims 27.8 against 20.9); else the tiles
// are dealt over as many CTAs as the GPU holds, each with two per warp at least.
Kv4DecodePlan kv4_decode_plan(int batch, int hq, int hkv, int head_dim, int tokens, int sms) {
  Kv4DecodePlan pl = {};
  constexpr int W = kKv4DecodeWarps;
  pl.tiles = (tokens + 15) / 16;
  const long long pairs = static_cast<long long>(batch) * hkv, slots = (head_dim == 256 ? 2LL : 4LL) * sms;
  const int s = std::min(16, (pl.tiles + W - 1) / W);
  if (pairs * s <= slots && pl.tiles <= 16 * W * s) {
    pl.splits = s;
    return pl;
  }
  // a whole number of CTAs a pair, or of pairs a CTA, where that leaves few slots empty: equal
  // lengths are then not cut (64 sequences x 8 kv heads of 4096 tokens: 39.4 us with 512 CTAs,
  // 46 with all 592)
  long long n = slots;
  if (pairs <= slots) {
    if (slots / pairs * pairs * 10 >= slots * 8) n = slots / pairs * pairs;
  } else {
    const long long c = (pairs + slots - 1) / slots;
    if ((pairs + c - 1) / c * 10 >= slots * 9) n = (pairs + c - 1) / c;
  }
  pl.ctas = static_cast<int>(std::min(n, (pairs * pl.tiles + 2 * W - 1) / (2 * W)));
  pl.span_bytes = (static_cast<size_t>(pairs) * 8 + 15) / 16 * 16;
  pl.ws_bytes = pl.span_bytes + static_cast<size_t>(pl.ctas) * 2 * b2::kv4_part_floats(hq / hkv, head_dim) * sizeof(float);
  return pl;
}

// tokens that a call's splits cover: those of the selected pages, or max_len
int kv4_decode_tokens(int n_sel, int page, int max_len) {
  return n_sel > 0 ? n_sel * page : max_len;
}

}  // namespace

extern "C" {

static int kv4_rows_call(bool append, const void* k, const void* v, int64_t ld_k, int64_t ld_v, int rows, void* pool,
                         const int32_t* table, const int32_t* pos, const int32_t* cu, uint16_t* summary,
                         const Kv4Shape& s, float theta, int flags, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  st = kv4_check(s);
  if (st != B2_OK) return st;
  if (!pool || !table || !pos) return fail(B2_ERR_ARG, "null pointer argument");
  if (flags & ~(append ? B2_KV4_NO_ROPE | B2_KV4_ROWS_F32 : B2_KV4_ROWS_F32)) return fail(B2_ERR_ARG, "unknown flags 0x%x", flags);
  if (rows < 0) return fail(B2_ERR_ARG, "negative row count");
  if (!cu && rows != s.batch) return fail(B2_ERR_ARG, "%d rows for %d sequences: row offsets are needed", rows, s.batch);
  if (append && !(flags & B2_KV4_NO_ROPE) && !(theta > 0.f)) return fail(B2_ERR_ARG, "theta must be > 0");
  if (rows == 0) return B2_OK;
  if (!k || !v) return fail(B2_ERR_ARG, "null pointer argument");
  const int64_t width = static_cast<int64_t>(s.hkv) * s.head_dim;
  if (rows > 1 && (ld_k < width || ld_v < width)) return fail(B2_ERR_ARG, "row stride below n_kv_heads * head_dim");
  if (!aligned(pool, 16)) return fail(B2_ERR_ALIGN, "the pool must be 16-byte aligned");
  const int f32 = (flags & B2_KV4_ROWS_F32) ? 1 : 0;
  if (!append) {  // rows stored 16 bytes at a time
    const int64_t per = f32 ? 4 : 8;
    if (!aligned(k, 16) || !aligned(v, 16) || (rows > 1 && (ld_k % per || ld_v % per)))
      return fail(B2_ERR_ALIGN, "gathered rows must be 16-byte aligned");
  }
  b2::Kv4RowsParams p = {};
  p.k = k;
  p.v = v;
  p.ld_k = ld_k;
  p.ld_v = ld_v;
  p.pool = static_cast<uint8_t*>(pool);
  p.table = table;
  p.pos = pos;
  p.cu = cu;
  p.summary = reinterpret_cast<__nv_bfloat16*>(summary);
  p.rows = rows;
  p.batch = s.batch;
  p.hkv = s.hkv;
  p.page = s.page;
  p.max_pages = s.max_pages;
  p.n_pages = s.n_pages;
  p.is_f32 = f32;
  const int64_t quad = f32 ? 16 : 8;
  p.wide = aligned(k, quad) && aligned(v, quad) && ld_k % 4 == 0 && ld_v % 4 == 0;
  // a sequence of n rows touches at most n / page + 2 pages
  const int jobs = cu ? rows / s.page + 2 * s.batch : s.batch;
  Kv4Launch l(dim3(jobs, s.hkv, 1), append ? b2::kKv4AppendThreads : b2::kKv4GatherThreads, stream);
  const b2::Kv4Rope& rope = kv4_rope(theta, s.head_dim, append ? flags : B2_KV4_NO_ROPE);
  const cudaError_t e = kv4_by_dim(s.head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (append) return cudaLaunchKernelEx(&l.cfg, b2::kv4_append_kernel<D>, p, rope);
    return f32 ? cudaLaunchKernelEx(&l.cfg, b2::kv4_gather_kernel<D, float>, p)
               : cudaLaunchKernelEx(&l.cfg, b2::kv4_gather_kernel<D, __nv_bfloat16>, p);
  });
  if (e != cudaSuccess) return cuda_fail(e, append ? "kv4 append launch" : "kv4 gather launch");
  return B2_OK;
}

int b2_kv4_append(const void* k, const void* v, int64_t ld_k, int64_t ld_v, int rows, uint8_t* pool,
                  const int32_t* table, const int32_t* pos, const int32_t* cu, uint16_t* summary, int batch,
                  int n_kv_heads, int head_dim, int page, int max_pages, int n_pages, float theta, int flags,
                  void* stream) {
  return kv4_rows_call(true, k, v, ld_k, ld_v, rows, pool, table, pos, cu, summary,
                       {batch, n_kv_heads, head_dim, page, max_pages, n_pages}, theta, flags, stream);
}

int b2_kv4_gather(void* k, void* v, int64_t ld_k, int64_t ld_v, int rows, const uint8_t* pool, const int32_t* table,
                  const int32_t* pos, const int32_t* cu, int batch, int n_kv_heads, int head_dim, int page,
                  int max_pages, int n_pages, int flags, void* stream) {
  return kv4_rows_call(false, k, v, ld_k, ld_v, rows, const_cast<uint8_t*>(pool), table, pos, cu, nullptr,
                       {batch, n_kv_heads, head_dim, page, max_pages, n_pages}, 0.f, flags, stream);
}

static int kv4_decode_check(const Kv4Shape& s, int hq, int n_sel, int max_len) {
  int st = kv4_check(s);
  if (st != B2_OK) return st;
  st = kv4_heads(hq, s.hkv);
  if (st != B2_OK) return st;
  if (n_sel < 0 || static_cast<long long>(n_sel) * s.page > (1LL << 30))
    return fail(B2_ERR_ARG, "n_sel %d: 0 or more, over 2^30 tokens at most", n_sel);
  if (max_len < 1 || max_len > static_cast<long long>(s.max_pages) * s.page)
    return fail(B2_ERR_ARG, "max_len %d outside 1..max_pages * page", max_len);
  return B2_OK;
}

int b2_kv4_decode_workspace_size(int batch, int n_q_heads, int n_kv_heads, int head_dim, int page, int n_sel,
                                 int max_len, size_t* bytes) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  if (!bytes) return fail(B2_ERR_ARG, "null bytes pointer");
  if (max_len < 1 || page < 1 || n_sel < 0) return fail(B2_ERR_ARG, "bad lengths");
  st = kv4_decode_check({batch, n_kv_heads, head_dim, page, (max_len - 1) / page + 1, 1}, n_q_heads,
                        n_sel, max_len);
  if (st != B2_OK) return st;
  *bytes = kv4_decode_plan(batch, n_q_heads, n_kv_heads, head_dim, kv4_decode_tokens(n_sel, page, max_len), di.sms).ws_bytes;
  return B2_OK;
}

int b2_kv4_decode(const float* q, int64_t ld_q, const uint8_t* pool, const int32_t* table, const int32_t* pos,
                  const int32_t* sel, int n_sel, int batch, int n_q_heads, int n_kv_heads, int head_dim, int page,
                  int max_pages, int n_pages, int max_len, float theta, float scale, void* out, int64_t ldo,
                  void* workspace, size_t workspace_bytes, int flags, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  if ((sel == nullptr) != (n_sel == 0)) return fail(B2_ERR_ARG, "sel and n_sel go together");
  st = kv4_decode_check({batch, n_kv_heads, head_dim, page, max_pages, n_pages}, n_q_heads, n_sel, max_len);
  if (st != B2_OK) return st;
  if (!q || !pool || !table || !pos || !out) return fail(B2_ERR_ARG, "null pointer argument");
  if (flags & ~(B2_KV4_NO_ROPE | B2_KV4_OUT_F32)) return fail(B2_ERR_ARG, "unknown flags 0x%x", flags);
  if (!(flags & B2_KV4_NO_ROPE) && !(theta > 0.f)) return fail(B2_ERR_ARG, "theta must be > 0");
  const int64_t width = static_cast<int64_t>(n_q_heads) * head_dim;
  if (batch > 1 && (ld_q < width || ldo < width)) return fail(B2_ERR_ARG, "row stride below n_q_heads * head_dim");
  if (!aligned(pool, 16)) return fail(B2_ERR_ALIGN, "the pool must be 16-byte aligned");
  const Kv4DecodePlan pl =
      kv4_decode_plan(batch, n_q_heads, n_kv_heads, head_dim, kv4_decode_tokens(n_sel, page, max_len), di.sms);
  if (pl.ws_bytes && (!workspace || workspace_bytes < pl.ws_bytes || !aligned(workspace, 16)))
    return fail(B2_ERR_WORKSPACE, "kv4 decode needs %zu bytes of 16-byte aligned workspace", pl.ws_bytes);
  if ((pl.tiles + static_cast<long long>(b2::kKv4RunOverhead)) * n_kv_heads > (1LL << 30)) return fail(B2_ERR_ARG, "a sequence of over 2^34 tokens x kv heads");
  b2::Kv4DecodeParams p = {};
  p.q = q;
  p.ld_q = ld_q;
  p.pool = pool;
  p.table = table;
  p.pos = pos;
  p.sel = sel;
  p.out = out;
  p.ldo = ldo;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.batch = batch;
  p.hq = n_q_heads;
  p.hkv = n_kv_heads;
  p.page = page;
  p.max_pages = max_pages;
  p.n_pages = n_pages;
  p.n_sel = n_sel;
  p.splits = pl.splits;
  p.max_len = max_len;
  p.out_f32 = (flags & B2_KV4_OUT_F32) ? 1 : 0;
  const b2::Kv4Rope& rope = kv4_rope(theta, head_dim, flags);
  cudaError_t e = kv4_by_dim(head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    auto kernel = b2::kv4_decode_kernel<D, kKv4DecodeWarps>;
    constexpr size_t smem = b2::kv4_decode_smem<D, kKv4DecodeWarps>();
    static std::atomic<unsigned long long> ready{0};  // devices on which the kernel's attributes are set
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(ready.load() >> dev & 1)) {
      cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (r == cudaSuccess) r = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (r != cudaSuccess) return r;
      ready.fetch_or(1ull << dev);
    }
    if (pl.splits) {
      Kv4Launch l(dim3(pl.splits * n_kv_heads, batch, 1), kKv4DecodeWarps * 32, stream, smem);
      l.cluster(pl.splits);
      return cudaLaunchKernelEx(&l.cfg, kernel, p, rope);
    }
    // dealt over the grid, a slice of the batch at a time: the weights of a slice fit 32 bits
    const int slice = static_cast<int>(std::min<long long>(b2::kKv4MaxDealt, (1LL << 30) / ((pl.tiles + static_cast<long long>(b2::kKv4RunOverhead)) * n_kv_heads)));
    for (int b0 = 0; b0 < batch; b0 += slice) {
      b2::Kv4DecodeParams part = p;
      part.batch = std::min(slice, batch - b0);
      part.q = q + b0 * ld_q;
      part.table = table + static_cast<size_t>(b0) * max_pages;
      part.pos = pos + b0;
      if (sel) part.sel = sel + static_cast<size_t>(b0) * n_kv_heads * n_sel;
      part.out = static_cast<char*>(out) + b0 * ldo * (p.out_f32 ? 4 : 2);
      part.spans = static_cast<int2*>(workspace);
      part.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.span_bytes);
      Kv4Launch l(dim3(pl.ctas, 1, 1), kKv4DecodeWarps * 32, stream, smem);
      cudaError_t r = cudaLaunchKernelEx(&l.cfg, kernel, part, rope);
      if (r != cudaSuccess) return r;
      // few pairs with many parts each: a CTA per head, up to 16 threads to an output's parts (8
      // sequences x 8 kv heads of 8192: 19.0 us against 21.7 with a CTA per kv head, but 16 of
      // 4096, with 4.6 parts a pair, 20.5 against 17.7)
      const int grp = n_q_heads / n_kv_heads;
      const bool few = pl.ctas > 8 * part.batch * n_kv_heads;
      Kv4Launch j(dim3(n_kv_heads, part.batch, few ? grp : 1), few ? std::min(4 * D, b2::kKv4JoinMost) : grp * D / 4, stream);
      r = cudaLaunchKernelEx(&j.cfg, b2::kv4_join_kernel<D>, part);
      if (r != cudaSuccess) return r;
    }
    return cudaSuccess;
  });
  if (e != cudaSuccess) return cuda_fail(e, "kv4 decode launch");
  return B2_OK;
}

static int kv4_select_check(int page, int n_sel, int max_len, int* key_pages) {
  if (page < 1 || max_len < 1) return fail(B2_ERR_ARG, "bad lengths");
  *key_pages = (max_len - 1) / page + 1;
  if (n_sel < 1) return fail(B2_ERR_ARG, "n_sel must be >= 1");
  if (*key_pages > kKv4MaxSelectPages)
    return fail(B2_ERR_ARG, "selection among %d pages: at most %d", *key_pages, kKv4MaxSelectPages);
  return B2_OK;
}

int b2_kv4_select(const float* q, int64_t ld_q, const uint16_t* summary, const int32_t* table, const int32_t* pos,
                  int32_t* sel, int n_sel, int batch, int n_q_heads, int n_kv_heads, int head_dim, int page,
                  int max_pages, int n_pages, int max_len, float theta, int flags, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  st = kv4_decode_check({batch, n_kv_heads, head_dim, page, max_pages, n_pages}, n_q_heads, 0, max_len);
  if (st != B2_OK) return st;
  int pages = 0;
  st = kv4_select_check(page, n_sel, max_len, &pages);
  if (st != B2_OK) return st;
  if (!q || !summary || !table || !pos || !sel) return fail(B2_ERR_ARG, "null pointer argument");
  if (flags & ~B2_KV4_NO_ROPE) return fail(B2_ERR_ARG, "unknown flags 0x%x", flags);
  if (!(flags & B2_KV4_NO_ROPE) && !(theta > 0.f)) return fail(B2_ERR_ARG, "theta must be > 0");
  if (batch > 1 && ld_q < static_cast<int64_t>(n_q_heads) * head_dim)
    return fail(B2_ERR_ARG, "row stride below n_q_heads * head_dim");
  if (!aligned(summary, 16)) return fail(B2_ERR_ALIGN, "the summaries must be 16-byte aligned");
  b2::Kv4SelectParams p = {};
  p.q = q;
  p.ld_q = ld_q;
  p.summary = reinterpret_cast<const __nv_bfloat16*>(summary);
  p.table = table;
  p.pos = pos;
  p.sel = sel;
  p.batch = batch;
  p.hq = n_q_heads;
  p.hkv = n_kv_heads;
  p.page = page;
  p.max_pages = max_pages;
  p.n_pages = n_pages;
  p.n_sel = n_sel;
  p.max_len = max_len;
  p.key_pages = pages;
  const b2::Kv4Rope& rope = kv4_rope(theta, head_dim, flags);
  // CTAs of a cluster: one per group of pages that its warps take at once, up to 8, and no more
  // than the GPU holds in all, two per SM (16 sequences x 8 kv heads of up to 1024 pages: 13.9 us
  // so, 19.8 at four per SM, 26.7 in clusters of 8)
  const int group = b2::kKv4SelectThreads / 32 * 16;
  const long long pairs = static_cast<long long>(batch) * n_kv_heads;
  p.ctas = static_cast<int>(std::max(1LL, std::min({8LL, static_cast<long long>((pages + group - 1) / group), 2LL * di.sms / pairs})));
  const size_t smem = static_cast<size_t>(pages) * 12;
  const cudaError_t e = kv4_by_dim(head_dim, [&](auto d) {
    auto kernel = b2::kv4_select_kernel<decltype(d)::value>;
    static std::atomic<unsigned long long> ready{0};  // devices on which the kernel's attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(ready.load() >> dev & 1)) {
      const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kKv4MaxSelectPages * 12);
      if (r != cudaSuccess) return r;
      ready.fetch_or(1ull << dev);
    }
    Kv4Launch l(dim3(p.ctas * n_kv_heads, batch, 1), b2::kKv4SelectThreads, stream, smem);
    l.cluster(p.ctas);
    return cudaLaunchKernelEx(&l.cfg, kernel, p, rope);
  });
  if (e != cudaSuccess) return cuda_fail(e, "kv4 select launch");
  return B2_OK;
}

static int kv4_page_data(uint8_t* pool, int64_t page_bytes, uint8_t* summary, int64_t summary_bytes, int layers,
                         int n_pages, b2::Kv4PageData* d) {
  if (!pool) return fail(B2_ERR_ARG, "null pool");
  if (layers < 1 || layers > 65535 || n_pages < 1) return fail(B2_ERR_ARG, "bad pool: %d layers of %d pages", layers, n_pages);
  if (page_bytes < 16 || page_bytes % 16 || (summary && (summary_bytes < 16 || summary_bytes % 16)))
    return fail(B2_ERR_ARG, "the bytes of a page must be a multiple of 16");
  if (!aligned(pool, 16) || !aligned(summary, 16)) return fail(B2_ERR_ALIGN, "pool and summaries must be 16-byte aligned");
  d->base[0] = pool;
  d->bytes[0] = static_cast<unsigned long long>(page_bytes);
  d->base[1] = summary;
  d->bytes[1] = summary ? static_cast<unsigned long long>(summary_bytes) : 0;
  d->layers = layers;
  d->n_pages = n_pages;
  return B2_OK;
}

// CTAs that share one page's bytes: each thread about four 16-byte pieces
static int kv4_copy_parts(const b2::Kv4PageData& d) {
  return static_cast<int>(std::min<unsigned long long>(64, (d.bytes[0] + d.bytes[1] + 16383) / 16384));
}

int b2_kv4_copy_pages(uint8_t* pool, int64_t page_bytes, uint8_t* summary, int64_t summary_bytes, int layers,
                      int n_pages, const int32_t* src, const int32_t* dst, int n, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  b2::Kv4PageData d;
  st = kv4_page_data(pool, page_bytes, summary, summary_bytes, layers, n_pages, &d);
  if (st != B2_OK) return st;
  if (n < 0 || n > 65535) return fail(B2_ERR_ARG, "%d copies: 0..65535", n);
  if (n == 0) return B2_OK;
  if (!src || !dst) return fail(B2_ERR_ARG, "null pointer argument");
  Kv4Launch l(dim3(kv4_copy_parts(d), layers, n), b2::kKv4CopyThreads, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, b2::kv4_copy_kernel, d, static_cast<const int*>(src), static_cast<const int*>(dst));
  if (e != cudaSuccess) return cuda_fail(e, "kv4 copy launch");
  return B2_OK;
}

// need, copy, the number of free pages found, then those
static size_t kv4_reorder_ws(int batch, int max_pages, int n_pages) {
  const size_t ids = std::min(static_cast<size_t>(batch) * max_pages, static_cast<size_t>(n_pages));
  return (2 * static_cast<size_t>(batch) + 1 + ids) * sizeof(int);
}

int b2_kv4_reorder_workspace_size(int batch, int max_pages, int n_pages, size_t* bytes) {
  if (!bytes) return fail(B2_ERR_ARG, "null bytes pointer");
  if (batch < 1 || max_pages < 1 || n_pages < 1) return fail(B2_ERR_ARG, "empty page table or pool");
  *bytes = kv4_reorder_ws(batch, max_pages, n_pages);
  return B2_OK;
}

int b2_kv4_reorder(uint8_t* pool, int64_t page_bytes, uint8_t* summary, int64_t summary_bytes, int layers, int n_pages,
                   const int32_t* table, const int32_t* lens, const int32_t* refs, const int32_t* parent,
                   const int32_t* reserve, int batch, int max_pages, int page, int32_t* table_out, int32_t* lens_out,
                   int32_t* refs_out, int32_t* info, void* workspace, size_t workspace_bytes, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  b2::Kv4ReorderParams p = {};
  st = kv4_page_data(pool, page_bytes, summary, summary_bytes, layers, n_pages, &p.data);
  if (st != B2_OK) return st;
  if (batch < 1 || batch > 65535 || max_pages < 1 || page < 1) return fail(B2_ERR_ARG, "bad page table shape");
  if (!table || !lens || !refs || !parent || !table_out || !lens_out || !refs_out || !info)
    return fail(B2_ERR_ARG, "null pointer argument");
  if (table == table_out || lens == lens_out || refs == refs_out)
    return fail(B2_ERR_ARG, "the new rows need buffers of their own");
  const size_t need = kv4_reorder_ws(batch, max_pages, n_pages);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(B2_ERR_WORKSPACE, "kv4 reorder needs %zu bytes of 16-byte aligned workspace", need);
  p.table = table;
  p.lens = lens;
  p.refs = refs;
  p.parent = parent;
  p.reserve = reserve;
  p.table_out = table_out;
  p.lens_out = lens_out;
  p.refs_out = refs_out;
  p.info = info;
  p.need = static_cast<int*>(workspace);
  p.copy = p.need + batch;
  p.n_found = p.copy + batch;
  p.free_ids = p.n_found + 1;
  p.batch = batch;
  p.max_pages = max_pages;
  p.page = page;
  Kv4Launch a(dim3(b2::kKv4PlanCtas, 1, 1), b2::kKv4PlanThreads, stream);
  cudaError_t e = cudaLaunchKernelEx(&a.cfg, b2::kv4_reorder_plan_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "kv4 reorder launch (plan)");
  Kv4Launch c(dim3(kv4_copy_parts(p.data), batch, layers), b2::kKv4CopyThreads, stream);
  e = cudaLaunchKernelEx(&c.cfg, b2::kv4_reorder_fill_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "kv4 reorder launch (copies)");
  return B2_OK;
}

int b2_kv4_compact_workspace_size(int n_pages, size_t* bytes) {
  if (!bytes) return fail(B2_ERR_ARG, "null bytes pointer");
  if (n_pages < 1) return fail(B2_ERR_ARG, "empty pool");
  *bytes = 3 * static_cast<size_t>(n_pages) * sizeof(int);
  return B2_OK;
}

int b2_kv4_compact(uint8_t* pool, int64_t page_bytes, uint8_t* summary, int64_t summary_bytes, int layers, int n_pages,
                   const int32_t* table, const int32_t* refs, int batch, int max_pages, int32_t* table_out,
                   int32_t* refs_out, int32_t* info, void* workspace, size_t workspace_bytes, void* stream) {
  DevInfo di;
  int st = device_info(&di);
  if (st != B2_OK) return st;
  b2::Kv4CompactParams p = {};
  st = kv4_page_data(pool, page_bytes, summary, summary_bytes, layers, n_pages, &p.data);
  if (st != B2_OK) return st;
  if (batch < 1 || max_pages < 1) return fail(B2_ERR_ARG, "bad page table shape");
  if (!table || !refs || !table_out || !refs_out || !info) return fail(B2_ERR_ARG, "null pointer argument");
  if (table == table_out || refs == refs_out) return fail(B2_ERR_ARG, "the new rows need buffers of their own");
  const size_t need = 3 * static_cast<size_t>(n_pages) * sizeof(int);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(B2_ERR_WORKSPACE, "kv4 compact needs %zu bytes of 16-byte aligned workspace", need);
  p.table = table;
  p.refs = refs;
  p.table_out = table_out;
  p.refs_out = refs_out;
  p.info = info;
  p.to = static_cast<int*>(workspace);
  p.src = p.to + n_pages;
  p.dst = p.src + n_pages;
  p.batch = batch;
  p.max_pages = max_pages;
  Kv4Launch a(dim3(1, 1, 1), b2::kKv4ScanThreads, stream);
  cudaError_t e = cudaLaunchKernelEx(&a.cfg, b2::kv4_compact_plan_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "kv4 compact launch (plan)");
  Kv4Launch c(dim3(8 * di.sms, 1, 1), b2::kKv4CopyThreads, stream);
  e = cudaLaunchKernelEx(&c.cfg, b2::kv4_compact_move_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "kv4 compact launch (moves)");
  return B2_OK;
}

}  // extern "C"
