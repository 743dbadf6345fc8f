// Decode attention over the 4-bit paged KV cache: one query token per sequence.
//
//   q of head j rotated to position pos; for every token t of 0..pos (or of the selected
//   pages' tokens up to pos), with K[t] = d n + m and V[t] = e c + f (codes n, c):
//     s[t] = scale * (d (q . n) + m sum(q)),   p = softmax(s),
//     out  = sum_t (p[t] e[t]) c[t] + sum_t p[t] f[t]
//
// The codes enter mma.sync m16n8k16 as they are: a nibble in the low bits of an fp16 is the
// subnormal n * 2^-24 (or n * 2^-20 four bits up), exact, so a word of 8 codes becomes four
// A registers with one shift and four ANDs, no conversion and no offset to take off again;
// the scales multiply the products' fp32 sums.  S^T = K Q^T (16 tokens x 8 heads per
// instruction), O^T = V^T P^T; P moves from the accumulator's layout to the B operand's
// with movmatrix.
//
// Weights are taken against a running reference R per head (log2 units) instead of the
// running maximum: w = 2^(s - R) e goes into the product as fp16, R is raised, and the sums
// rescaled, only when some w passes 2^10.  R covers s + log2 e, so that w keeps fp16's 11
// bits whatever the size of the values; the sums L = sum 2^(s - R) and sum 2^(s - R) f stay
// in fp32.
#pragma once

#include "kv4_cell.cuh"

namespace b2 {

constexpr int kKv4MaxGroup = 8;  // q heads per kv head: the N of the MMA

struct Kv4DecodeParams {
  const float* q;  // [batch][ld_q], head j at j * D
  long long ld_q;
  const uint8_t* pool;
  const int* table;  // [batch][max_pages]
  const int* pos;    // [batch], -1: nothing to attend
  const int* sel;    // [batch][hkv][n_sel] page indices, ascending, or null
  void* out;         // [batch][ldo]
  float* part;       // [batch][hkv][n_splits] x (o [grp][D], R [grp], L [grp]) of splits not clustered
  long long ldo;
  float scale_log2;
  int batch, hq, hkv, page, max_pages, n_pages, n_sel;
  int n_splits, clustered;  // CTAs per (sequence, kv head); joined in a cluster or through part
  int max_tiles;            // tiles of the longest sequence planned for
  int out_f32;
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The query heads of one (sequence, kv head), ready as B operands: fp16 of q * scale * log2 e *
// 2^-ex (the head's largest in [1, 2)), odd dims / 16 to meet the nibbles four bits up.
template <int D>
struct Kv4Query {
  static constexpr int G = D / kKv4Group;
  uint32_t b[G][4][2][32];          // B fragments by lane
  float sum[G][kKv4MaxGroup];       // sum of the fp16 q over the group, * 2^-24
  float unit[kKv4MaxGroup];         // 2^24 * 2^ex
  __half h[kKv4MaxGroup][D];
};

template <int D, int THREADS>
__device__ __forceinline__ void kv4_load_query(const Kv4DecodeParams& p, const Kv4Rope& rope, int b, int kvh, int pos,
                                               Kv4Query<D>& Q) {
  constexpr int G = D / kKv4Group, J = D / 32, W = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = p.hq / p.hkv;
  for (int j = warp; j < kKv4MaxGroup; j += W) {
    float x[J];
    const float* src = p.q + static_cast<size_t>(b) * p.ld_q + static_cast<size_t>(kvh * grp + j) * D + lane;
#pragma unroll
    for (int i = 0; i < J; ++i) x[i] = j < grp ? src[32 * i] : 0.f;
    if (rope.on) {
#pragma unroll
      for (int i = 0; i < J / 2; ++i) {
        double u = static_cast<double>(pos) * rope.turn[lane + 32 * i];
        u -= rint(u);
        float sn, cs;
        sincospif(2.f * static_cast<float>(u), &sn, &cs);
        const float a = x[i], c = x[i + J / 2];
        x[i] = a * cs - c * sn;
        x[i + J / 2] = c * cs + a * sn;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < J; ++i) {
      x[i] *= p.scale_log2;
      top = fmaxf(top, fabsf(x[i]));
    }
    top = warp_max(top);
    int ex = 0;
    if (top > 0.f && top < INFINITY) ex = max(-100, min(100, static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127));
    const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const __half hv = __float2half_rn(x[2 * g + e] * down);
        s += __half2float(hv);
        Q.h[j][64 * g + 32 * e + lane] = hv;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) Q.sum[g][j] = s * 5.9604644775390625e-8f;  // 2^-24
    }
    if (lane == 0) Q.unit[j] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23) * 16777216.f;
  }
  __syncthreads();
  // fragment (g, w, sub) of k-step 2 w + sub: b0 = dims (o, o + 4), b1 = dims (o + 1, o + 5) / 16
  // with o = 16 c + 8 w + 2 sub
  for (int e = threadIdx.x; e < G * 4 * 32; e += THREADS) {
    const int l = e & 31, ks = e >> 5 & 3, g = e >> 7;
    const __half* src = &Q.h[l >> 2][64 * g + 16 * (l & 3) + 8 * (ks >> 1) + 2 * (ks & 1)];
    const __half s16 = __float2half_rn(0.0625f);
    const __half2 v0 = __halves2half2(src[0], src[4]), v1 = __halves2half2(__hmul(src[1], s16), __hmul(src[5], s16));
    Q.b[g][ks][0][l] = *reinterpret_cast<const uint32_t*>(&v0);
    Q.b[g][ks][1][l] = *reinterpret_cast<const uint32_t*>(&v1);
  }
  __syncthreads();
}

// Running state of one warp: heads 2c and 2c + 1 of the lane.
template <int D>
struct Kv4State {
  static constexpr int G = D / kKv4Group;
  float o[G][4][4];   // O^T accumulators, m-tile i of group g: dims 8g'+i and 8g'+4+i
  float m[G][2];      // sum p f
  float l[2], r[2];
};

// 2^x, flushing what is below fp32's normal range: a weight that small is nothing beside 1
__device__ __forceinline__ float kv4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// NT tiles of 16 tokens; the G cells of tile n start at cell + n * stride, left[n] of its
// tokens count.
template <int D, int NT>
__device__ __forceinline__ void kv4_tiles(const uint8_t* tile0, int stride, const int (&left)[NT],
                                          const uint32_t (&qb)[D / 64][4][2], const float (&qs)[D / 64][2],
                                          const float (&unit)[2], Kv4State<D>& st) {
  constexpr int G = D / kKv4Group;
  constexpr uint32_t kLo = 0x000F000Fu, kHi = 0x00F000F0u;
  const int lane = threadIdx.x & 31, gl = lane >> 2, c = lane & 3;
  float y[NT][4], e[NT][G][2], f[NT][G][2], emax[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint8_t* at = tile0 + n * stride + g * kKv4CellBytes;
      const uint4 kw = *reinterpret_cast<const uint4*>(at + gl * 64 + c * 16);
      const uint2 km = *reinterpret_cast<const uint2*>(at + kKv4KMeta + gl * 8);
      const uint2 vm = *reinterpret_cast<const uint2*>(at + kKv4VMeta + gl * 8);
      float a[4] = {0.f, 0.f, 0.f, 0.f};
      // words kw.x, kw.y are token gl's, kw.z, kw.w token gl + 8's
      mma_f16_m16n8k16(a[0], a[1], a[2], a[3], kw.x & kLo, kw.z & kLo, kw.x & kHi, kw.z & kHi, qb[g][0][0], qb[g][0][1]);
      mma_f16_m16n8k16(a[0], a[1], a[2], a[3], (kw.x >> 8) & kLo, (kw.z >> 8) & kLo, (kw.x >> 8) & kHi,
                       (kw.z >> 8) & kHi, qb[g][1][0], qb[g][1][1]);
      mma_f16_m16n8k16(a[0], a[1], a[2], a[3], kw.y & kLo, kw.w & kLo, kw.y & kHi, kw.w & kHi, qb[g][2][0], qb[g][2][1]);
      mma_f16_m16n8k16(a[0], a[1], a[2], a[3], (kw.y >> 8) & kLo, (kw.w >> 8) & kLo, (kw.y >> 8) & kHi,
                       (kw.w >> 8) & kHi, qb[g][3][0], qb[g][3][1]);
      const float d0 = bf16lo_to_f32(km.x), m0 = bf16hi_to_f32(km.x), d1 = bf16lo_to_f32(km.y), m1 = bf16hi_to_f32(km.y);
      y[n][0] = fmaf(d0, a[0], fmaf(m0, qs[g][0], y[n][0]));
      y[n][1] = fmaf(d0, a[1], fmaf(m0, qs[g][1], y[n][1]));
      y[n][2] = fmaf(d1, a[2], fmaf(m1, qs[g][0], y[n][2]));
      y[n][3] = fmaf(d1, a[3], fmaf(m1, qs[g][1], y[n][3]));
      e[n][g][0] = fmaxf(bf16lo_to_f32(vm.x), kKv4MinStep);
      f[n][g][0] = bf16hi_to_f32(vm.x);
      e[n][g][1] = fmaxf(bf16lo_to_f32(vm.y), kKv4MinStep);
      f[n][g][1] = bf16hi_to_f32(vm.y);
    }
    if (left[n] < kKv4Tile) {  // what lies behind the last token may hold anything
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (gl + 8 * i >= left[n]) {
          y[n][2 * i] = y[n][2 * i + 1] = -INFINITY;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            e[n][g][i] = kKv4MinStep;
            f[n][g][i] = 0.f;
          }
        }
    }
    emax[n][0] = e[n][0][0];
    emax[n][1] = e[n][0][1];
#pragma unroll
    for (int g = 1; g < G; ++g) {
      emax[n][0] = fmaxf(emax[n][0], e[n][g][0]);
      emax[n][1] = fmaxf(emax[n][1], e[n][g][1]);
    }
  }
  float pr[NT][4], top = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) pr[n][i] = kv4_ex2(fmaf(y[n][i], unit[i & 1], -st.r[i & 1]));
    top = fmaxf(top, fmaxf(fmaxf(pr[n][0], pr[n][1]) * emax[n][0], fmaxf(pr[n][2], pr[n][3]) * emax[n][1]));
  }
  if (__any_sync(0xffffffffu, top > 1024.f)) {
    // raise R to the largest s + log2 e seen, and rescale what has been summed against the old one
    float r[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i & 1] = fmaxf(r[i & 1], fmaf(y[n][i], unit[i & 1], log2f(emax[n][i >> 1])));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) r[i] = fmaxf(r[i], __shfl_xor_sync(0xffffffffu, r[i], o));
      r[i] = fmaxf(r[i], st.r[i]);
      const float s = kv4_ex2(st.r[i] - r[i]);
      st.r[i] = r[i];
      st.l[i] *= s;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        st.m[g][i] *= s;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          st.o[g][k][i] *= s;
          st.o[g][k][i + 2] *= s;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) pr[n][i] = kv4_ex2(fmaf(y[n][i], unit[i & 1], -st.r[i & 1]));
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    st.l[0] += pr[n][0] + pr[n][2];
    st.l[1] += pr[n][1] + pr[n][3];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      st.m[g][0] = fmaf(pr[n][0], f[n][g][0], fmaf(pr[n][2], f[n][g][1], st.m[g][0]));
      st.m[g][1] = fmaf(pr[n][1], f[n][g][0], fmaf(pr[n][3], f[n][g][1], st.m[g][1]));
      const uint32_t b0 = movmatrix_trans(pack_f16x2(pr[n][0] * e[n][g][0], pr[n][1] * e[n][g][0]));
      const uint32_t b1 = movmatrix_trans(pack_f16x2(pr[n][2] * e[n][g][1], pr[n][3] * e[n][g][1]));
      const uint4 v = *reinterpret_cast<const uint4*>(tile0 + n * stride + g * kKv4CellBytes + kKv4VCodes + gl * 64 + c * 16);
      float(&o)[4][4] = st.o[g];
      mma_f16_m16n8k16(o[0][0], o[0][1], o[0][2], o[0][3], v.x & kLo, v.y & kLo, v.z & kLo, v.w & kLo, b0, b1);
      mma_f16_m16n8k16(o[1][0], o[1][1], o[1][2], o[1][3], v.x & kHi, v.y & kHi, v.z & kHi, v.w & kHi, b0, b1);
      mma_f16_m16n8k16(o[2][0], o[2][1], o[2][2], o[2][3], (v.x >> 8) & kLo, (v.y >> 8) & kLo, (v.z >> 8) & kLo,
                       (v.w >> 8) & kLo, b0, b1);
      mma_f16_m16n8k16(o[3][0], o[3][1], o[3][2], o[3][3], (v.x >> 8) & kHi, (v.y >> 8) & kHi, (v.z >> 8) & kHi,
                       (v.w >> 8) & kHi, b0, b1);
    }
  }
}

__device__ __forceinline__ void kv4_store_out(const Kv4DecodeParams& p, int b, int head, int D, int d, float v) {
  const size_t i = static_cast<size_t>(b) * p.ldo + static_cast<size_t>(head) * D + d;
  if (p.out_f32) static_cast<float*>(p.out)[i] = v;
  else static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}

// Work split: CTA (split, kv head, sequence), W warps.  A sequence's tiles are dealt to its
// CTAs in equal runs (by its own length, so that no CTA of a long sequence has more than its
// share and short ones cost little), a run's stages to the warps in turn.  Every warp fills a
// ring of its own with bulk copies, one per tile, a lane each, several stages ahead, and
// looks the pages up 32 tiles at a time.  Splits of one (sequence, kv head) form a cluster
// and are joined through its shared memory; more than 16 go through the workspace.
template <int D>
struct Kv4Ring {
  static constexpr int G = D / kKv4Group;
  static constexpr int kTileBytes = G * kKv4CellBytes;
  static constexpr int kTiles = D == 64 ? 2 : 1;   // tiles of a stage, taken together
  static constexpr int kStages = D == 256 ? 3 : 4;
  static constexpr int kStageBytes = kTiles * kTileBytes;
};
template <int D, int W>
__host__ __device__ constexpr size_t kv4_decode_smem() {
  return static_cast<size_t>(W) * Kv4Ring<D>::kStages * Kv4Ring<D>::kStageBytes;
}

template <int D, int W>
__global__ void __launch_bounds__(W * 32) kv4_decode_kernel(const Kv4DecodeParams p,
                                                            const __grid_constant__ Kv4Rope rope) {
  using Ring = Kv4Ring<D>;
  constexpr int G = D / kKv4Group, ST = Ring::kTiles, NS = Ring::kStages;
  extern __shared__ __align__(128) uint8_t rings[];
  __shared__ Kv4Query<D> Q;
  __shared__ __align__(8) uint64_t full[W][NS];
  __shared__ int left_s[W][NS][ST];
  __shared__ float mr[W][kKv4MaxGroup], ml[W][kKv4MaxGroup];
  __shared__ int abort_flag;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, c = lane & 3;
  const int grp = p.hq / p.hkv, tpp = p.page / kKv4Tile;

  if (lane < NS) mbar_init(smem_u32(&full[warp][lane]), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  pdl_wait();
  pdl_launch_dependents();
  const int pos = p.pos[b];
  if (pos < -1 || pos >= static_cast<long long>(p.max_pages) * p.page ||
      (!p.sel && pos >= p.max_tiles * static_cast<long long>(kKv4Tile))) {
    if (threadIdx.x == 0) record_error(kDevBadPosition);
    return;  // the whole sequence and cluster, before any barrier: nothing is read or written
  }
  __syncwarp();

  // ---- this warp's tiles: index i -> stage i / ST -> tile
  const int* row = p.table + static_cast<size_t>(b) * p.max_pages;
  const int* sel = p.sel ? p.sel + (static_cast<size_t>(b) * p.hkv + kvh) * p.n_sel : nullptr;
  const size_t head_bytes = static_cast<size_t>(tpp) * Ring::kTileBytes;
  const int n_tiles = sel ? p.n_sel * tpp : pos / kKv4Tile + (pos >= 0);
  const int groups = (n_tiles + ST - 1) / ST;  // stages of the whole sequence
  const int g_lo = static_cast<int>(static_cast<long long>(groups) * split / p.n_splits);
  const int g_hi = static_cast<int>(static_cast<long long>(groups) * (split + 1) / p.n_splits);
  const int n_stages = max(0, (g_hi - g_lo - warp + W - 1) / W);
  // lane's tile of the 32 that begin with tile index i0: its address, or its page's lookup
  auto find = [&](int i0, int& left) -> const uint8_t* {
    const int i = i0 + lane;
    left = 0;
    if (i >= n_stages * ST) return nullptr;
    const int tile = (g_lo + warp + i / ST * W) * ST + i % ST;
    if (tile >= n_tiles) return nullptr;
    int pg = tile / tpp;
    const int in_page = tile - pg * tpp;
    if (sel) {  // an entry that does not rise above the one before it counts for nothing
      const int at = pg;
      pg = sel[at];
      if (pg < 0 || pg >= p.max_pages || (at > 0 && pg <= sel[at - 1])) return nullptr;
    }
    const long long first = static_cast<long long>(pg) * p.page + in_page * kKv4Tile;
    if (first > pos) return nullptr;
    const int id = row[pg];
    if (id < 0 || id >= p.n_pages) {
      record_error(kDevBadPosition);
      return nullptr;
    }
    left = static_cast<int>(min(static_cast<long long>(kKv4Tile), pos + 1 - first));
    return p.pool + (static_cast<size_t>(id) * p.hkv + kvh) * head_bytes + static_cast<size_t>(in_page) * Ring::kTileBytes;
  };
  uint8_t* ring = rings + static_cast<size_t>(warp) * NS * Ring::kStageBytes;
  const uint64_t once = l2_evict_first_policy();
  int left_now, left_next;
  const uint8_t* at_now = find(0, left_now);
  const uint8_t* at_next = n_stages * ST > 32 ? find(32, left_next) : nullptr;
  // stage s into its slot: the lanes that hold its tiles copy them
  auto issue = [&](int s) {
    const int i = s * ST;
    if (i > 0 && i % 32 == 0) {
      at_now = at_next;
      left_now = left_next;
      if (i + 32 < n_stages * ST) at_next = find(i + 32, left_next);
    }
    const int mine = lane - i % 32;  // this lane's tile of the stage, if 0 .. ST - 1
    const bool in = mine >= 0 && mine < ST;
    const int count = __popc(__ballot_sync(0xffffffffu, in && left_now > 0));
    const uint32_t bar = smem_u32(&full[warp][s % NS]);
    if (in) left_s[warp][s % NS][mine] = left_now;
    if (lane == 0) mbar_arrive_expect_tx(bar, count * Ring::kTileBytes);
    __syncwarp();
    if (in && left_now > 0)
      bulk_g2s(smem_u32(ring + (s % NS) * Ring::kStageBytes + mine * Ring::kTileBytes), at_now, Ring::kTileBytes, bar, once);
  };
  int issued = 0;
  for (; issued < min(NS, n_stages); ++issued) issue(issued);

  // ---- the query, while the first stages are on their way
  kv4_load_query<D, W * 32>(p, rope, b, kvh, max(pos, 0), Q);
  uint32_t qb[G][4][2];
  float qs[G][2], unit[2] = {Q.unit[2 * c], Q.unit[2 * c + 1]};
  Kv4State<D> st;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      qb[g][k][0] = Q.b[g][k][0][lane];
      qb[g][k][1] = Q.b[g][k][1][lane];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qs[g][e] = Q.sum[g][2 * c + e];
      st.m[g][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) st.o[g][i][0] = st.o[g][i][1] = st.o[g][i][2] = st.o[g][i][3] = 0.f;
  }
  st.l[0] = st.l[1] = 0.f;
  st.r[0] = st.r[1] = -1e30f;

  int s = 0;
  for (; s < n_stages; ++s) {
    // a wait that runs out ends this warp's work: the result is void, and reported
    const bool here = mbar_wait_bounded(smem_u32(&full[warp][s % NS]), (s / NS) & 1, &abort_flag, kDevTimeoutFull);
    if (!__all_sync(0xffffffffu, here)) break;
    int left[ST];
#pragma unroll
    for (int n = 0; n < ST; ++n) left[n] = left_s[warp][s % NS][n];
    kv4_tiles<D, ST>(ring + (s % NS) * Ring::kStageBytes, Ring::kTileBytes, left, qb, qs, unit, st);
    __syncwarp();  // every lane has read the slot
    if (issued < n_stages) issue(issued++);
  }
  if (s < n_stages)  // copies still in flight land before the ring is used for anything else
    for (; s < issued; ++s) {
      const uint64_t t0 = globaltimer();
      while (!mbar_try_wait(smem_u32(&full[warp][s % NS]), (s / NS) & 1))
        if (globaltimer() - t0 > B2_WAIT_TIMEOUT_NS) {
          record_error(kDevTimeoutDrain);
          break;
        }
    }

  // ---- the warp's sums over its token lanes, then the warps through shared memory
  float(*mo)[kKv4MaxGroup][D + 1] = reinterpret_cast<float(*)[kKv4MaxGroup][D + 1]>(rings);
  static_assert(W * kKv4MaxGroup * (D + 1) * 4 <= kv4_decode_smem<D, W>(), "the sums fit the rings");
  __syncthreads();  // every warp is done with its ring
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], o);
#pragma unroll
      for (int g = 0; g < G; ++g) st.m[g][e] += __shfl_xor_sync(0xffffffffu, st.m[g][e], o);
    }
    if (gl == 0) {
      ml[warp][2 * c + e] = st.l[e];
      mr[warp][2 * c + e] = st.r[e];
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float scale = i & 1 ? 1048576.f : 16777216.f;  // 2^20, 2^24
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mo[warp][2 * c + e][64 * g + 8 * gl + i] = fmaf(st.o[g][i][e], scale, st.m[g][e]);
        mo[warp][2 * c + e][64 * g + 8 * gl + 4 + i] = fmaf(st.o[g][i][2 + e], scale, st.m[g][e]);
      }
    }
  __syncthreads();
  // the CTA's sums over Q's memory (last read before the loop): o [grp][D], then R and L
  float* cta = reinterpret_cast<float*>(&Q);
  static_assert(sizeof(Kv4Query<D>) >= kKv4MaxGroup * (D + 2) * 4, "the CTA's sums fit the query's memory");
  for (int e = threadIdx.x; e < grp * D; e += W * 32) {
    const int j = e / D, d = e % D;
    float R = -1e30f, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (ml[w][j] != 0.f) R = fmaxf(R, mr[w][j]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (ml[w][j] == 0.f) continue;
      const float f = kv4_ex2(mr[w][j] - R);
      L = fmaf(ml[w][j], f, L);
      O = fmaf(mo[w][j][d], f, O);
    }
    if (p.n_splits == 1) {
      kv4_store_out(p, b, kvh * grp + j, D, d, L == 0.f ? 0.f : O / L);
    } else {
      float* part = p.clustered ? cta : p.part + ((static_cast<size_t>(b) * p.hkv + kvh) * p.n_splits + split) * grp * (D + 2);
      part[e] = O;
      if (d == 0) {
        part[grp * D + j] = R;
        part[grp * D + grp + j] = L;
      }
    }
  }
  if (!p.clustered) return;
  cluster_sync_all();
  // every CTA of the cluster joins a share of the outputs
  const uint32_t base = smem_u32(cta);
  for (int e = split * W * 32 + threadIdx.x; e < grp * D; e += p.n_splits * W * 32) {
    const int j = e / D;
    float R = -1e30f, L = 0.f, O = 0.f;
    for (int k = 0; k < p.n_splits; ++k)
      if (ld_dsmem_f32(base + (grp * D + grp + j) * 4, k) != 0.f) R = fmaxf(R, ld_dsmem_f32(base + (grp * D + j) * 4, k));
    for (int k = 0; k < p.n_splits; ++k) {
      const float l = ld_dsmem_f32(base + (grp * D + grp + j) * 4, k);
      const float f = l == 0.f ? 0.f : kv4_ex2(ld_dsmem_f32(base + (grp * D + j) * 4, k) - R);
      const float o = ld_dsmem_f32(base + e * 4, k);
      if (l != 0.f) {
        L = fmaf(l, f, L);
        O = fmaf(o, f, O);
      }
    }
    kv4_store_out(p, b, kvh * grp + j, D, e % D, L == 0.f ? 0.f : O / L);
  }
  cluster_sync_all();  // no CTA's shared memory goes while another reads it
}

// Joins the splits: one CTA per (q head, sequence), a thread per dim.
template <int D>
__global__ void __launch_bounds__(D) kv4_combine_kernel(const Kv4DecodeParams p) {
  const int head = blockIdx.x, b = blockIdx.y, d = threadIdx.x, grp = p.hq / p.hkv;
  pdl_wait();
  pdl_launch_dependents();
  const int pos = p.pos[b];
  if (pos < -1 || pos >= static_cast<long long>(p.max_pages) * p.page ||
      (!p.sel && pos >= p.max_tiles * static_cast<long long>(kKv4Tile)))
    return;
  const int j = head % grp;
  const size_t step = static_cast<size_t>(grp) * (D + 2);
  const float* part = p.part + (static_cast<size_t>(b) * p.hkv + head / grp) * p.n_splits * step;
  float R = -1e30f, L = 0.f, O = 0.f;
  for (int s = 0; s < p.n_splits; ++s)
    if (part[s * step + grp * D + grp + j] != 0.f) R = fmaxf(R, part[s * step + grp * D + j]);
  for (int s = 0; s < p.n_splits; ++s) {
    const float l = part[s * step + grp * D + grp + j];
    if (l == 0.f) continue;
    const float w = kv4_ex2(part[s * step + grp * D + j] - R);
    L = fmaf(l, w, L);
    O = fmaf(part[s * step + j * D + d], w, O);
  }
  kv4_store_out(p, b, head, D, d, L == 0.f ? 0.f : O / L);
}

}  // namespace b2
