// Decode attention over the 4-bit paged KV cache: one query token per sequence.
//
//   q of head j rotated to position pos; for every token t of 0..pos (or of the selected
//   pages' tokens up to pos), with K[t] = d n + m and V[t] = e c + f (codes n, c):
//     s[t] = scale * (d (q . n) + m sum(q)),   p = softmax(s),
//     out  = sum_t (p[t] e[t]) c[t] + sum_t p[t] f[t]
//
// The codes enter mma.sync m16n8k16 as they are: an integer below 2^10 in the low bits of an
// fp16 is the subnormal n * 2^-24, exact.  A byte of two codes a + 16 b goes in twice, whole
// and as its low nibble a: two byte permutations and two ANDs make four A registers of a word
// of 8 codes, without a conversion or an offset.  For the scores a q_a + b q_b is
// (a + 16 b) (q_b / 16) + a (q_a - q_b / 16); of the values' sums, sum w b is
// (sum w (a + 16 b) - sum w a) / 16 at the end.  The scales multiply the products' fp32 sums.
// S^T = K Q^T (16 tokens x 8 heads per instruction), O^T = V^T P^T; P moves from the
// accumulator's layout to the B operand's with movmatrix.
//
// The fp16 weight w is off by up to 2^-11 of the fp32 one, u, and the tensor cores' fp32 sums are
// truncated, not rounded.  Both would add up over a long sequence, as codes are never negative
// (32 sequences of 32768 equal scores: 8e-3 of the output's norm), so sums are kept around zero:
//   out = sum w (c - 7.5) + sum p (f + 7.5 e),  sum w (c - 7.5) = sum w c - 7.5 sum w,
// the last sum in fp32; and every other tile enters negated, as (-w) (15 - c), whose like sum is
// sum (-w) (15 - c) - 7.5 sum (-w).  What stays is one rounding of a weight against half the
// range of the values (that case: 2.0e-4; random queries over 512 to 32768 tokens 2.7e-4 to
// 3.0e-4, half of it q's rounding, and 4.1e-4 to 6.4e-4 with the plain sums).  64 sequences of
// 4096 take 39.4 us so and took 37.5; with a product by -7.5 after each one instead, 43.4.
//
// Weights are taken against a running reference R per head (log2 units) instead of the
// running maximum: w = 2^(s - R) e goes into the product as fp16, R is raised, and the sums
// rescaled, only when some w passes 2^10.  R covers s + log2 e of the largest e of a token's
// groups of 64 dims.  A group whose own largest weight then lies below 2^-10 is weighed in a unit
// of its own, a power of two by head and group that its sums carry to the end, so that its w keep
// fp16's bits too: rare in earnest, so tiles are first taken as if all units were 1 (256 sequences
// of 2048 of 256 dims 75.0 us so, 73.5 without units, 79.0 with them in every tile).  The sums
// L = sum 2^(s - R) and sum 2^(s - R) f stay in fp32; with the least e, 2^-40, the weights 2^(s - R)
// reach 2^50, and f may be 2^60 in size.
#pragma once

#include "kv4_cell.cuh"

namespace b2 {

constexpr int kKv4MaxGroup = 8;  // q heads per kv head: the N of the MMA

// a CTA's sums of one pair: o [grp][D], R [grp], L [grp], up to 16 bytes
__host__ __device__ constexpr int kv4_part_floats(int grp, int D) { return (grp * (D + 2) + 3) / 4 * 4; }

struct Kv4DecodeParams {
  const float* q;  // [batch][ld_q], head j at j * D
  long long ld_q;
  const uint8_t* pool;
  const int* table;  // [batch][max_pages]
  const int* pos;    // [batch], -1: nothing to attend
  const int* sel;    // [batch][hkv][n_sel] page indices, ascending, or null
  void* out;         // [batch][ldo]
  float* part;       // [grid][2][kv4_part_floats]: the ends of pairs that several CTAs share
  long long ldo;
  float scale_log2;
  int batch, hq, hkv, page, max_pages, n_pages, n_sel;
  int max_len;    // tokens of the longest sequence planned for (without sel)
  int splits;     // CTAs of a (sequence, kv head), a cluster; 0: the tiles are dealt over the grid
  int2* spans;    // [batch][hkv] the CTAs that share a pair, or x = -1 (dealt over the grid)
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

// The query heads of one (sequence, kv head), ready as B operands: of q * scale * log2 e *
// 2^-ex (the head's largest in [1, 2)), h1 = fp16(odd dim) / 16 and h0 = fp16(even dim - h1).
// Fragment (g, ks) of lane (head, c), with o = 16 c + 4 ks: h1 of (o + 1, o + 3), then h0 of
// (o, o + 2).
template <int D>
struct Kv4Query {
  static constexpr int G = D / kKv4Group;
  __half b[G][4][2][32][2];
  float sum[G][kKv4MaxGroup];  // sum over the group of q as the fragments have it, * 2^-24
  float unit[kKv4MaxGroup];    // 2^24 * 2^ex
};

// A warp's heads of the query as they are stored (warp, warp + W, ..), dims lane + 32 i.
template <int D, int W>
struct Kv4RawQuery {
  static constexpr int H = kKv4MaxGroup / W;
  float x[H][D / 32];
};
template <int D, int W>
__device__ __forceinline__ void kv4_load_query(const Kv4DecodeParams& p, int b, int kvh, Kv4RawQuery<D, W>& q) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = p.hq / p.hkv;
#pragma unroll
  for (int h = 0; h < Kv4RawQuery<D, W>::H; ++h) {
    const int j = warp + h * W;
    const float* src = p.q + static_cast<size_t>(b) * p.ld_q + static_cast<size_t>(kvh * grp + j) * D + lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q.x[h][i] = j < grp ? src[32 * i] : 0.f;
  }
}

template <int D, int W>
__device__ __forceinline__ void kv4_prepare_query(const Kv4DecodeParams& p, const Kv4Rope& rope, int pos,
                                                  Kv4RawQuery<D, W>& q, Kv4Query<D>& Q) {
  constexpr int G = D / kKv4Group, J = D / 32, H = Kv4RawQuery<D, W>::H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float top[H], s[H][G];
#pragma unroll
  for (int h = 0; h < H; ++h) top[h] = 0.f;
#pragma unroll
  for (int i = 0; i < J / 2; ++i) {
    float sn = 0.f, cs = 1.f;
    if (rope.on) {
      double u = static_cast<double>(pos) * kv4_turn(rope, lane + 32 * i);
      u -= rint(u);
      sincospif(2.f * static_cast<float>(u), &sn, &cs);
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float a = q.x[h][i] * p.scale_log2, z = q.x[h][i + J / 2] * p.scale_log2;
      q.x[h][i] = a * cs - z * sn;
      q.x[h][i + J / 2] = z * cs + a * sn;
      top[h] = fmaxf(top[h], fmaxf(fabsf(q.x[h][i]), fabsf(q.x[h][i + J / 2])));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int h = 0; h < H; ++h) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
#pragma unroll
  for (int h = 0; h < H; ++h) {
    int ex = 0;
    if (top[h] > 0.f && top[h] < INFINITY)
      ex = max(-100, min(100, static_cast<int>((__float_as_uint(top[h]) >> 23) & 255u) - 127));
    const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
    const int j = warp + h * W;
#pragma unroll
    for (int i = 0; i < J; ++i) {
      const int d = (lane + 32 * i) & 63;  // this lane's dim of the group
      const float x = q.x[h][i] * down;
      const float h1 = __half2float(__float2half_rn(__half2float(__float2half_rn(x)) * 0.0625f));  // for odd lanes
      const float beside = __shfl_xor_sync(0xffffffffu, h1, 1);
      const __half v = __float2half_rn(lane & 1 ? h1 : x - beside);
      const float as_is = lane & 1 ? 16.f * h1 : __half2float(v) + beside;
      s[h][i / 2] = i % 2 ? s[h][i / 2] + as_is : as_is;
      Q.b[i / 2][d >> 2 & 3][1 - (lane & 1)][4 * j + (d >> 4)][d >> 1 & 1] = v;
    }
    if (lane == 0) Q.unit[j] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23) * 16777216.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g) s[h][g] += __shfl_xor_sync(0xffffffffu, s[h][g], o);
  if (lane == 0) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g) Q.sum[g][warp + h * W] = s[h][g] * 5.9604644775390625e-8f;  // 2^-24
  }
}

constexpr float kKv4NoScore = -3.402823466e38f;  // R before the first token: below any finite score

// Running state of one warp: heads 2c and 2c + 1 of the lane.
template <int D>
struct Kv4State {
  static constexpr int G = D / kKv4Group;
  float o[G][4][4];   // O^T accumulators of group g, rows 8 (lane / 4) + i and + 4: even i the sum of
                      // w a (dim i), odd i that of w (a + 16 b) (dims i - 1 and i), negated tiles as said
  float m[G][2];      // sum p (f + 7.5 e) - 7.5 w, w negated with its tile
  float l[2], r[2];
};

// A group whose largest weight is not below this is weighed as it is: 2^-15 of that weight is
// then what fp16's subnormals lose.
constexpr float kKv4NearOne = 0x1p-10f;

// Orders this thread's accesses to shared memory before later bulk copies into it.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 2^x, flushing what is below fp32's normal range: a weight that small is nothing beside 1
__device__ __forceinline__ float kv4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 over the power of two at or below x (2^-60 <= x <= 2^60)
__device__ __forceinline__ float kv4_power_inv(float x) {
  return __uint_as_float(0x7F000000u - (__float_as_uint(x) & 0x7F800000u));
}

// A B with nothing to add to.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// m - 7.5 w, w an fp16, in one rounding
__device__ __forceinline__ float kv4_less_middle(uint32_t w, float m) {
  float d;
  asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(static_cast<uint16_t>(w)), "h"(static_cast<uint16_t>(0xC780u)), "f"(m));
  return d;
}

__device__ __forceinline__ uint32_t f16x2_max_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// NT tiles of 16 tokens; the G cells of tile n start at tile0 + n * stride.  index: the first
// tile's place in its stage; odd ones are negated.
// ANY: only left[n] of a tile's tokens count, and the groups' units (times; scaled: some are not
// 1) are set as they have to be; returns whether they are all 1.  Else the tiles are full and the
// units 1; where one has to be set nothing is done (false).
template <int D, int NT, bool ANY>
__device__ __forceinline__ bool kv4_tiles(const uint8_t* tile0, int stride, int index, const int* left,
                                          const uint32_t (&qb)[D / 64][4][2], const float (&qs)[D / 64][2],
                                          const float (&unit)[2], float (*times)[kKv4MaxGroup], bool scaled, Kv4State<D>& st) {
  constexpr int G = D / kKv4Group;
  constexpr uint32_t kLo = 0x000F000Fu;
  const int lane = threadIdx.x & 31, gl = lane >> 2, c = lane & 3;
  float y[NT][4];
  uint2 vm[NT][G];  // (e, f) of tokens gl and gl + 8 as they are stored
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint8_t* at = tile0 + n * stride + g * kKv4CellBytes;
      const uint4 kw = *reinterpret_cast<const uint4*>(at + gl * 64 + c * 16);
      const uint2 km = *reinterpret_cast<const uint2*>(at + kKv4KMeta + gl * 8);
      vm[n][g] = *reinterpret_cast<const uint2*>(at + kKv4VMeta + gl * 8);
      float a[4];
      // words kw.x, kw.y are token gl's, kw.z, kw.w token gl + 8's
      const uint32_t t0[2] = {kw.x, kw.y}, t1[2] = {kw.z, kw.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t sel = k & 1 ? 0x4342u : 0x4140u;  // a word's bytes 0 and 1, or 2 and 3, 16 bits each
        const uint32_t y0 = prmt(t0[k >> 1], 0u, sel), y1 = prmt(t1[k >> 1], 0u, sel);
        if (k == 0) mma_f16_first(a, y0, y1, y0 & kLo, y1 & kLo, qb[g][k][0], qb[g][k][1]);
        else mma_f16_m16n8k16(a[0], a[1], a[2], a[3], y0, y1, y0 & kLo, y1 & kLo, qb[g][k][0], qb[g][k][1]);
      }
      const float d0 = bf16lo_to_f32(km.x), m0 = bf16hi_to_f32(km.x), d1 = bf16lo_to_f32(km.y), m1 = bf16hi_to_f32(km.y);
      y[n][0] = fmaf(d0, a[0], fmaf(m0, qs[g][0], y[n][0]));
      y[n][1] = fmaf(d0, a[1], fmaf(m0, qs[g][1], y[n][1]));
      y[n][2] = fmaf(d1, a[2], fmaf(m1, qs[g][0], y[n][2]));
      y[n][3] = fmaf(d1, a[3], fmaf(m1, qs[g][1], y[n][3]));
    }
    if (ANY) {  // what lies behind the last token may hold anything
      constexpr uint32_t kNothing = 0x2B80u;  // e = 2^-40, f = 0
      if (gl >= left[n]) {
        y[n][0] = y[n][1] = -INFINITY;
#pragma unroll
        for (int g = 0; g < G; ++g) vm[n][g].x = kNothing;
      }
      if (gl + 8 >= left[n]) {
        y[n][2] = y[n][3] = -INFINITY;
#pragma unroll
        for (int g = 0; g < G; ++g) vm[n][g].y = kNothing;
      }
    }
  }
  float pr[NT][4];
  uint32_t w[NT][G][2];  // the weights of heads 2c, 2c + 1, for token gl and token gl + 8
  // weights against the present R (weigh) and the groups' units (pack); whether one of them has
  // come to 2^10, or is not a number.  Against a new R the scores are rounded as they were for it:
  // past 2^27 an unrounded product may lie further above R than fp16 reaches.
  auto weigh = [&](bool anew) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pr[n][i] = kv4_ex2(anew ? __fmul_rn(y[n][i], unit[i & 1]) - st.r[i & 1] : fmaf(y[n][i], unit[i & 1], -st.r[i & 1]));
  };
  auto pack = [&]() -> bool {
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float e0 = bf16lo_to_f32(vm[n][g].x), e1 = bf16lo_to_f32(vm[n][g].y);
        const float u0 = ANY && G > 1 && scaled ? times[g][2 * c] : 1.f, u1 = ANY && G > 1 && scaled ? times[g][2 * c + 1] : 1.f;
        w[n][g][0] = pack_f16x2(pr[n][0] * u0 * e0, pr[n][1] * u1 * e0);
        w[n][g][1] = pack_f16x2(pr[n][2] * u0 * e1, pr[n][3] * u1 * e1);
        top = f16x2_max_nan(top, f16x2_max_nan(w[n][g][0], w[n][g][1]));
      }
    return (top + 0x1C001C00u) & 0x80008000u;  // 0x6400 is 2^10
  };
  weigh(false);
  if (__any_sync(0xffffffffu, pack())) {
    // raise R to the largest s + log2 e seen, and rescale what has been summed against the old one
    float r[2] = {-INFINITY, -INFINITY}, fall[2];
    const float before[2] = {st.r[0], st.r[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float e = kKv4MinStep;
#pragma unroll
        for (int g = 0; g < G; ++g) e = fmaxf(e, bf16lo_to_f32(i < 2 ? vm[n][g].x : vm[n][g].y));
        r[i & 1] = fmaxf(r[i & 1], __fmul_rn(y[n][i], unit[i & 1]) + log2f(e));
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) r[i] = fmaxf(r[i], __shfl_xor_sync(0xffffffffu, r[i], o));
      r[i] = fmaxf(r[i], st.r[i]);
      fall[i] = kv4_ex2(st.r[i] - r[i]);
      st.r[i] = r[i];
    }
    weigh(true);
    float step[G][2];  // what the groups' units change by
#pragma unroll
    for (int g = 0; g < G; ++g) step[g][0] = step[g][1] = 1.f;
    if (G > 1) {  // does every group have a weight near 1, for every head?
      auto most = [&](int g, int i) {
        float x = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          x = fmaxf(x, fmaxf(pr[n][i] * bf16lo_to_f32(vm[n][g].x), pr[n][i + 2] * bf16lo_to_f32(vm[n][g].y)));
        return x;
      };
      bool near = !scaled;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = most(g, i);
          const unsigned large = __ballot_sync(0xffffffffu, x >= kKv4NearOne);
          near = near && (large >> c & 0x11111111u) != 0 && x < 2.f;
        }
      if (!__all_sync(0xffffffffu, near)) {
        if (!ANY) {
          st.r[0] = before[0];
          st.r[1] = before[1];
          return false;
        }
        bool one = true;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x = most(g, i);
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float old = times[g][2 * c + i];
            x = fmaxf(x, fall[i] * kv4_power_inv(old));  // or the largest that it had
            float now = x >= kKv4NearOne && x < 2.f ? 1.f : kv4_power_inv(fminf(fmaxf(x, 0x1p-60f), 0x1p60f));
            if (st.r[i] == kKv4NoScore) now = old;  // no score yet
            one = one && now == 1.f;
            step[g][i] = now * kv4_power_inv(old);
            __syncwarp();
            times[g][2 * c + i] = now;  // the same from all lanes of the head
          }
        __syncwarp();
        scaled = !__all_sync(0xffffffffu, one);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      st.l[i] *= fall[i];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float f = fall[i] * step[g][i];
        st.m[g][i] *= f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          st.o[g][k][i] *= f;
          st.o[g][k][i + 2] *= f;
        }
      }
    }
    pack();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    st.l[0] += pr[n][0] + pr[n][2];
    st.l[1] += pr[n][1] + pr[n][3];
    const uint32_t negate = (index + n) & 1 ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float f0 = fmaf(7.5f, bf16lo_to_f32(vm[n][g].x), bf16hi_to_f32(vm[n][g].x));
      const float f1 = fmaf(7.5f, bf16lo_to_f32(vm[n][g].y), bf16hi_to_f32(vm[n][g].y));
      const float u0 = ANY && G > 1 && scaled ? times[g][2 * c] : 1.f, u1 = ANY && G > 1 && scaled ? times[g][2 * c + 1] : 1.f;
      st.m[g][0] = fmaf(pr[n][0] * u0, f0, fmaf(pr[n][2] * u0, f1, st.m[g][0]));
      st.m[g][1] = fmaf(pr[n][1] * u1, f0, fmaf(pr[n][3] * u1, f1, st.m[g][1]));
      const uint32_t w0 = w[n][g][0] ^ (negate & 0x80008000u), w1 = w[n][g][1] ^ (negate & 0x80008000u);
      st.m[g][0] = kv4_less_middle(w0 & 0xFFFFu, kv4_less_middle(w1 & 0xFFFFu, st.m[g][0]));
      st.m[g][1] = kv4_less_middle(w0 >> 16, kv4_less_middle(w1 >> 16, st.m[g][1]));
      const uint32_t b0 = movmatrix_trans(w0), b1 = movmatrix_trans(w1);
      uint4 v = *reinterpret_cast<const uint4*>(tile0 + n * stride + g * kKv4CellBytes + kKv4VCodes + gl * 64 + c * 16);
      v.x ^= negate;
      v.y ^= negate;
      v.z ^= negate;
      v.w ^= negate;
      float(&o)[4][4] = st.o[g];
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // bytes 0 and 2, then 1 and 3: the same dims of two tokens
        const uint32_t pick = k ? 0x4341u : 0x4240u;
        const uint32_t a0 = prmt(v.x, 0u, pick), a1 = prmt(v.y, 0u, pick), a2 = prmt(v.z, 0u, pick), a3 = prmt(v.w, 0u, pick);
        mma_f16_m16n8k16(o[2 * k][0], o[2 * k][1], o[2 * k][2], o[2 * k][3], a0 & kLo, a1 & kLo, a2 & kLo, a3 & kLo, b0, b1);
        mma_f16_m16n8k16(o[2 * k + 1][0], o[2 * k + 1][1], o[2 * k + 1][2], o[2 * k + 1][3], a0, a1, a2, a3, b0, b1);
      }
    }
  }
  return ANY ? !scaled : true;
}


__device__ __forceinline__ void kv4_store_out(const Kv4DecodeParams& p, int b, int head, int D, int d, float v) {
  const size_t i = static_cast<size_t>(b) * p.ldo + static_cast<size_t>(head) * D + d;
  if (p.out_f32) static_cast<float*>(p.out)[i] = v;
  else static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}

// Work split.  A pair is a (sequence, kv head); its tiles of 16 tokens go to CTAs of W warps
// in one of two ways.
//   Few tiles in all: a cluster of `splits` CTAs per pair, joined through its shared memory.
//   Else the tiles of all pairs, in a row, are dealt to as many CTAs as the GPU holds at
//   once, the same number to each whatever the lengths: a CTA takes the end of one pair, some
//   whole ones and the beginning of another, and a second kernel joins the pairs that were
//   cut.  (One grid row of CTAs per pair left SMs without work at lengths of 1 to 4096, and
//   every wave of CTAs after the first costs its start and end again.)
// Inside a CTA the stages of a pair go to the warps in turn; a stage is 4608 bytes (at D = 256
// 9216, two tiles, of which one enters negated), or fewer tiles where warps would be left
// without one.  Every warp fills a ring of its own with bulk copies, one per
// run of tiles that lie in a row, and looks the pages up 32 tiles at a time.
//
// What bounds it: the latency of a tile's chain (products, exponentials, products) with 8 to 16
// warps per SM; 55% of the issue slots, 48% of the ALU pipe and 44% of DRAM are used.  64
// sequences x 8 kv heads of 4096 tokens (152 MB of cache, 23.2 us at the measured HBM rate) take
// 39.4 us, 3.9 TB/s; 64 x 8 of 2048 of 128 dims (152 MB) 42.5; 256 x 2 of 2048 of 256 dims (305
// MB, 46.5 us) 75.0 us, 4.1 TB/s.  With a tile's arithmetic left out the rest takes 28.4, 30.1
// and 57.5; with the copies left out the first takes 37.9.  Measured and dropped, at these three:
// stages of half the size 45.2, 45.4 and no change; three stages (fewer CTAs per SM) 48.7, 56.2 and
// 113.8; 5 to 8 CTAs per SM (registers spill); a tile's scores beside the values of the one
// before.  At D = 64 two tiles are taken at a time (one: 40.4), at 128 one (two: 43.6); at 256
// one takes 254 registers.  At 128 four CTAs per SM spill 112 bytes, three with 168 registers
// none: 48.6, though 20.2 against 22.0 for 16 sequences of 1 to 4096.
constexpr int kKv4RunOverhead = 32;
template <int D>
struct Kv4Ring {
  static constexpr int G = D / kKv4Group;
  static constexpr int kTileBytes = G * kKv4CellBytes;
  static constexpr int kTiles = D == 256 ? 2 : 4 / G;  // tiles of a stage at most
  static constexpr int kStages = 2;
  static constexpr int kStageBytes = kTiles * kTileBytes;
  // what a run costs beside its tiles, its start and end, in tiles of a CTA (16 sequences of 1 to
  // 4096 tokens, D = 64: 32 tiles 15.8 us, 16 16.0; D = 128: 16 22.0, 8 23.6 to 23.9, 32 22.1)
  static constexpr int kOverhead = kKv4RunOverhead / G;
};
template <int D, int W>
__host__ __device__ constexpr size_t kv4_decode_smem() {
  return static_cast<size_t>(W) * Kv4Ring<D>::kStages * Kv4Ring<D>::kStageBytes;
}

constexpr int kKv4MaxDealt = 1024;  // sequences of a launch whose tiles are dealt over the grid

// Tiles of sequence b: 0 where it has no token, or (reported by the caller) a bad position.
__device__ __forceinline__ int kv4_seq_tiles(const Kv4DecodeParams& p, int pos, bool& bad) {
  bad = pos < -1 || pos >= static_cast<long long>(p.max_pages) * p.page ||
        (!p.sel && pos >= p.max_len);
  if (bad || pos < 0) return 0;
  return p.sel ? p.n_sel * (p.page / kKv4Tile) : pos / kKv4Tile + 1;
}

// Tiles [t_lo, t_hi) of one pair, as a CTA takes them.
struct Kv4Run {
  int b, kvh, pos, n_tiles, t_lo, t_hi;
  int lg, n_stages;  // tiles of a stage: 1 << lg; this warp's stages
};

template <int D, int W>
__global__ void __launch_bounds__(W * 32, D == 256 ? 2 : 4) kv4_decode_kernel(const Kv4DecodeParams p,
                                                                             const __grid_constant__ Kv4Rope rope) {
  using Ring = Kv4Ring<D>;
  constexpr int G = D / kKv4Group, ST = Ring::kTiles, NS = Ring::kStages, NT = D == 64 ? 2 : 1;
  constexpr int kBehind = 32;
  constexpr int kPush = kKv4MaxGroup * D + 16;  // floats of a cluster's o that one CTA joins, over all CTAs
  constexpr int kArea = kPush + 2 * 16 * kKv4MaxGroup > kKv4MaxDealt + 1 ? kPush + 2 * 16 * kKv4MaxGroup : kKv4MaxDealt + 1;
  extern __shared__ __align__(128) uint8_t rings[];
  __shared__ Kv4Query<D> Q;
  __shared__ __align__(8) uint64_t full[W][NS];
  __shared__ int left_s[W][NS][ST];
  __shared__ float mr[W][kKv4MaxGroup], ml[W][kKv4MaxGroup];
  __shared__ float times_s[W][G][kKv4MaxGroup];  // D > 64: what a group's weights in o and m are multiplied by
  __shared__ int area[kArea];  // dealt: weights of the sequences below; cluster: what the CTAs push
  __shared__ int abort_flag, scan[W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, c = lane & 3;
  const int grp = p.hq / p.hkv, tpp = p.page / kKv4Tile;
  const size_t head_bytes = static_cast<size_t>(tpp) * Ring::kTileBytes;
  const uint64_t once = l2_evict_first_policy();
  uint8_t* const ring = rings + static_cast<size_t>(warp) * NS * Ring::kStageBytes;
  const uint32_t bar0 = smem_u32(&full[warp][0]), ring_s = smem_u32(ring);
  int in_slot = 0, slot = 0;
  uint32_t parity = 0;

  if (lane < NS) mbar_init(bar0 + lane * 8, 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  if (p.splits > 1) cluster_arrive_relaxed();  // waited for before anything is pushed
  pdl_wait();
  pdl_launch_dependents();
  __syncwarp();

  // ---- this CTA's tiles: its split of one pair, or its share of all
  Kv4Run run;
  Kv4RawQuery<D, W> raw;
  int* const before = area;  // dealt: before[b] = weight of a kv head's pairs below sequence b
  int u = 0, u1 = 0;         // dealt: the CTA's share, in weights of pairs: overhead, then tiles
  if (p.splits) {
    run.kvh = blockIdx.x / p.splits;
    run.b = blockIdx.y;
    kv4_load_query<D, W>(p, run.b, run.kvh, raw);
    run.pos = p.pos[run.b];
    bool bad;
    run.n_tiles = kv4_seq_tiles(p, run.pos, bad);
    if (bad) {
      if (threadIdx.x == 0) record_error(kDevBadPosition);
      if (p.splits > 1) cluster_wait_acquire();
      return;  // the whole cluster: nothing is read or written
    }
    const int split = blockIdx.x % p.splits;
    run.t_lo = static_cast<int>(static_cast<long long>(run.n_tiles) * split / p.splits);
    run.t_hi = static_cast<int>(static_cast<long long>(run.n_tiles) * (split + 1) / p.splits);
  } else {
    int sum = 0;
    for (int b0 = 0; b0 < p.batch; b0 += W * 32) {
      const int i = b0 + threadIdx.x;
      bool bad = false;
      const int tiles = i < p.batch ? kv4_seq_tiles(p, p.pos[i], bad) : 0;
      // a sequence without tiles: its rows become zeros, but for a bad position
      if (i < p.batch && tiles == 0 && i % gridDim.x == blockIdx.x) {
        if (bad) record_error(kDevBadPosition);
        for (int h = 0; h < p.hkv; ++h) p.spans[static_cast<size_t>(i) * p.hkv + h] = make_int2(bad ? -1 : -2, 0);
      }
      const int mine = tiles ? tiles + Ring::kOverhead : 0;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      int below = sum;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < warp) below += scan[w];
        sum += scan[w];
      }
      if (i < p.batch) before[i] = below + incl - mine;
      if (b0 + W * 32 < p.batch) __syncthreads();
    }
    if (threadIdx.x == 0) before[p.batch] = sum;
    __syncthreads();
    const int total = sum * p.hkv;  // below 2^30
    const int n_cta = min(total, static_cast<int>(gridDim.x));
    if (static_cast<int>(blockIdx.x) >= n_cta) return;
    // the share's ends: equal parts of all weights, but a pair's own end where that is within 3%
    // of a part, so that pairs of nearly one length are not cut in a piece and a crumb
    const int each = total / n_cta, rest = total - each * n_cta, me = blockIdx.x;
    auto edge = [&](int i, int& b) -> int {
      const int at = each * i + min(i, rest);
      b = 0;
      if (i == n_cta) return total;
      int hi = p.batch;  // the last sequence that begins at or below `at`, and has tiles
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (before[mid] * p.hkv <= at) b = mid;
        else hi = mid;
      }
      const int weight = before[b + 1] - before[b], in = (at - before[b] * p.hkv) % weight;
      return in <= each / 32 ? at - in : weight - in <= each / 32 ? at + weight - in : at;
    };
    int b;
    u1 = edge(me + 1, b);
    u = edge(me, b);
    if (u >= u1) return;
    // (an end moved up may be the next sequence's beginning: next() steps on to it)
    run.b = b;
    run.kvh = min((u - before[b] * p.hkv) / (before[b + 1] - before[b]), p.hkv - 1);
  }
  // dealt: the next pair of the share that has tiles in it; false behind the last.  A share may
  // end inside a pair's overhead, which leaves it none of the tiles.
  auto next = [&]() -> bool {
    while (u < u1) {
      const int weight = before[run.b + 1] - before[run.b];
      const int in = u - before[run.b] * p.hkv - run.kvh * weight;
      if (in >= weight) {  // on to the next pair
        if (++run.kvh == p.hkv) {
          run.kvh = 0;
          do ++run.b;
          while (before[run.b + 1] == before[run.b]);
        }
        continue;
      }
      const int out = min(weight, in + (u1 - u));
      u += out - in;
      run.n_tiles = weight - Ring::kOverhead;
      run.t_lo = max(0, in - Ring::kOverhead);
      run.t_hi = max(0, out - Ring::kOverhead);
      if (run.t_hi > run.t_lo) return true;
    }
    return false;
  };
  // lane's tile of the 32 that begin with the warp's i0-th: its address, how much of it counts
  auto find = [&](int i0, int& left) -> const uint8_t* {
    const int i = i0 + lane;
    left = 0;
    if (i >= run.n_stages << run.lg) return nullptr;
    const int tile = run.t_lo + ((warp + (i >> run.lg) * W) << run.lg) + (i & ((1 << run.lg) - 1));
    if (tile >= run.t_hi) return nullptr;
    int pg = tile / tpp;
    const int in_page = tile - pg * tpp;
    if (p.sel) {  // an entry that does not rise above the one before it counts for nothing
      const int* sel = p.sel + (static_cast<size_t>(run.b) * p.hkv + run.kvh) * p.n_sel + pg;
      const int low = pg > 0 ? sel[-1] : -1;
      pg = *sel;
      if (pg < 0 || pg >= p.max_pages || pg <= low) return nullptr;
    }
    const long long first = static_cast<long long>(pg) * p.page + in_page * kKv4Tile;
    if (first > run.pos) return nullptr;
    const int id = p.table[static_cast<size_t>(run.b) * p.max_pages + pg];
    if (id < 0 || id >= p.n_pages) {
      record_error(kDevBadPosition);
      return nullptr;
    }
    left = static_cast<int>(min(static_cast<long long>(kKv4Tile), run.pos + 1 - first));
    if (in_page && i & ((1 << run.lg) - 1)) left |= kBehind;
    return p.pool + (static_cast<size_t>(id) * p.hkv + run.kvh) * head_bytes + static_cast<size_t>(in_page) * Ring::kTileBytes;
  };
  // (kBehind: the tile lies behind the lane below's in memory and in its stage)
  int left_now, left_next = 0;
  const uint8_t *at_now, *at_next;
  // of the 32 tiles at hand: those with tokens, those full; this lane's copy: the tiles that lie
  // in a row from its own on, as far as its stage goes
  unsigned some, full_tiles;
  int copy_bytes;
  auto survey = [&]() {
    some = __ballot_sync(0xffffffffu, left_now > 0);
    full_tiles = __ballot_sync(0xffffffffu, (left_now & ~kBehind) == kKv4Tile);
    const unsigned first = __ballot_sync(0xffffffffu, left_now > 0 && !(left_now & kBehind));
    const int row = __ffs(static_cast<int>(~((some & ~first) >> lane >> 1)));
    copy_bytes = first >> lane & 1 ? row * Ring::kTileBytes : 0;
  };
  // the run's first lookups and query on their way (cluster: the query is already)
  auto begin = [&]() {
    run.lg = 0;
    while ((2 << run.lg) <= ST && ((run.t_hi - run.t_lo) >> run.lg) > W) ++run.lg;
    run.n_stages = max(0, (((run.t_hi - run.t_lo + (1 << run.lg) - 1) >> run.lg) - warp + W - 1) / W);
    at_now = find(0, left_now);
    at_next = run.n_stages << run.lg > 32 ? find(32, left_next) : nullptr;
  };
  if (!p.splits) {
    if (!next()) return;
    kv4_load_query<D, W>(p, run.b, run.kvh, raw);
    run.pos = p.pos[run.b];
  }
  begin();

  while (true) {
    // ---- the run's first stages, then the query while they are on their way
    int issued = 0;
    unsigned whole = 0;  // bit s: every tile of the stage in slot s is there and full
    auto issue = [&]() {  // the next stage into slot `in_slot`: the lanes that hold its tiles copy them
      const int i = issued << run.lg, o = i & 31;
      if (o == 0) {
        if (i > 0) {
          at_now = at_next;
          left_now = left_next;
          if (i + 32 < run.n_stages << run.lg) at_next = find(i + 32, left_next);
        }
        survey();
      }
      const unsigned tiles = (1u << (1 << run.lg)) - 1u;
      const uint32_t bar = bar0 + in_slot * 8, mine = lane - o;
      const bool all = __popc(full_tiles >> o & tiles) == ST;
      whole = (whole & ~(1u << in_slot)) | static_cast<unsigned>(all) << in_slot;
      if (lane == 0) mbar_arrive_expect_tx(bar, __popc(some >> o & tiles) * Ring::kTileBytes);
      __syncwarp();
      if (mine < 1u << run.lg) {
        left_s[warp][in_slot][mine] = left_now & ~kBehind;
        if (copy_bytes)
          bulk_g2s(ring_s + in_slot * Ring::kStageBytes + mine * Ring::kTileBytes, at_now, copy_bytes, bar, once);
      }
      in_slot = in_slot + 1 == NS ? 0 : in_slot + 1;
      ++issued;
    };
    // a stage with fewer tiles than it has room for: the others count for nothing
    if (lane < ST * NS) left_s[warp][lane / ST][lane % ST] = 0;
    __syncwarp();
    while (issued < min(NS, run.n_stages)) issue();
    kv4_prepare_query<D, W>(p, rope, max(run.pos, 0), raw, Q);
    __syncthreads();
    uint32_t qb[G][4][2];
    float qs[G][2], unit[2] = {Q.unit[2 * c], Q.unit[2 * c + 1]};
    Kv4State<D> st;
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qb[g][k][0] = *reinterpret_cast<const uint32_t*>(&Q.b[g][k][0][lane][0]);
        qb[g][k][1] = *reinterpret_cast<const uint32_t*>(&Q.b[g][k][1][lane][0]);
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
    st.r[0] = st.r[1] = kKv4NoScore;
    if (G > 1 && lane < G * kKv4MaxGroup) times_s[warp][lane / kKv4MaxGroup][lane % kKv4MaxGroup] = 1.f;
    __syncwarp();
    bool scaled = false;  // some group's unit is not 1

    int done = 0;
    for (; done < run.n_stages; ++done) {
      const uint32_t bar = bar0 + slot * 8;
      if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
        // a wait that runs out ends this warp's work: the result is void, and reported
        const bool here = mbar_wait_bounded(bar, parity, &abort_flag, kDevTimeoutFull);
        if (!__all_sync(0xffffffffu, here)) break;
      }
      const uint8_t* stage = ring + slot * Ring::kStageBytes;
      int n = 0;
      if (!scaled && whole >> slot & 1) {
#pragma unroll
        for (; n < ST; n += NT)
          if (!kv4_tiles<D, NT, false>(stage + n * Ring::kTileBytes, Ring::kTileBytes, n, nullptr, qb, qs, unit, nullptr,
                                       scaled, st))
            break;
      }
#pragma unroll 1
      for (; n < 1 << run.lg; n += NT)
        scaled = !kv4_tiles<D, NT, true>(stage + n * Ring::kTileBytes, Ring::kTileBytes, n, &left_s[warp][slot][n], qb, qs,
                                         unit, times_s[warp], scaled, st);
      __syncwarp();  // every lane has read the slot
      if (issued < run.n_stages) issue();
      if (++slot == NS) {
        slot = 0;
        parity ^= 1;
      }
    }
    for (; done < issued; ++done) {  // given up: copies in flight land before the ring is used otherwise
      const uint64_t t0 = globaltimer();
      while (!mbar_try_wait(bar0 + slot * 8, parity))
        if (globaltimer() - t0 > B2_WAIT_TIMEOUT_NS) {
          record_error(kDevTimeoutDrain);
          break;
        }
      if (++slot == NS) {
        slot = 0;
        parity ^= 1;
      }
    }

    // ---- the next run's lookups set out before this one's sums are joined
    const int b = run.b, kvh = run.kvh, t_lo = run.t_lo, t_hi = run.t_hi, n_tiles = run.n_tiles;
    const bool more = !p.splits && next();
    if (more) {
      kv4_load_query<D, W>(p, run.b, run.kvh, raw);
      if (run.b != b) run.pos = p.pos[run.b];
      begin();
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
        for (int e = 0; e < 4; ++e) {
          const float sum = i & 1 ? st.o[g][i][e] - st.o[g][i - 1][e] : st.o[g][i][e];
          const float back = G > 1 ? kv4_power_inv(times_s[warp][g][2 * c + (e & 1)]) : 1.f;
          mo[warp][2 * c + (e & 1)][64 * g + 8 * gl + 2 * (e & 2) + i] = fmaf(sum, scale, st.m[g][e & 1]) * back;
        }
      }
    if (p.splits > 1) cluster_wait_acquire();  // the cluster's CTAs have all begun
    __syncthreads();
    const bool alone = p.splits ? p.splits == 1 : t_hi - t_lo == n_tiles;
    const int split = p.splits ? blockIdx.x % p.splits : 0;
    const int share = p.splits ? (grp * D + p.splits - 1) / p.splits : 1;  // outputs that a CTA of the cluster joins
    const uint32_t push_o = smem_u32(area), push_rl = push_o + kPush * 4;
    float* part = p.part + (2 * static_cast<size_t>(blockIdx.x) + (t_lo == 0)) * kv4_part_floats(grp, D);
    for (int e = threadIdx.x; e < grp * D; e += W * 32) {
      const int j = e / D, d = e % D;
      float R = kKv4NoScore, L = 0.f, O = 0.f;
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
      if (alone) {
        kv4_store_out(p, b, kvh * grp + j, D, d, L == 0.f ? 0.f : O / L);
      } else if (p.splits) {
        st_dsmem_f32(push_o + (split * share + e % share) * 4, e / share, O);
        if (d == 0)
          for (int k = 0; k < p.splits; ++k) {
            st_dsmem_f32(push_rl + ((split * kKv4MaxGroup + j) * 2) * 4, k, R);
            st_dsmem_f32(push_rl + ((split * kKv4MaxGroup + j) * 2 + 1) * 4, k, L);
          }
      } else {
        part[e] = O;
        if (d == 0) {
          part[grp * D + j] = R;
          part[grp * D + grp + j] = L;
        }
      }
    }
    if (p.splits) {
      if (alone) return;
      // ---- the cluster: this CTA's share of the outputs from what all have pushed
      cluster_sync_all();
      const float* o = reinterpret_cast<const float*>(area);
      const float* rl = o + kPush;
      for (int i = threadIdx.x; i < share; i += W * 32) {
        const int e = split * share + i, j = e / D;
        if (e >= grp * D) break;
        float R = kKv4NoScore, L = 0.f, O = 0.f;
        for (int k = 0; k < p.splits; ++k)
          if (rl[(k * kKv4MaxGroup + j) * 2 + 1] != 0.f) R = fmaxf(R, rl[(k * kKv4MaxGroup + j) * 2]);
        for (int k = 0; k < p.splits; ++k) {
          const float l = rl[(k * kKv4MaxGroup + j) * 2 + 1];
          if (l == 0.f) continue;
          const float f = kv4_ex2(rl[(k * kKv4MaxGroup + j) * 2] - R);
          L = fmaf(l, f, L);
          O = fmaf(o[k * share + i], f, O);
        }
        kv4_store_out(p, b, kvh * grp + j, D, e % D, L == 0.f ? 0.f : O / L);
      }
      return;
    }
    if (threadIdx.x == 0) {
      int2* span = p.spans + static_cast<size_t>(b) * p.hkv + kvh;
      if (t_lo == 0) span->x = alone ? -1 : static_cast<int>(blockIdx.x);
      if (t_hi == n_tiles) span->y = blockIdx.x;
    }
    if (!more) return;
    fence_proxy_async();  // the rings' bytes go from these threads back to the copies
    __syncthreads();      // the sums in the rings have been read
  }
}

// Joins the pairs that several CTAs share, and clears the rows of sequences without tokens:
// grid (kv head, sequence, share of the heads).  A thread joins four outputs of one head (one
// each, at D = 64: 20.7 us where four took 15.0 for one sequence of 32768); threads beyond the outputs
// take every further part of them (many parts a pair).
// The parts' loads set out together: the kernel is two trips to L2 long.
constexpr int kKv4JoinMost = 512;
template <int D>
__global__ void __launch_bounds__(kKv4JoinMost) kv4_join_kernel(const Kv4DecodeParams p) {
  constexpr int V = 4;
  __shared__ float sh[2 + V][kKv4JoinMost];
  const int kvh = blockIdx.x, b = blockIdx.y, grp = p.hq / p.hkv, tid = threadIdx.x;
  const int heads = grp / gridDim.z, j0 = blockIdx.z * heads, quads = heads * D / V;
  pdl_wait();
  pdl_launch_dependents();
  const int2 span = p.spans[static_cast<size_t>(b) * p.hkv + kvh];
  if (span.x == -1) return;
  const int step = kv4_part_floats(grp, D), n = span.x < 0 ? 0 : span.y - span.x + 1;
  const int slices = blockDim.x / quads;  // 1 where the heads have more outputs than this is 4 of
  const int e = (tid % quads) * V, slice = tid / quads;
  const int at = j0 * D + e, rl = grp * D + j0 + e / D;
  const float* base = p.part + (2 * static_cast<size_t>(max(span.x, 0)) + 1) * step;  // the pair's first part
  float R = kKv4NoScore, L = 0.f, O[V] = {};
  auto add = [&](float r, float l, const float (&o)[V]) {
    if (l == 0.f) return;
    const float m = fmaxf(R, r), f = kv4_ex2(R - m), g = kv4_ex2(r - m);
    R = m;
    L = fmaf(L, f, l * g);
#pragma unroll
    for (int i = 0; i < V; ++i) O[i] = fmaf(O[i], f, o[i] * g);
  };
  for (int k0 = slice; k0 < n; k0 += 4 * slices) {
    float r[4], l[4], o[4][V];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // part k > 0 is the first place of the k-th CTA behind the span's first
      const int k = k0 + i * slices;
      const float* part = base + (k ? static_cast<ptrdiff_t>(2 * k - 1) * step : 0);
      r[i] = k < n ? part[rl] : 0.f;
      l[i] = k < n ? part[rl + grp] : 0.f;
#pragma unroll
      for (int x = 0; x < V; ++x) o[i][x] = k < n ? part[at + x] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) add(r[i], l[i], o[i]);
  }
  if (slices > 1) {
    sh[0][tid] = R;
    sh[1][tid] = L;
#pragma unroll
    for (int i = 0; i < V; ++i) sh[2 + i][tid] = O[i];
    __syncthreads();
    if (slice > 0) return;
    for (int k = 1; k < slices; ++k) {
      const int t = tid + k * quads;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = sh[2 + i][t];
      add(sh[0][t], sh[1][t], o);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    kv4_store_out(p, b, kvh * grp + j0 + e / D, D, e % D + i, L == 0.f ? 0.f : O[i] / L);
}

}  // namespace b2
