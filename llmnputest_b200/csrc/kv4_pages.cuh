// The pages of the 4-bit KV cache as rows of a page table hold them: forking, freeing,
// reserving (reorder), compacting and copying.  Everything is decided on the device, from
// the reference counts alone: a page is free when no row holds it (refs 0), and of the free
// pages the lowest are given out first, in the order of the rows, so that the outcome does
// not turn on the order in which CTAs run (the counts are whole numbers).
#pragma once

#include "kv4_cell.cuh"

namespace b2 {

// What a page is made of: `rows` arrays (layers) of the pool and of the summaries.
struct Kv4PageData {
  uint8_t* base[2];            // the pool, the summaries (or null)
  unsigned long long bytes[2];  // of one page in one layer, multiples of 16
  int layers, n_pages;
};

// One page of one layer from src to dst, by the whole CTA.
__device__ __forceinline__ void kv4_copy_page(const Kv4PageData& d, int layer, int src, int dst, int part, int parts) {
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    if (!d.base[a]) continue;
    const size_t n = d.bytes[a] / 16;
    const uint4* from = reinterpret_cast<const uint4*>(d.base[a] + (static_cast<size_t>(layer) * d.n_pages + src) * d.bytes[a]);
    uint4* to = reinterpret_cast<uint4*>(d.base[a] + (static_cast<size_t>(layer) * d.n_pages + dst) * d.bytes[a]);
    for (size_t i = static_cast<size_t>(part) * blockDim.x + threadIdx.x; i < n; i += static_cast<size_t>(parts) * blockDim.x)
      to[i] = from[i];
  }
}

constexpr int kKv4CopyThreads = 256;
constexpr int kDevNoPage = 7;  // the pool had no free page left

// Copies of listed pages: grid (parts, layers, pairs).  Entries outside the pool are skipped.
__global__ void __launch_bounds__(kKv4CopyThreads) kv4_copy_kernel(const Kv4PageData d, const int* src, const int* dst) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = src[blockIdx.z], t = dst[blockIdx.z];
  if (s < 0 || t < 0 || s == t) return;
  if (s >= d.n_pages || t >= d.n_pages) {
    if (threadIdx.x == 0) record_error(kDevBadPosition);
    return;
  }
  kv4_copy_page(d, blockIdx.y, s, t, blockIdx.x, gridDim.x);
}

struct Kv4ReorderParams {
  Kv4PageData data;
  const int *table, *lens, *refs, *parent, *reserve;  // reserve may be null
  int *table_out, *lens_out, *refs_out, *info;        // info[4]: free pages left, copied, missing, 0
  int* need;  // [batch] pages each row lacks, then their sums below each row
  int* copy;  // [batch] 0, or 1 + which of the row's missing pages is a copy of its parent's last one
  int* free_ids;  // [total needed] at most batch * max_pages
  int* n_found;   // how many of them there are
  int batch, max_pages, page;
};

constexpr int kKv4ScanThreads = 1024;
constexpr int kKv4PlanThreads = 512, kKv4PlanCtas = 8;

// The new rows' entries and counts, and the lowest free pages in order, by one cluster (one
// grid after another would be three launches and two copies, and the host's time for those is
// what bounds a reorder):
//   the counts copied; a warp per row takes the old row's holds back, the new one's up and
//   counts what it lacks; every CTA counts the free pages of its share of the pool; then lists
//   as many of them, from the lowest on, as all rows lack.
__global__ void __launch_bounds__(kKv4PlanThreads) __cluster_dims__(kKv4PlanCtas, 1, 1)
    kv4_reorder_plan_kernel(const Kv4ReorderParams p) {
  constexpr int W = kKv4PlanThreads / 32;
  __shared__ int warps[32], free_s[kKv4PlanCtas];
  const int rank = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_pages = p.data.n_pages;
  pdl_wait();
  pdl_launch_dependents();
  for (int i = rank * kKv4PlanThreads + tid; i < n_pages; i += kKv4PlanCtas * kKv4PlanThreads) p.refs_out[i] = p.refs[i];
  if (rank == 0 && tid < 4) p.info[tid] = 0;
  cluster_sync_all();

  for (int b = rank * W + warp; b < p.batch; b += kKv4PlanCtas * W) {
    int par = p.parent[b];
    if (par < -1 || par >= p.batch) {
      if (lane == 0) record_error(kDevBadPosition);
      par = -1;
    }
    bool taken = false;  // an earlier row goes on with the same one
    if (par >= 0)
      for (int i = lane; i < b; i += 32) taken |= p.parent[i] == par;
    const bool first = !__any_sync(0xffffffffu, taken);
    const int len = par >= 0 ? max(p.lens[par], 0) : 0;
    const int full = len / p.page;
    const long long tokens = static_cast<long long>(len) + (p.reserve ? max(p.reserve[b], 0) : 0);
    const long long want = (tokens + p.page - 1) / p.page;
    const int* mine = p.table + static_cast<size_t>(b) * p.max_pages;
    const int* theirs = p.table + static_cast<size_t>(max(par, 0)) * p.max_pages;
    int* out = p.table_out + static_cast<size_t>(b) * p.max_pages;
    int lack = 0, below = 0;
    for (int j = lane; j < p.max_pages; j += 32) {
      const int old = mine[j];
      int id = par >= 0 && (first || j < full) ? theirs[j] : -1;
      if (id < 0 || id >= n_pages) id = -1;
      if (old != id) {  // a row that goes on as it was changes no count
        if (old >= 0 && old < n_pages) atomicSub(&p.refs_out[old], 1);
        if (id >= 0) atomicAdd(&p.refs_out[id], 1);
      }
      out[j] = id;
      lack += id < 0 && j < want;
      below += id < 0 && j < full;
    }
    lack = __reduce_add_sync(0xffffffffu, lack);
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) {
      p.need[b] = lack;
      const bool copies = par >= 0 && !first && len % p.page != 0 && full < p.max_pages && theirs[full] >= 0 &&
                          theirs[full] < n_pages;
      p.copy[b] = copies ? 1 + below : 0;
      p.lens_out[b] = len;
      if (want > p.max_pages) {
        record_error(kDevNoPage);
        atomicAdd(&p.info[2], static_cast<int>(min(want - p.max_pages, 0x7FFFFFFFll)));
      }
    }
  }
  cluster_sync_all();

  // free pages of this CTA's share; the rows' needs in all (read past L1: others wrote them)
  const int share = (n_pages + kKv4PlanCtas - 1) / kKv4PlanCtas;
  const int lo = min(n_pages, rank * share), hi = min(n_pages, lo + share);
  int mine = 0, free_here, total = 0;
  for (int i = lo + tid; i < hi; i += kKv4PlanThreads) mine += __ldcg(&p.refs_out[i]) == 0;
  kv4_block_before(mine, warps, free_here);
  for (int b0 = 0; b0 < p.batch; b0 += kKv4PlanThreads) {
    const int b = b0 + tid, v = b < p.batch ? __ldcg(&p.need[b]) : 0;
    int sum;
    kv4_block_before(v, warps, sum);
    total += sum;
  }
  if (tid < kKv4PlanCtas) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&free_s[rank])), "r"(tid));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(free_here) : "memory");
  }
  cluster_sync_all();
  int found = 0, all = 0;
  for (int k = 0; k < kKv4PlanCtas; ++k) {
    if (k < rank) found += free_s[k];
    all += free_s[k];
  }
  for (int i0 = lo; i0 < hi && found < total; i0 += kKv4PlanThreads) {
    const int i = i0 + tid;
    const int is_free = i < hi && __ldcg(&p.refs_out[i]) == 0;
    int sum;
    const int at = found + kv4_block_before(is_free, warps, sum);
    if (is_free && at < total) {
      p.free_ids[at] = i;
      p.refs_out[i] = 1;
    }
    found += sum;
  }
  if (rank == 0) {  // every CTA has summed the needs: they become the sums below each row
    int below = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kKv4PlanThreads) {
      const int b = b0 + tid, v = b < p.batch ? __ldcg(&p.need[b]) : 0;
      int sum;
      const int before = kv4_block_before(v, warps, sum);
      if (b < p.batch) p.need[b] = below + before;
      below += sum;
    }
    if (tid == 0) {
      *p.n_found = min(all, total);
      p.info[0] = all - min(all, total);
      if (all < total) {
        record_error(kDevNoPage);
        atomicAdd(&p.info[2], total - all);
      }
    }
  }
}

// Row blockIdx.y's missing pages filled in (CTAs of layer 0, part 0) and its parent's last
// page copied: grid (parts, batch, layers).
__global__ void __launch_bounds__(kKv4CopyThreads) kv4_reorder_fill_kernel(const Kv4ReorderParams p) {
  __shared__ int warps[32];
  const int b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int found = *p.n_found, rank0 = p.need[b];
  const int par = p.parent[b];
  const int copy_rank = rank0 + p.copy[b] - 1;
  const bool copies = p.copy[b] != 0;
  if (blockIdx.x == 0 && layer == 0) {
    int* out = p.table_out + static_cast<size_t>(b) * p.max_pages;
    const int len = p.lens_out[b];
    const long long want = (static_cast<long long>(len) + (p.reserve ? max(p.reserve[b], 0) : 0) + p.page - 1) / p.page;
    const int end = static_cast<int>(min(want, static_cast<long long>(p.max_pages)));
    int rank = rank0;
    for (int j0 = 0; j0 < end; j0 += kKv4CopyThreads) {
      const int j = j0 + tid;
      const int hole = j < end && out[j] < 0;
      int sum;
      const int at = rank + kv4_block_before(hole, warps, sum);
      if (hole && at < found) out[j] = p.free_ids[at];
      rank += sum;
    }
    __syncthreads();
    if (tid == 0 && copies) {
      if (copy_rank >= found) p.lens_out[b] = len / p.page * p.page;  // its last page could not be had
      else atomicAdd(&p.info[1], 1);
    }
  }
  if (!copies || copy_rank >= found) return;
  const int src = p.table[static_cast<size_t>(par) * p.max_pages + p.lens[par] / p.page];
  kv4_copy_page(p.data, layer, src, p.free_ids[copy_rank], blockIdx.x, gridDim.x);
}

struct Kv4CompactParams {
  Kv4PageData data;
  const int *table, *refs;
  int *table_out, *refs_out, *info;  // info[4]: live pages, pages moved, 0, 0
  int *to;         // [n_pages] where each live page goes
  int *src, *dst;  // [n_pages] the moves
  int batch, max_pages;
};

// One CTA: live pages counted, then the k-th free page below their number takes the k-th
// live page at or above it.
__global__ void __launch_bounds__(kKv4ScanThreads) kv4_compact_plan_kernel(const Kv4CompactParams p) {
  __shared__ int warps[32];
  const int tid = threadIdx.x, n = p.data.n_pages;
  pdl_wait();
  pdl_launch_dependents();
  int mine = 0, live;
  for (int i = tid; i < n; i += kKv4ScanThreads) mine += p.refs[i] > 0;
  kv4_block_before(mine, warps, live);
  int holes = 0, moves = 0;
  for (int i0 = 0; i0 < n; i0 += kKv4ScanThreads) {
    const int i = i0 + tid;
    const bool on = i < n && p.refs[i] > 0;
    const bool hole = i < n && i < live && !on, move = on && i >= live;
    int sum;
    const int h = holes + kv4_block_before(hole, warps, sum);
    holes += sum;
    const int m = moves + kv4_block_before(move, warps, sum);
    moves += sum;
    if (hole) p.dst[h] = i;
    if (move) p.src[m] = i;
    if (i < n) {
      p.to[i] = on && i < live ? i : -1;
      p.refs_out[i] = on && i < live ? p.refs[i] : 0;
    }
  }
  __syncthreads();  // one CTA: its own global writes above are visible to it
  for (int k = tid; k < moves; k += kKv4ScanThreads) {
    p.to[p.src[k]] = p.dst[k];
    p.refs_out[p.dst[k]] = p.refs[p.src[k]];
  }
  if (tid == 0) {
    p.info[0] = live;
    p.info[1] = moves;
    p.info[2] = p.info[3] = 0;
  }
}

// The table's entries and the pages' bytes: CTAs share the entries, then the (move, layer) pairs.
__global__ void __launch_bounds__(kKv4CopyThreads) kv4_compact_move_kernel(const Kv4CompactParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const size_t n = static_cast<size_t>(p.batch) * p.max_pages;
  for (size_t i = static_cast<size_t>(blockIdx.x) * kKv4CopyThreads + threadIdx.x; i < n;
       i += static_cast<size_t>(gridDim.x) * kKv4CopyThreads) {
    const int id = p.table[i];
    p.table_out[i] = id >= 0 && id < p.data.n_pages ? p.to[id] : -1;
  }
  const long long work = static_cast<long long>(p.info[1]) * p.data.layers;
  for (long long w = blockIdx.x; w < work; w += gridDim.x) {
    const int k = static_cast<int>(w / p.data.layers);
    kv4_copy_page(p.data, static_cast<int>(w % p.data.layers), p.src[k], p.dst[k], 0, 1);
  }
}

}  // namespace b2
