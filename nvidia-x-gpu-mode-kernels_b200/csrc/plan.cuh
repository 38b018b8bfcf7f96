// The plan of an operator in which every token picks its own weights: the
// slots (token, choice) are put in order of their index (expert, adapter), each
// index's rows starting at a multiple of `align`, and the row tiles to walk
// are listed.  Everything stays on the GPU: the host never learns the counts.
//
// A slot whose index is not in [0, indexes) goes to the index `other`, or is
// left out where `other` is negative.
//
// One cluster of C CTAs: each counts its share of the slots in shared memory
// (an atomic gives a slot its place among its share's equals), the counts are
// exchanged through distributed shared memory, every CTA scans them, and the
// slots' rows follow.  Which of two slots of one index comes first depends on
// the atomics' order; no result depends on it, since a row's arithmetic does
// not depend on its place.
//
// C = 8 above 4096 slots: counting is bound by the atomics of one SM.
#pragma once
#include <algorithm>
#include "common.h"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

constexpr int kPlanMaxIndexes = 1024;
constexpr int kPlanThreads = 1024;

// One row tile.  All tiles of an index are adjacent in the list, from `first`
// on, so item i of a walk over (index, column tile, row tile), row tiles
// fastest, is found with one division: list[i / column_tiles] names the index.
struct __align__(16) PlanTile {
  int index;     // expert or adapter
  int row0;      // the index's first row
  int first;     // its first tile in the list
  int tiles;     // its number of tiles
  int rows;      // its number of rows
  int pad[3];
};

struct Plan {
  int* head;          // [0] number of tiles
  PlanTile* tiles;
  int* row;           // [slots]: row of each slot, -1 for a slot without an index
  int* slot;          // [rows], or null: the slot of each row, -1 for padding
};

inline int64_t plan_max_tiles(int64_t slots, int64_t indexes, int tile) {
  return slots / tile + std::min(slots, indexes);
}
// Rows of the ordered layout, padding included.
inline int64_t plan_max_rows(int64_t slots, int64_t indexes, int align) {
  return slots + std::min(slots, indexes) * (align - 1);
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int C>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* __restrict__ ids, int n, int indexes,
                                                            int other, int align, int tile, Plan p) {
  __shared__ uint32_t hist[kPlanMaxIndexes];
  __shared__ int start[kPlanMaxIndexes];
  __shared__ int warp_rows[32], warp_tiles[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int me = C > 1 ? (int)cluster_ctarank() : 0;
  griddep_launch();
  hist[tid] = 0;
  __syncthreads();
  const int share = (n + C - 1) / C;
  const int lo = me * share, hi = min(n, lo + share);
  for (int s = lo + tid; s < hi; s += kPlanThreads) {
    int e = ids[s];
    if ((unsigned)e >= (unsigned)indexes) e = other;
    p.row[s] = e >= 0 ? (int)atomicAdd(&hist[e], 1u) : -1;
  }
  if (C > 1) cluster_sync();
  else __syncthreads();
  // thread e: index e
  int before = 0, rows = 0;
  if (C > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int v = (int)ld_cluster_u32(mapa(smem_u32(&hist[tid]), c));
      if (c < me) before += v;
      rows += v;
    }
  } else {
    rows = (int)hist[tid];
  }
  const int span = (rows + align - 1) / align * align, tiles = (rows + tile - 1) / tile;
  int r = span, t = tiles;                       // inclusive scans
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) r += a, t += b;
  }
  if (lane == 31) warp_rows[warp] = r, warp_tiles[warp] = t;
  __syncthreads();
  if (warp == 0) {
    int a = warp_rows[lane], b = warp_tiles[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int c = __shfl_up_sync(0xffffffffu, a, o), d = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) a += c, b += d;
    }
    warp_rows[lane] = a;
    warp_tiles[lane] = b;
  }
  __syncthreads();
  const int row0 = r - span + (warp ? warp_rows[warp - 1] : 0);
  const int first = t - tiles + (warp ? warp_tiles[warp - 1] : 0);
  start[tid] = row0 + before;
  if (me == 0) {
    if (tid == 0) p.head[0] = warp_tiles[31];
    for (int m = 0; m < tiles; ++m) {
      PlanTile q;
      q.index = tid; q.row0 = row0; q.first = first; q.tiles = tiles; q.rows = rows;
      q.pad[0] = q.pad[1] = q.pad[2] = 0;
      p.tiles[first + m] = q;
    }
    if (p.slot)
      for (int i = rows; i < span; ++i) p.slot[row0 + i] = -1;
  }
  __syncthreads();
  for (int s = lo + tid; s < hi; s += kPlanThreads) {
    if (p.row[s] < 0) continue;                  // written by this thread above
    const int e = ids[s];
    const int at = p.row[s] + start[(unsigned)e < (unsigned)indexes ? e : other];
    p.row[s] = at;
    if (p.slot) p.slot[at] = s;
  }
  if (C > 1) cluster_sync();                     // the others have read this CTA's counts
}

inline int launch_plan(const int32_t* ids, int64_t n, int64_t indexes, int other, int align, int tile, const Plan& p,
                       cudaStream_t stream) {
  if (n <= 4096) {
    plan_kernel<1><<<1, kPlanThreads, 0, stream>>>(ids, (int)n, (int)indexes, other, align, tile, p);
    return check_launch("plan_kernel");
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 8;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(8);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, plan_kernel<8>, ids, (int)n, (int)indexes, other, align, tile, p);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "cudaLaunchKernelEx(plan)");
}

// Launches a kernel that may start while its predecessor in the stream drains
// (it waits with griddep_wait before touching the predecessor's memory).
template <typename... Args>
int launch_after(void (*kern)(Args...), const char* name, unsigned grid, unsigned block, size_t smem,
                 cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, name);
}

}  // namespace
}  // namespace nvfp4
