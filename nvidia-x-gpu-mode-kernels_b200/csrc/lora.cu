// Low-rank adapters of many requests, added to a shared projection's output:
//
//   out[t] = fp16( base[t] + scale_i * ((x[t] . A_i^T) . B_i^T) ),   i = adapters[t]
//
// A_i [r, K], B_i [N, r] (fp16), of which adapter i uses its first ranks[i] rows / columns.  Tokens without
// an adapter (an index outside [0, n)) keep base.  Bytes bound both forms: x, base and out once, and the
// matrices of the adapters in use.
//
// The products run on mma.sync (fp16 operands, fp32 accumulators): with ranks of 16 to 128 there is too
// little arithmetic per byte for tensor memory and its round trips to pay.  u = x . A^T enters the second
// product as two fp16 halves, u = 2^-p (hi + lo), 2^p bringing the token's largest |u| to 2^14: 22 bits of
// u survive, whatever its range, and the sum stays in fp32.
//
// The k index of an mma is summed over, so its 16 slots may stand for any 16 elements as long as both operands
// agree.  Slots {2q, 2q+1, 2q+8, 2q+9} of lane quarter q stand for 4 consecutive elements: fragments are loaded
// from memory as they lie there, 8 or 16 bytes a lane, without shared memory.
//
// Few tokens (decode_kernel): one launch.  A cluster of 8 CTAs takes up to 8 tokens of one adapter: each
// CTA sums an eighth of K for all ranks, the partial u's are exchanged through distributed shared memory and each
// CTA writes an eighth of N.  B is prefetched into L2 at the start, so both matrices stream at once.
//
// Many tokens: the plan (plan.cuh) orders them by adapter; shrink_kernel computes u, expand_kernel adds u . B^T.
#include <cuda_fp16.h>
#include <algorithm>
#include <cstring>
#include "common.h"
#include "plan.cuh"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

constexpr int kLoraMaxRank = 128;
constexpr int kLoraMaxAdapters = kPlanMaxIndexes - 1;   // one index of the plan is for tokens without an adapter

struct LoraArgs {
  const __half* base;
  const __half* x;
  const __half* a;
  const __half* b;
  const int32_t* adapters;
  const float* scales;       // or null: 1
  const int32_t* ranks;      // or null: r
  __half* out;
  int64_t ld_base, ldx, lda, a_stride, ldb, b_stride, ldo;   // elements
  int T, K, N, r, n;
  int vec;                   // base and out rows 16-byte aligned
  int in_place;              // out is base
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int lora_rank(const LoraArgs& p, int i) {
  if (i < 0) return 0;
  return p.ranks ? max(0, min(p.ranks[i], p.r)) : p.r;
}

// The power of two that brings magnitude m to [2^14, 2^15), and its inverse.
__device__ __forceinline__ void half_scale(float m, float& up, float& down) {
  int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
  if (m == 0.f || e == 128) e = 14;                      // nothing to bring up, or infinite already
  const int q = min(14 - e, 126);
  up = __uint_as_float((uint32_t)(q + 127) << 23);
  down = __uint_as_float((uint32_t)(127 - q) << 23);
}

__device__ __forceinline__ void split_halves(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// Four consecutive halves of a row of B from element k on, zeros from element `rank` on (which may hold anything).
__device__ __forceinline__ uint2 load_b(const __half* row, int k, int rank) {
  uint2 v = *reinterpret_cast<const uint2*>(row + k);
  if (k + 4 > rank) {
    if (k + 3 >= rank) v.y &= 0x0000ffffu;
    if (k + 2 >= rank) v.y = 0;
    if (k + 1 >= rank) v.x &= 0x0000ffffu;
    if (k >= rank) v.x = 0;
  }
  return v;
}

// out[8 columns] = base + d, vectorised where the rows allow it.
__device__ __forceinline__ void add_eight(const LoraArgs& p, int64_t t, int col, const float (&d)[8]) {
  const __half* src = p.base + t * p.ld_base + col;
  __half* dst = p.out + t * p.ldo + col;
  if (p.vec && col + 8 <= p.N) {
    const uint4 v = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      const __half2 h = __floats2half2_rn(f.x + d[2 * j], f.y + d[2 * j + 1]);
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < p.N) dst[j] = __float2half_rn(__half2float(src[j]) + d[j]);
  }
}

// ------------------------------------------------------------------ few tokens

constexpr int kCluster = 8;
constexpr int kDecodeWarps = 8;

// RT: 16-row tiles of the largest rank.
template <int RT>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kDecodeWarps * 32) decode_kernel(const LoraArgs p) {
  constexpr int R = RT * 16;
  __shared__ float part[kDecodeWarps][R][8];             // each warp's share of K; later the warps' output patches
  __shared__ float mine[R][8];                           // this CTA's share of K
  __shared__ __align__(16) __half hi[8][R + 8], lo[8][R + 8];
  __shared__ float down[8];
  __shared__ int tok[8];
  __shared__ int ntok;
  static_assert(sizeof(part) >= kDecodeWarps * 8 * 68 * 4 || RT < 8, "patch");
  __shared__ float patch_small[RT < 8 ? kDecodeWarps * 8 * 68 : 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int rank_in_cluster = (int)cluster_ctarank();
  const int t0 = (int)(blockIdx.x / kCluster);
  int i = p.adapters[t0];
  if ((unsigned)i >= (unsigned)p.n) i = -1;
  const int groups = (p.N + 63) / 64;                    // 64 columns per warp and step
  const int glo = groups * rank_in_cluster / kCluster, ghi = groups * (rank_in_cluster + 1) / kCluster;
  if (i < 0) {                                           // the whole cluster leaves together
    if (!p.in_place)
      for (int c = glo * 64 + tid; c < min(p.N, ghi * 64); c += blockDim.x)
        p.out[t0 * p.ldo + c] = p.base[t0 * p.ld_base + c];
    return;
  }
  // Tokens of one adapter go in eights, in token order; the first of an eight takes it.
  int before = 0;
  for (int s0 = 0; s0 < t0; s0 += blockDim.x) before += __syncthreads_count(s0 + tid < t0 && p.adapters[s0 + tid] == i);
  if (before % 8) return;
  if (warp == 0) {
    if (lane < 8) tok[lane] = -1;
    __syncwarp();
    int found = 0;
    for (int s0 = t0; s0 < p.T && found < 8; s0 += 32) {
      const bool hit = s0 + lane < p.T && p.adapters[s0 + lane] == i;
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      const int at = found + __popc(hits & ((1u << lane) - 1));
      if (hit && at < 8) tok[at] = s0 + lane;
      found += __popc(hits);
    }
    if (lane == 0) ntok = min(found, 8);
  }
  const int rank = lora_rank(p, i);
  const int steps_r = (rank + 15) / 16;
  const __half* A = p.a + i * p.a_stride;
  const __half* B = p.b + i * p.b_stride;
  {
    // B's rows of this CTA, on their way into L2 while A streams
    const int n0 = glo * 64, n1 = min(p.N, ghi * 64);
    const char* lo_b = reinterpret_cast<const char*>(B + n0 * p.ldb);
    const int64_t bytes = n1 > n0 ? ((int64_t)(n1 - 1 - n0) * p.ldb + rank) * 2 : 0;
    for (int64_t o = (int64_t)tid * 128; o < bytes; o += (int64_t)blockDim.x * 128)
      asm volatile("prefetch.global.L2 [%0];" :: "l"(lo_b + o));
  }
  __syncthreads();
  // ---- u = x . A^T over this CTA's share of K: ranks are the mma's rows, tokens its columns
  {
    float acc[RT][4] = {};
    const int ksteps = (p.K + 31) / 32;
    const int klo = ksteps * rank_in_cluster / kCluster, khi = ksteps * (rank_in_cluster + 1) / kCluster;
    const __half* xr = g < ntok ? p.x + (int64_t)tok[g] * p.ldx : nullptr;
    for (int ks = klo + warp; ks < khi; ks += kDecodeWarps) {
      const int k = ks * 32 + q * 8;
      const bool in = k < p.K;                           // K is a multiple of 8
      uint4 xv = make_uint4(0, 0, 0, 0);
      if (xr && in) xv = *reinterpret_cast<const uint4*>(xr + k);
      uint4 av[RT][2];
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = m * 16 + h * 8 + g;
          av[m][h] = make_uint4(0, 0, 0, 0);
          if (row < rank && in) av[m][h] = *reinterpret_cast<const uint4*>(A + row * p.lda + k);
        }
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        mma_16816(acc[m], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv.x, xv.y);
        mma_16816(acc[m], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv.z, xv.w);
      }
    }
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      *reinterpret_cast<float2*>(&part[warp][m * 16 + g][2 * q]) = make_float2(acc[m][0], acc[m][1]);
      *reinterpret_cast<float2*>(&part[warp][m * 16 + g + 8][2 * q]) = make_float2(acc[m][2], acc[m][3]);
    }
  }
  __syncthreads();
  for (int e = tid; e < R * 8; e += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) s += part[w][e >> 3][e & 7];
    mine[e >> 3][e & 7] = s;
  }
  cluster_sync();
  // every CTA adds all shares in the same order: the same u everywhere
  {
    const float scale = p.scales ? p.scales[i] : 1.f;
    float* u = &part[0][0][0];
    for (int e = tid; e < R * 8; e += blockDim.x) {
      const uint32_t here = smem_u32(&mine[e >> 3][e & 7]);
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < kCluster; ++c) s += __uint_as_float(ld_cluster_u32(mapa(here, c)));
      u[e] = s * scale;
    }
    __syncthreads();
    // warp w: token w
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < R; e += 32)
      if (e + lane < R) m = fmaxf(m, fabsf(u[(e + lane) * 8 + warp]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float up, dn;
    half_scale(m, up, dn);
#pragma unroll
    for (int e = 0; e < R; e += 32)
      if (e + lane < R) split_halves(u[(e + lane) * 8 + warp] * up, hi[warp][e + lane], lo[warp][e + lane]);
    if (lane == 0) down[warp] = dn;
  }
  cluster_sync();      // also: nobody leaves while its share is being read
  // ---- out += u . B^T over this CTA's share of N: columns are the mma's rows, tokens its columns
  uint32_t uh[RT][2], ul[RT][2];
#pragma unroll
  for (int s = 0; s < RT; ++s) {
    const uint2 h = *reinterpret_cast<const uint2*>(&hi[g][s * 16 + 4 * q]);
    const uint2 l = *reinterpret_cast<const uint2*>(&lo[g][s * 16 + 4 * q]);
    uh[s][0] = h.x; uh[s][1] = h.y;
    ul[s][0] = l.x; ul[s][1] = l.y;
  }
  float* patch = (RT < 8 ? patch_small : &part[0][0][0]) + warp * 8 * 68;
  for (int gr = glo + warp; gr < ghi; gr += kDecodeWarps) {
    const int n0 = gr * 64;
    float acc[4][4] = {};
#pragma unroll
    for (int s = 0; s < RT; ++s) {
      if (s >= steps_r) break;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int r0 = n0 + m * 16 + g, r1 = r0 + 8;
        uint2 b0 = make_uint2(0, 0), b1 = make_uint2(0, 0);
        if (r0 < p.N) b0 = load_b(B + r0 * p.ldb, s * 16 + 4 * q, rank);
        if (r1 < p.N) b1 = load_b(B + r1 * p.ldb, s * 16 + 4 * q, rank);
        mma_16816(acc[m], b0.x, b1.x, b0.y, b1.y, uh[s][0], uh[s][1]);
        mma_16816(acc[m], b0.x, b1.x, b0.y, b1.y, ul[s][0], ul[s][1]);
      }
    }
    // [token][column] patch, so that lanes write runs of a token's columns
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      patch[(2 * q) * 68 + m * 16 + g] = acc[m][0];
      patch[(2 * q + 1) * 68 + m * 16 + g] = acc[m][1];
      patch[(2 * q) * 68 + m * 16 + g + 8] = acc[m][2];
      patch[(2 * q + 1) * 68 + m * 16 + g + 8] = acc[m][3];
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = h * 4 + (lane >> 3), c = (lane & 7) * 8;
      if (j < ntok && n0 + c < p.N) {
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = patch[j * 68 + c + e] * down[j];
        add_eight(p, tok[j], n0 + c, d);
      }
    }
    __syncwarp();
  }
}

// ------------------------------------------------------------------ many tokens

constexpr int kTile = 64;                // tokens per tile of the plan
constexpr int kShrinkTokens = 32;        // tokens per CTA of the first product
constexpr int kShrinkWarps = 8;
constexpr int kExpandWarps = 8;

struct LoraRows {
  const int* ntiles;
  const PlanTile* tiles;
  const int* slot;                       // token of each row, -1 for padding
  __half* hi;                            // [rows][R], R = r rounded up to 16, 32, 64, 128
  __half* lo;
  float* down;                           // [rows]
};

// u of 32 tokens of one adapter: tokens are the mma's rows, ranks its columns; the warps share K.
template <int RT>
__global__ void __launch_bounds__(kShrinkWarps * 32) shrink_kernel(const LoraArgs p, const LoraRows w) {
  constexpr int R = RT * 16, NT = RT * 2;
  extern __shared__ __align__(16) float part[];          // [warps][32 tokens][R]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  griddep_launch();
  griddep_wait();
  const int total = *w.ntiles * (kTile / kShrinkTokens);
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const PlanTile tile = w.tiles[item / 2];
    const int tr = (item / 2 - tile.first) * kTile + (item & 1) * kShrinkTokens;   // first token within the adapter
    if (tile.index >= p.n || tr >= tile.rows) continue;
    const int row0 = tile.row0 + tr;
    const int rank = lora_rank(p, tile.index);
    const __half* A = p.a + tile.index * p.a_stride;
    const __half* xr[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int s = w.slot[row0 + m * 8 + g];
      xr[m] = s >= 0 ? p.x + (int64_t)s * p.ldx : nullptr;
    }
    float acc[2][NT][4] = {};
    for (int k0 = warp * 32; k0 < p.K; k0 += kShrinkWarps * 32) {
      const int k = k0 + q * 8;
      const bool in = k < p.K;
      uint4 xv[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        xv[m] = make_uint4(0, 0, 0, 0);
        if (xr[m] && in) xv[m] = *reinterpret_cast<const uint4*>(xr[m] + k);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 av = make_uint4(0, 0, 0, 0);
        if (nt * 8 + g < rank && in) av = *reinterpret_cast<const uint4*>(A + (nt * 8 + g) * p.lda + k);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma_16816(acc[m][nt], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av.x, av.y);
          mma_16816(acc[m][nt], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av.z, av.w);
        }
      }
    }
    __syncthreads();                                     // the previous item's sums are read
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* at = part + (warp * kShrinkTokens + m * 16 + g) * R + nt * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[m][nt][0], acc[m][nt][1]);
        *reinterpret_cast<float2*>(at + 8 * R) = make_float2(acc[m][nt][2], acc[m][nt][3]);
      }
    __syncthreads();
    const float scale = p.scales ? p.scales[tile.index] : 1.f;
    for (int t = warp; t < kShrinkTokens; t += kShrinkWarps) {
      float u[(R + 31) / 32];
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < (R + 31) / 32; ++e) {
        u[e] = 0.f;
        if (e * 32 + lane < R) {
#pragma unroll
          for (int v = 0; v < kShrinkWarps; ++v) u[e] += part[(v * kShrinkTokens + t) * R + e * 32 + lane];
        }
        u[e] *= scale;
        m = fmaxf(m, fabsf(u[e]));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float up, dn;
      half_scale(m, up, dn);
      const int64_t row = row0 + t;
#pragma unroll
      for (int e = 0; e < (R + 31) / 32; ++e)
        if (e * 32 + lane < R) {
          __half h, l;
          split_halves(u[e] * up, h, l);
          w.hi[row * R + e * 32 + lane] = h;
          w.lo[row * R + e * 32 + lane] = l;
        }
      if (lane == 0) w.down[row] = dn;
    }
  }
}

// out += u . B^T for 64 tokens of one adapter and a run of columns: a warp takes 64 tokens x 32 columns at a time.
// The 8 columns of mma tile j stand for columns 8 (c / 2) + 2 j + c % 2 of the 32, so that the four tiles give
// a lane 8 consecutive columns of a token.
template <int RT>
__global__ void __launch_bounds__(kExpandWarps * 32) expand_kernel(const LoraArgs p, const LoraRows w, int nsplit) {
  constexpr int R = RT * 16, LD = R + 8;
  extern __shared__ __align__(16) __half us[];           // hi [64][LD], lo [64][LD]
  __shared__ int tok[kTile];
  __shared__ float down[kTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  griddep_launch();
  griddep_wait();
  const int total = *w.ntiles * nsplit;
  const int groups = (p.N + 31) / 32;
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const PlanTile tile = w.tiles[item / nsplit];
    const int part = item % nsplit;
    const int row0 = tile.row0 + (item / nsplit - tile.first) * kTile;
    const bool none = tile.index >= p.n;
    const int rank = none ? 0 : lora_rank(p, tile.index);
    const int steps = (rank + 15) / 16;
    __syncthreads();
    if (tid < kTile) {
      tok[tid] = w.slot[row0 + tid];
      down[tid] = tok[tid] >= 0 && !none ? w.down[row0 + tid] : 0.f;
    }
    if (!none)
      for (int e = tid; e < kTile * R / 8; e += blockDim.x) {
        const int t = e / (R / 8), c = e % (R / 8) * 8;
        *reinterpret_cast<uint4*>(us + t * LD + c) = *reinterpret_cast<const uint4*>(w.hi + (int64_t)(row0 + t) * R + c);
        *reinterpret_cast<uint4*>(us + (kTile + t) * LD + c) = *reinterpret_cast<const uint4*>(w.lo + (int64_t)(row0 + t) * R + c);
      }
    __syncthreads();
    const __half* B = none ? nullptr : p.b + tile.index * p.b_stride;
    const int glo = groups * part / nsplit, ghi = groups * (part + 1) / nsplit;
    for (int gr = glo + warp; gr < ghi; gr += kExpandWarps) {
      const int n0 = gr * 32;
      float acc[4][4][4] = {};                           // [16 tokens][column tile]
#pragma unroll
      for (int s = 0; s < RT; ++s) {
        if (s >= steps) break;
        uint2 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
          b[j] = make_uint2(0, 0);
          if (col < p.N) b[j] = load_b(B + col * p.ldb, s * 16 + 4 * q, rank);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __half* at = us + (h * kTile + m * 16 + g) * LD + s * 16 + 4 * q;
            const uint2 u0 = *reinterpret_cast<const uint2*>(at), u1 = *reinterpret_cast<const uint2*>(at + 8 * LD);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_16816(acc[m][j], u0.x, u1.x, u0.y, u1.y, b[j].x, b[j].y);
          }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = m * 16 + h * 8 + g;
          if (tok[t] < 0) continue;
          float d[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            d[2 * j] = acc[m][j][2 * h] * down[t];
            d[2 * j + 1] = acc[m][j][2 * h + 1] * down[t];
          }
          if (n0 + 8 * q < p.N) add_eight(p, tok[t], n0 + 8 * q, d);
        }
    }
  }
}

// Up to this many tokens take decode_kernel.
constexpr int kDecodeTokens = 128;

struct LoraLayout {
  int R;                                 // rank the kernels are built for
  int64_t rows, max_tiles;
  int64_t tiles, row, slot, hi, lo, down, bytes;
};

LoraLayout lora_layout(int64_t T, int64_t r, int64_t n) {
  LoraLayout m;
  std::memset(&m, 0, sizeof(m));
  m.R = r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128;
  if (T <= kDecodeTokens) return m;
  m.rows = plan_max_rows(T, n + 1, kTile);
  m.max_tiles = plan_max_tiles(T, n + 1, kTile);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  take(256);
  m.tiles = take(m.max_tiles * (int64_t)sizeof(PlanTile));
  m.row = take(T * 4);
  m.slot = take(m.rows * 4);
  m.hi = take(m.rows * m.R * 2);
  m.lo = take(m.rows * m.R * 2);
  m.down = take(m.rows * 4);
  m.bytes = at;
  return m;
}

int lora_check(int64_t T, int64_t r, int64_t n) {
  if (T < 0 || T > (1 << 24)) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: need 0..2^24 tokens");
  if (r < 16 || r > kLoraMaxRank || r % 16) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: the largest rank must be a multiple of 16 up to %d", kLoraMaxRank);
  if (n < 1 || n > kLoraMaxAdapters) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: 1..%d adapters", kLoraMaxAdapters);
  return NVFP4_OK;
}

template <int RT>
int lora_run(const LoraArgs& p, const LoraLayout& m, uint8_t* ws, cudaStream_t stream) {
  if (p.T <= kDecodeTokens) {
    decode_kernel<RT><<<p.T * kCluster, kDecodeWarps * 32, 0, stream>>>(p);
    return check_launch("decode_kernel");
  }
  const Plan plan = {reinterpret_cast<int*>(ws), reinterpret_cast<PlanTile*>(ws + m.tiles),
                     reinterpret_cast<int*>(ws + m.row), reinterpret_cast<int*>(ws + m.slot)};
  // tokens without an adapter become adapter n's, which only copies; in place they are left out
  int rc = launch_plan(p.adapters, p.T, p.n, p.in_place ? -1 : p.n, kTile, kTile, plan, stream);
  if (rc) return rc;
  const LoraRows rows = {plan.head, plan.tiles, plan.slot, reinterpret_cast<__half*>(ws + m.hi),
                         reinterpret_cast<__half*>(ws + m.lo), reinterpret_cast<float*>(ws + m.down)};
  constexpr int kShrinkSmem = kShrinkWarps * kShrinkTokens * RT * 16 * 4;
  constexpr int kExpandSmem = 2 * kTile * (RT * 16 + 8) * 2;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(NVFP4_ERR_UNSUPPORTED, "device index out of range");
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(shrink_kernel<RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kShrinkSmem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shrink)");
    attr_set[dev] = true;
  }
  const int64_t most = m.max_tiles;
  if ((rc = launch_after(shrink_kernel<RT>, "shrink_kernel",
                         (unsigned)std::min<int64_t>(most * (kTile / kShrinkTokens), (int64_t)sm_count() * 2),
                         kShrinkWarps * 32, kShrinkSmem, stream, p, rows)))
    return rc;
  // enough items for four rounds over the SMs, at least eight column groups (one per warp) each
  const int nsplit = (int)std::max<int64_t>(1, std::min<int64_t>((p.N + 255) / 256, (int64_t)sm_count() * 8 * kTile / p.T));
  return launch_after(expand_kernel<RT>, "expand_kernel", (unsigned)std::min<int64_t>(most * nsplit, (int64_t)sm_count() * 2),
                      kExpandWarps * 32, kExpandSmem, stream, p, rows, nsplit);
}

}  // namespace
}  // namespace nvfp4

extern "C" int nvfp4_lora_workspace(int64_t T, int64_t r, int64_t n, int64_t* bytes) {
  using namespace nvfp4;
  if (!bytes) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_workspace: null output");
  const int rc = lora_check(T, r, n);
  if (rc) return rc;
  *bytes = lora_layout(T, r, n).bytes;
  return NVFP4_OK;
}

extern "C" int nvfp4_lora_add(const void* base, int64_t ld_base, const void* x, int64_t ldx, const void* a, int64_t lda,
                              int64_t a_stride, const void* b, int64_t ldb, int64_t b_stride, const int32_t* adapters,
                              const float* scales, const int32_t* ranks, int64_t T, int64_t K, int64_t N, int64_t r,
                              int64_t n, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  using namespace nvfp4;
  int rc = lora_check(T, r, n);
  if (rc) return rc;
  if (K < 8 || K % 8 || K > (1 << 24) || N < 1 || N > (1 << 24))
    return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: K must be a positive multiple of 8 and N positive (at most 2^24)");
  if (T == 0) return NVFP4_OK;
  if (!base || !x || !a || !b || !adapters || !out) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: null pointer");
  if ((T > 1 && (ld_base < N || ldx < K || ldo < N)) || lda < K || ldb < r || (n > 1 && (a_stride < 0 || b_stride < 0)))
    return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: a row stride is below the row length, or an adapter stride is negative");
  if (T == 1) ld_base = ldo = N, ldx = K;
  if (n == 1) a_stride = b_stride = 0;
  if (!aligned16(x) || !aligned16(a) || !aligned16(b) || (ldx | lda | ldb | a_stride | b_stride) % 8)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_lora_add: x, a and b need 16-byte aligned rows");
  if ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(out)) & 1)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_lora_add: fp16 pointer not 2-byte aligned");
  if ((reinterpret_cast<uintptr_t>(adapters) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(ranks)) & 3)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_lora_add: adapters, scales and ranks must be 4-byte aligned");
  if (base == out && ld_base != ldo) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: out is base but has another row stride");
  const LoraLayout m = lora_layout(T, r, n);
  if (m.bytes && !workspace) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: null workspace");
  if (workspace_bytes < m.bytes)
    return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)m.bytes);
  if (m.bytes && (reinterpret_cast<uintptr_t>(workspace) & 255)) return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_lora_add: workspace not 256-byte aligned");
  LoraArgs p;
  p.base = static_cast<const __half*>(base); p.x = static_cast<const __half*>(x);
  p.a = static_cast<const __half*>(a); p.b = static_cast<const __half*>(b);
  p.adapters = adapters; p.scales = scales; p.ranks = ranks; p.out = static_cast<__half*>(out);
  p.ld_base = ld_base; p.ldx = ldx; p.lda = lda; p.a_stride = a_stride; p.ldb = ldb; p.b_stride = b_stride; p.ldo = ldo;
  p.T = (int)T; p.K = (int)K; p.N = (int)N; p.r = (int)r; p.n = (int)n;
  p.vec = aligned16(base) && aligned16(out) && ld_base % 8 == 0 && ldo % 8 == 0;
  p.in_place = base == out;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (m.R) {
    case 16: return lora_run<1>(p, m, ws, st);
    case 32: return lora_run<2>(p, m, ws, st);
    case 64: return lora_run<4>(p, m, ws, st);
    default: return lora_run<8>(p, m, ws, st);
  }
}
