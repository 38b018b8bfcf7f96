// Low-rank adapters of many requests, added to a shared projection's output:
//
//   out[t] = fp16( base[t] + scale_i * ((x[t] . A_i^T) . B_i^T) ),   i = adapters[t]
//
// A_i [r, K], B_i [N, r] (fp16), of which adapter i uses its first ranks[i] rows / columns.  Tokens without
// an adapter (an index outside [0, n)) keep base.  The floor of both forms is their bytes: x, base and out once,
// and the matrices of the adapters in use.
//
// The products run on mma.sync (fp16 operands, fp32 accumulators): with ranks of 16 to 128 there is little arithmetic
// per byte for tensor memory's round trips.  u = x . A^T enters the second product as two fp16 halves, u = 2^-p (hi + lo),
// with a 2^p per token that brings its largest |u| to [2^14, 2^15): each u keeps 22 bits, or is off by at most 2^-39 of the
// largest, where lo reaches the end of fp16's range.  The sum stays in fp32.
//
// The k index of an mma is summed over, so its 16 slots may stand for any 16 elements as long as both operands
// agree.  Two mma's take 32 elements, slots {2q, 2q+1, 2q+8, 2q+9} of lane q of 4 standing for elements 8q..8q+3 in
// the first and 8q+4..8q+7 in the second: fragments are loaded as they lie in memory, 16 bytes a lane.
//
// Few tokens (decode_kernel): one launch.  A cluster of CTAs takes up to 8 tokens of one adapter: each CTA
// sums its share of K for all ranks, the partial u's are exchanged through distributed shared memory and each CTA
// writes its share of N, whose first two steps of B are under way during the exchange.  K = 4096, N = 14336: one token
// of rank 16 5.3 us, 64 tokens of 32 adapters of rank 64 21 us (43 MB, 7 by bytes): with 13 warps an SM the latency of its
// loads bounds it.  Prefetching B into L2 from the start took 24 us, asking for one step behind the exchange 21.
//
// Many tokens: the plan (plan.cuh) orders them by adapter; shrink_kernel computes u, expand_kernel adds u . B^T.
#include <cuda_fp16.h>
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>
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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int lora_rank(const LoraArgs& p, int i) {
  if (i < 0) return 0;
  return p.ranks ? max(0, min(p.ranks[i], p.r)) : p.r;
}

// The power of two that brings magnitude m to [2^14, 2^15), and its inverse.  Without it where m is in fp16's range
// already, lo would end at 2^-25 however small m: entries of 2^-20 beside one of 2^-2 would keep 6 bits.  At most 2^110.
__device__ __forceinline__ void half_scale(float m, float& up, float& down) {
  int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
  if (m == 0.f || e == 128) e = 14;                          // nothing to bring up, or infinite already
  const int q = min(14 - e, 110);
  up = __uint_as_float((uint32_t)(q + 127) << 23);
  down = __uint_as_float((uint32_t)(127 - q) << 23);
}

// (a0 * m + c0, a1 * m + c1)
__device__ __forceinline__ float2 fma_pair(float a0, float a1, float m, float2 c) {
  float2 r;
  asm("{\n .reg .b64 a, m, c;\n mov.b64 a, {%2, %3};\n mov.b64 m, {%4, %4};\n mov.b64 c, {%5, %6};\n fma.rn.f32x2 a, a, m, c;\n"
      " mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a0), "f"(a1), "f"(m), "f"(c.x), "f"(c.y));
  return r;
}

__device__ __forceinline__ void split_halves(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// Zeros from element `rank` on (the row may hold anything there) in eight consecutive halves from element k on.
__device__ __forceinline__ uint4 below_rank(uint4 v, int k, int rank) {
  if (k + 8 > rank) {
    uint32_t* w = &v.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (k + 2 * j + 1 >= rank) w[j] &= 0x0000ffffu;
      if (k + 2 * j >= rank) w[j] = 0;
    }
  }
  return v;
}

// out[8 columns] = base + scale * d in 16-byte aligned rows; `v` holds base where all 8 columns exist.
__device__ __forceinline__ void add_eight(const LoraArgs& p, int64_t t, int col, const float (&d)[8], float scale, uint4 v) {
  __half* dst = p.out + t * p.ldo + col;
  if (col + 8 <= p.N) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      const __half2 h = __floats2half2_rn(fmaf(d[2 * j], scale, f.x), fmaf(d[2 * j + 1], scale, f.y));
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
    const __half* src = p.base + t * p.ld_base + col;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < p.N) dst[j] = __float2half_rn(fmaf(d[j], scale, __half2float(src[j])));
  }
}

__device__ __forceinline__ void cp_async_16(void* dst, const void* src, bool copy) {   // zeros if not `copy`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_u32(dst)), "l"(src), "r"(copy ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// ------------------------------------------------------------------ few tokens

constexpr int kDecodeWarps = 8;

__device__ __forceinline__ int cluster_nctas() {
  uint32_t v;
  asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(v));
  return (int)v;
}

constexpr int kDecodeTokens = 256;       // most tokens of one call
static_assert(kDecodeTokens <= kDecodeWarps * 32, "a thread per token");

template <int RT>
struct DecodeCfg {
  static constexpr int R = RT * 16;
  static constexpr int POOL = kDecodeWarps * (R > 36 ? R : 36) * 8;   // floats
  static constexpr int smem(int ncta) { return (POOL + ncta * R * 8) * 4; }
};

// Into how many parts an item's columns may go: every warp of a cluster has a step of 32 columns.
__host__ __device__ constexpr int decode_parts(int N, int ncta) {
  return ((N + 31) / 32 + ncta * kDecodeWarps - 1) / (ncta * kDecodeWarps);
}

// The two halves of a cluster barrier.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(addr), "f"(v) : "memory");
}

// RT: 16-row tiles of the largest rank, even.  VEC: base and out have 16-byte aligned rows.
template <int RT, bool VEC>
__global__ void __launch_bounds__(kDecodeWarps * 32, RT <= 4 ? 2 : 1) decode_kernel(const __grid_constant__ LoraArgs p) {
  constexpr int R = RT * 16, RS = RT / 2;                // RS: 32 ranks a step
  constexpr bool kAhead = RT <= 4;                       // registers for the next step's B
  extern __shared__ __align__(16) float dynamic[];
  // each warp's share of K, then u, in the end the warps' output patches
  float* const pool = dynamic;
  float(*const part)[R][8] = reinterpret_cast<float(*)[R][8]>(pool);
  float* const shares = dynamic + DecodeCfg<RT>::POOL;   // every CTA's share of K, [ncta][R][8]
  __shared__ __align__(16) __half hi[8][R + 8], lo[8][R + 8];
  __shared__ float down[8];
  __shared__ int key[kDecodeTokens], items[kDecodeTokens], tok[8], warp_items[kDecodeTokens / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int me = (int)cluster_ctarank(), ncta = cluster_nctas();
  // ---- the work list, the same in every CTA: tokens of one adapter go in eights, in token order, and an item is
  // the first token of an eight
  if (tid < p.T) {
    const int i = p.adapters[tid];
    key[tid] = (unsigned)i < (unsigned)p.n ? i : -1;
  }
  __syncthreads();
  bool leads = false;
  if (tid < p.T) {
    int before = 0;
    for (int s = 0; s < tid; ++s) before += key[s] == key[tid];
    leads = before % 8 == 0 && (key[tid] >= 0 || !p.in_place);
  }
  const unsigned leaders = __ballot_sync(0xffffffffu, leads);
  if (warp < kDecodeTokens / 32 && lane == 0) warp_items[warp] = __popc(leaders);
  __syncthreads();
  int nitems = 0, at = 0;
#pragma unroll
  for (int w = 0; w < kDecodeTokens / 32; ++w) {
    if (w == warp) at = nitems;
    nitems += warp_items[w];
  }
  if (leads) items[at + __popc(leaders & ((1u << lane) - 1))] = tid;
  __syncthreads();
  const int groups = (p.N + 31) / 32;                    // 32 columns per warp and step
  // Where clusters outnumber items, several share an item's columns, and each computes u (K = 4096, N = 14336: one token
  // of rank 16 6.5 -> 5.3 us, 16 of 16 adapters of rank 64 13.6 -> 12.1, 64 of one among 300 of rank 16 12.5 -> 8.1).  All
  // clusters run at once: the launch has no more than fit.
  const int clusters = (int)gridDim.x / ncta;
  const int parts = max(1, min(clusters / max(nitems, 1), decode_parts(p.N, ncta)));

  for (int work = (int)blockIdx.x / ncta; work < nitems * parts; work += clusters) {
    const int t0 = items[work / parts], i = key[t0], share = work % parts * ncta + me;
    const int glo = groups * share / (parts * ncta), ghi = groups * (share + 1) / (parts * ncta);
    if (warp == 0) {                                     // the eight's tokens; the previous item's readers have left
      if (lane < 8) tok[lane] = -1;
      __syncwarp();
      int found = 0;
      for (int s0 = t0; s0 < p.T && found < 8; s0 += 32) {
        const bool hit = s0 + lane < p.T && key[s0 + lane] == i;
        const unsigned hits = __ballot_sync(0xffffffffu, hit);
        const int to = found + __popc(hits & ((1u << lane) - 1));
        if (hit && to < 8) tok[to] = s0 + lane;
        found += __popc(hits);
      }
    }
    __syncthreads();
    if (i < 0) {                                         // no adapter: the rows stay what base says
      const int c0 = glo * 32, cols = min(p.N, ghi * 32) - c0;
      if (VEC) {
        const int chunks = (cols + 7) / 8;
#pragma unroll 4
        for (int e = tid; e < 8 * chunks; e += blockDim.x) {
          const int t = tok[e / chunks], c = c0 + e % chunks * 8;
          if (t < 0) continue;
          const float none[8] = {-0.f, -0.f, -0.f, -0.f, -0.f, -0.f, -0.f, -0.f};   // leaves base's own zeros as they are
          add_eight(p, t, c, none, 1.f, c + 8 <= p.N ? *reinterpret_cast<const uint4*>(p.base + t * p.ld_base + c) : make_uint4(0, 0, 0, 0));
        }
      } else {
#pragma unroll 8
        for (int e = tid; e < 8 * cols; e += blockDim.x) {
          const int t = tok[e / cols], c = c0 + e % cols;
          if (t >= 0) p.out[t * p.ldo + c] = p.base[t * p.ld_base + c];
        }
      }
      __syncthreads();
      continue;
    }
    cluster_arrive();                                    // this CTA runs, and has read the previous item's shares
    const int rank = lora_rank(p, i);
    const __half* A = p.a + i * p.a_stride;
    const __half* B = p.b + i * p.b_stride;
    const int j = lane >> 2, mytok = tok[j];             // this lane's token and columns in the end
    struct Step {
      uint4 b[RS][4], base;
      __half plain[8];                                   // unaligned rows: this lane's column of each token's base
    };
    auto ask = [&](int gr, Step& v) {                    // all that a step reads, before any of it is used
      if (gr >= ghi) return;
      const int n0 = gr * 32, c = n0 + (lane & 3) * 8;
      const __half* const from = B + (n0 + g) * p.ldb + 8 * q;
#pragma unroll
      for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          v.b[s][m] = make_uint4(0, 0, 0, 0);
          if (s * 32 + 8 * q < rank && n0 + m * 8 + g < p.N)
            v.b[s][m] = *reinterpret_cast<const uint4*>(from + m * 8 * p.ldb + s * 32);
        }
      if (VEC) {
        if (mytok >= 0 && c + 8 <= p.N) v.base = *reinterpret_cast<const uint4*>(p.base + mytok * p.ld_base + c);
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (tok[t] >= 0 && n0 + lane < p.N) v.plain[t] = p.base[tok[t] * p.ld_base + n0 + lane];
      }
    };
    Step one, two;
    // ---- u = x . A^T over this CTA's share of K: ranks are the mma's rows, tokens its columns
    {
      float acc[RT][4] = {};
      const int ksteps = (p.K + 31) / 32;
      const int klo = ksteps * me / ncta, khi = ksteps * (me + 1) / ncta;
      const __half* xr = tok[g] >= 0 ? p.x + (int64_t)tok[g] * p.ldx : nullptr;
#pragma unroll(RT <= 2 ? 2 : 1)
      for (int ks = klo + warp; ks < khi; ks += kDecodeWarps) {
        const int k = ks * 32 + q * 8;
        const bool in = k < p.K;                         // K is a multiple of 8
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
    if (kAhead) {                                        // in flight over the exchange
      ask(glo + warp, one);
      ask(glo + warp + kDecodeWarps, two);
    }
    __syncthreads();
    // this CTA's share goes to every CTA of the cluster, its own included, once all of them have arrived
    cluster_wait();
    for (int e = tid; e < R * 8; e += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) s += part[w][e >> 3][e & 7];
      const uint32_t there = smem_u32(shares + me * R * 8 + e);
      for (int c = 0; c < ncta; ++c) st_cluster_f32(mapa(there, c), s);
    }
    cluster_sync();
    // every CTA adds all shares in the same order: the same u everywhere
    {
      const float scale = p.scales ? p.scales[i] : 1.f;
      float* const u = pool;
      for (int e = tid; e < R * 8; e += blockDim.x) {
        float s = 0.f;
#pragma unroll 8
        for (int c = 0; c < ncta; ++c) s += shares[c * R * 8 + e];
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
    __syncthreads();
    // ---- out += u . B^T over this CTA's share of N: columns are the mma's rows, tokens its columns
    uint4 uh[RS], ul[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      uh[s] = *reinterpret_cast<const uint4*>(&hi[g][s * 32 + 8 * q]);
      ul[s] = *reinterpret_cast<const uint4*>(&lo[g][s * 32 + 8 * q]);
    }
    float(*const patch)[36] = reinterpret_cast<float(*)[36]>(pool + warp * 8 * 36);
    const float mydown = down[j];
    auto add = [&](int gr, Step& v) {
      if (gr >= ghi) return;
      const int n0 = gr * 32, c = n0 + (lane & 3) * 8;
      const float zero = rank > 0 ? 0.f : -0.f;
      float acc[2][4] = {{zero, zero, zero, zero}, {zero, zero, zero, zero}};
#pragma unroll
      for (int s = 0; s < RS; ++s) {
        if (s * 32 >= rank) break;
        if (rank & 7) {
#pragma unroll
          for (int m = 0; m < 4; ++m) v.b[s][m] = below_rank(v.b[s][m], s * 32 + 8 * q, rank);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint4 b0 = v.b[s][2 * m], b1 = v.b[s][2 * m + 1];
          mma_16816(acc[m], b0.x, b1.x, b0.y, b1.y, uh[s].x, uh[s].y);
          mma_16816(acc[m], b0.x, b1.x, b0.y, b1.y, ul[s].x, ul[s].y);
          mma_16816(acc[m], b0.z, b1.z, b0.w, b1.w, uh[s].z, uh[s].w);
          mma_16816(acc[m], b0.z, b1.z, b0.w, b1.w, ul[s].z, ul[s].w);
        }
      }
      // [token][column] patch, so that a lane gets a run of one token's columns
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        patch[2 * q][m * 16 + g] = acc[m][0];
        patch[2 * q + 1][m * 16 + g] = acc[m][1];
        patch[2 * q][m * 16 + g + 8] = acc[m][2];
        patch[2 * q + 1][m * 16 + g + 8] = acc[m][3];
      }
      __syncwarp();
      if (VEC) {
        if (mytok >= 0 && c < p.N) {
          const float4 d0 = *reinterpret_cast<const float4*>(&patch[j][(lane & 3) * 8]);
          const float4 d1 = *reinterpret_cast<const float4*>(&patch[j][(lane & 3) * 8 + 4]);
          const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
          add_eight(p, mytok, c, d, mydown, v.base);
        }
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (tok[t] >= 0 && n0 + lane < p.N)
            p.out[tok[t] * p.ldo + n0 + lane] = __float2half_rn(fmaf(patch[t][lane], down[t], __half2float(v.plain[t])));
      }
      __syncwarp();
    };
    if (kAhead) {
      for (int gr = glo + warp; gr < ghi; gr += 2 * kDecodeWarps) {
        add(gr, one);
        ask(gr + 2 * kDecodeWarps, one);
        add(gr + kDecodeWarps, two);
        ask(gr + 3 * kDecodeWarps, two);
      }
    } else {
      for (int gr = glo + warp; gr < ghi; gr += kDecodeWarps) {
        ask(gr, one);
        add(gr, one);
      }
    }
    __syncthreads();                                     // pool, tok and down are reused
  }
}

// ------------------------------------------------------------------ many tokens

constexpr int kTile = 128;               // tokens per tile of the plan
constexpr int kShrinkK = 128;            // elements of K per stage
constexpr int kShrinkStages = 3;
constexpr int kExpandCols = 64;          // columns per step of the second product
constexpr int kExpandStages = 3;
constexpr int kLoraThreads = 256;

struct LoraRows {
  const int* ntiles;
  const PlanTile* tiles;
  const int* slot;                       // token of each row, -1 for padding
  __half* hi;                            // [rows][R], R = r rounded up to 32, 64 or 128, laid out by u_at
  __half* lo;
  float* down;                           // [rows]
};

// Where u of (row, rank index k) lies: in blocks of 16 rows x 16 k, the 4 registers of an mma's first operand of
// each lane together.  Two neighbouring blocks hold 32 k, of which lane q of 4 has 8q..8q+3 and 8q+4..8q+7.
template <int R>
__device__ __forceinline__ int64_t u_at(int64_t row, int k) {
  const int64_t block = row / 16 * (R / 16) + k / 32 * 2 + k % 8 / 4;
  const int lane = (int)(row % 8) * 4 + k % 32 / 8, reg = k % 4 / 2 * 2 + (int)(row % 16) / 8;
  return (block * 32 + lane) * 8 + reg * 2 + k % 2;
}

// Row length in halves of a tile in shared memory that is read 16 bytes a lane, two neighbouring rows of 4 lanes
// at a time: rows 16 words apart modulo the 32 banks.
constexpr int padded_row(int halves) { return halves % 64 ? halves : halves + 32; }

template <int RT>
struct LoraCfg {
  static constexpr int R = RT * 16;
  static constexpr int LDR = padded_row(R);
  static constexpr int EXPAND_B = kExpandCols * LDR * 2;
  static constexpr int EXPAND_BASE = 8 * 4 * 512;        // a warp's 16 tokens x 64 columns, 4 pieces a lane
  static constexpr int EXPAND_SMEM = kExpandStages * (EXPAND_B + EXPAND_BASE);
};

// u of 32 or 64 tokens of one adapter: tokens are the mma's rows, ranks its columns.  x and A come through a ring
// of 128-element stages; two warps take half the tokens each over each quarter of a stage.  Rows are not padded: odd rows
// have the halves of each 128 bytes swapped, so that two neighbouring rows of 4 lanes, 16 bytes each, meet all banks once
// (two CTAs an SM fit; against padded rows 3000 tokens take 35.1 us instead of 37.8).  Where there are fewer tiles than
// places, a cluster of CTAs shares a tile's K (each a run of stages) and each finishes its share of the tokens.
// 8192 tokens, K = 4096, r = 64: 30 us (10 by bytes); latency, with 13 warps an SM.
template <int RT, int MT>
struct ShrinkCfg {
  static constexpr int R = RT * 16, TOKENS = 32 * MT;    // of a CTA
  static constexpr int STAGE = (TOKENS + R) * kShrinkK * 2;
  static constexpr int SMEM = kShrinkStages * STAGE;
  static_assert(SMEM >= 4 * TOKENS * R * 4, "the four shares of u");
};

template <int RT, int MT>
__global__ void __launch_bounds__(kLoraThreads, RT <= 4 ? 2 : 1) shrink_kernel(const __grid_constant__ LoraArgs p, const LoraRows w) {
  using C = ShrinkCfg<RT, MT>;
  constexpr int R = C::R, NT = RT * 2, TOKENS = C::TOKENS, PER = kTile / TOKENS, LD = kShrinkK, CHUNKS = kShrinkK / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int m0 = (warp & 1) * 16 * MT, share = warp >> 1;     // of kShrinkK: 32 elements, two mma's
  const int me = (int)cluster_ctarank(), ncta = cluster_nctas();
  griddep_launch();
  griddep_wait();
  const int total = *w.ntiles * PER;
  const int nk = (p.K + kShrinkK - 1) / kShrinkK;
  const int klo = nk * me / ncta, khi = nk * (me + 1) / ncta;
  for (int item = blockIdx.x / ncta; item < total; item += gridDim.x / ncta) {
    const PlanTile tile = w.tiles[item / PER];
    const int tr = (item / PER - tile.first) * kTile + item % PER * TOKENS;   // first token within the adapter
    if (tile.index >= p.n || tr >= tile.rows) continue;
    const int row0 = tile.row0 + tr;
    const int rank = lora_rank(p, tile.index);
    const __half* A = p.a + tile.index * p.a_stride;
    // this thread's pieces of a stage: 16 threads a row, 16 rows a pass
    const int pr = tid / CHUNKS, pc = tid % CHUNKS * 8, put = pc ^ (pr & 1) * 32;
    constexpr int XP = TOKENS / (kLoraThreads / CHUNKS), AP = (R + kLoraThreads / CHUNKS - 1) / (kLoraThreads / CHUNKS);
    const __half* xp[XP];
#pragma unroll
    for (int e = 0; e < XP; ++e) {
      const int s = w.slot[row0 + e * (kLoraThreads / CHUNKS) + pr];
      xp[e] = s >= 0 ? p.x + (int64_t)s * p.ldx : nullptr;
    }
    auto ask = [&](int ks) {
      if (ks < khi) {
        __half* const st = reinterpret_cast<__half*>(smem + ks % kShrinkStages * C::STAGE);
        const int k = ks * kShrinkK + pc;
#pragma unroll
        for (int e = 0; e < XP; ++e) {
          const bool in = xp[e] && k < p.K;
          cp_async_16(st + (e * (kLoraThreads / CHUNKS) + pr) * LD + put, in ? xp[e] + k : p.x, in);
        }
#pragma unroll
        for (int e = 0; e < AP; ++e) {
          const int row = e * (kLoraThreads / CHUNKS) + pr;
          const bool in = row < rank && k < p.K;
          if (row < R) cp_async_16(st + (TOKENS + row) * LD + put, in ? A + row * p.lda + k : p.a, in);
        }
      }
      cp_async_commit();
    };
    __syncthreads();                                     // the previous item's shared memory is read
#pragma unroll
    for (int s = 0; s < kShrinkStages - 1; ++s) ask(klo + s);
    const int get = (share * 32 + 8 * q) ^ (g & 1) * 32;
    float acc[MT][NT][4] = {};
    for (int ks = klo; ks < khi; ++ks) {
      cp_async_wait<kShrinkStages - 2>();
      __syncthreads();                                   // stage ks is here, stage ks - 1 free
      ask(ks + kShrinkStages - 1);
      const __half* const st = reinterpret_cast<const __half*>(smem + ks % kShrinkStages * C::STAGE);
      const __half* const xs = st + (m0 + g) * LD + get;
      const __half* const as = st + (TOKENS + g) * LD + get;
      uint4 x[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        x[m][0] = *reinterpret_cast<const uint4*>(xs + m * 16 * LD);
        x[m][1] = *reinterpret_cast<const uint4*>(xs + (m * 16 + 8) * LD);
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt += 2) {
        if (nt * 8 >= rank) break;
        const uint4 a0 = *reinterpret_cast<const uint4*>(as + nt * 8 * LD), a1 = *reinterpret_cast<const uint4*>(as + (nt + 1) * 8 * LD);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma_16816(acc[m][nt], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, a0.x, a0.y);
          mma_16816(acc[m][nt + 1], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, a1.x, a1.y);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma_16816(acc[m][nt], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, a0.z, a0.w);
          mma_16816(acc[m][nt + 1], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, a1.z, a1.w);
        }
      }
    }
    cp_async_wait<0>();
    __syncthreads();
    float* const part = reinterpret_cast<float*>(smem);  // [quarter of K][tokens][R]
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* at = part + (share * TOKENS + m0 + m * 16 + g) * R + nt * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[m][nt][0], acc[m][nt][1]);
        *reinterpret_cast<float2*>(at + 8 * R) = make_float2(acc[m][nt][2], acc[m][nt][3]);
      }
    __syncthreads();
    for (int e = tid; e < TOKENS * R; e += kLoraThreads)
      part[e] += part[e + TOKENS * R] + part[e + 2 * TOKENS * R] + part[e + 3 * TOKENS * R];
    if (ncta > 1) cluster_sync();                        // every CTA's sums are there
    else __syncthreads();
    const float scale = p.scales ? p.scales[tile.index] : 1.f;
    const int thi = TOKENS * (me + 1) / ncta;
    for (int t = TOKENS * me / ncta + warp; t < thi; t += kLoraThreads / 32) {
      float u[R / 32];
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < R / 32; ++e) {
        const float* at = part + t * R + e * 32 + lane;
        u[e] = *at;
        if (ncta > 1) {                                  // in the same order whoever adds them
          u[e] = 0.f;
          for (int c = 0; c < ncta; ++c) u[e] += __uint_as_float(ld_cluster_u32(mapa(smem_u32(at), c)));
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
      for (int e = 0; e < R / 32; ++e) {
        __half h, l;
        split_halves(u[e] * up, h, l);
        w.hi[u_at<R>(row, e * 32 + lane)] = h;
        w.lo[u_at<R>(row, e * 32 + lane)] = l;
      }
      if (lane == 0) w.down[row] = dn;
    }
    if (ncta > 1) cluster_sync();                        // the others have read this CTA's sums
  }
}

// out += u . B^T for 128 tokens of one adapter and a run of columns, 64 at a time: a warp takes 16 tokens, whose u
// stays in its registers.  B comes through a ring in shared memory that all warps read; base through a ring of
// which each lane reads back just what it asked for itself.
// 8192 tokens, N = 14336, r = 64: 112 us at 51 % of DRAM.  11 instructions for 32 outputs at 15 warps an SM bound it, not
// bytes (tensor memory, which would free the accumulators' registers, has not been tried)
// (registers: three CTAs an SM spill, 164 -> 230 us, four 267, in an earlier form).  Base is read before the products
// where registers allow (r = 64: 141.6 us a call against 151.0 with it read after them, r = 128: 305.5 and 270.6).
// The 8 columns of mma tile j of four stand for columns 8 (c / 2) + 2 j + c % 2 of 32, so that the four tiles
// give a lane 8 consecutive columns of a token.
template <int RT, bool VEC>
__global__ void __launch_bounds__(kLoraThreads, 2)
    expand_kernel(const __grid_constant__ LoraArgs p, const LoraRows w) {
  using C = LoraCfg<RT>;
  constexpr int R = C::R, LD = C::LDR, RS = RT / 2, CHUNKS = R / 8;
  constexpr int BROWS = kLoraThreads / CHUNKS;           // rows of B that the CTA copies in one go
  constexpr bool kBaseFirst = RT <= 4;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  uint8_t* const bases = smem + kExpandStages * C::EXPAND_B + warp * 2048 + lane * 16;
  // this thread's piece of each BROWS rows of B, and where this lane reads B
  const int bc = tid / CHUNKS, bk = tid % CHUNKS * 8;
  __half* const bput = reinterpret_cast<__half*>(smem) + bc * LD + bk;
  const __half* const bget = reinterpret_cast<const __half*>(smem) + (8 * (g >> 1) + (g & 1)) * LD + 8 * q;
  griddep_launch();
  griddep_wait();
  // all steps of all tiles in one row, an equal run of them for each CTA
  const int steps = (p.N + kExpandCols - 1) / kExpandCols;
  const int64_t total = (int64_t)*w.ntiles * steps;
  const int64_t end = total * (blockIdx.x + 1) / gridDim.x;
  for (int64_t at = total * blockIdx.x / gridDim.x; at < end;) {
    const int index = (int)(at / steps);
    const int lo = (int)(at - (int64_t)index * steps), hi = (int)min((int64_t)steps, lo + (end - at));
    at += hi - lo;
    const PlanTile tile = w.tiles[index];
    const int tr = (index - tile.first) * kTile;
    const int row0 = tile.row0 + tr + warp * 16;
    const bool none = tile.index >= p.n, live = tr + warp * 16 < tile.rows;
    const int rank = none ? 0 : lora_rank(p, tile.index);
    const __half* bsrc = none ? p.b : p.b + tile.index * p.b_stride + (int64_t)(lo * kExpandCols + bc) * p.ldb + bk;
    const bool bmine = bk < rank;                        // else zeros
    int tok[2];
    float down[2];
    const __half* src[2];                                // this lane's columns of its tokens' rows, at step lo
    __half* dst[2];
    uint4 u[2][2 * RS];                                  // [hi, lo][16 ranks]: first operands of the mma's
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      tok[h] = live ? w.slot[row0 + h * 8 + g] : -1;
      down[h] = tok[h] >= 0 && !none ? w.down[row0 + h * 8 + g] : 1.f;
      src[h] = p.base + (int64_t)max(tok[h], 0) * p.ld_base + lo * kExpandCols + 8 * q;
      dst[h] = p.out + (int64_t)max(tok[h], 0) * p.ldo + lo * kExpandCols + 8 * q;
    }
#pragma unroll
    for (int s = 0; s < 2 * RS; ++s) {
      u[0][s] = u[1][s] = make_uint4(0, 0, 0, 0);
      if (s / 2 * 32 < rank && live) {
        const int64_t from = ((int64_t)(row0 / 16) * (2 * RS) + s) * 32 + lane;
        u[0][s] = reinterpret_cast<const uint4*>(w.hi)[from];
        u[1][s] = reinterpret_cast<const uint4*>(w.lo)[from];
      }
    }
    int ring_in = 0, ahead = 0;                          // next ring to fill, its distance from lo in steps
    auto ask = [&]() {
      if (lo + ahead < hi) {
        const int n0 = (lo + ahead) * kExpandCols;
        if (rank > 0) {
#pragma unroll
          for (int e = 0; e < kExpandCols / BROWS; ++e) {
            const bool in = bmine && n0 + bc + e * BROWS < p.N;
            cp_async_16(bput + ring_in * (C::EXPAND_B / 2) + e * BROWS * LD, in ? bsrc + e * BROWS * p.ldb : p.b, in);
          }
          bsrc += kExpandCols * p.ldb;
        }
        if (VEC) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {                  // [column half][row half]
            if (tok[e & 1] >= 0 && n0 + (e >> 1) * 32 + 8 * q + 8 <= p.N)
              cp_async_16(bases + ring_in * C::EXPAND_BASE + e * 512, src[e & 1] + ahead * kExpandCols + (e >> 1) * 32, true);
          }
        }
        ring_in = ring_in + 1 == kExpandStages ? 0 : ring_in + 1;
        ++ahead;
      }
      cp_async_commit();
    };
    __syncthreads();                                     // the previous run's ring is read
#pragma unroll
    for (int s = 0; s < kExpandStages - 1; ++s) ask();
    int ring = 0;
    for (int st = lo; st < hi; ++st) {
      cp_async_wait<kExpandStages - 2>();
      __syncthreads();                                   // step st is here, step st - 1's ring free
      ask();
      if (live) {
        const __half* const bs = bget + ring * (C::EXPAND_B / 2);
        auto columns = [&](auto full) {
          // all 64 columns exist: without the code for the last ones 3 % less a call (8192 tokens, r = 64)
          constexpr bool FULL = decltype(full)::value;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int n0 = st * kExpandCols + half * 32, col = n0 + 8 * q, off = (st - lo) * kExpandCols + half * 32;
            __half plain[16];                              // !VEC: base of this lane's column for the 16 tokens
            if (!VEC) {
#pragma unroll
              for (int t = 0; t < 16; ++t) {
                const int tk = __shfl_sync(0xffffffffu, tok[t >> 3], (t & 7) * 4);
                plain[t] = tk >= 0 && n0 + lane < p.N ? p.base[tk * p.ld_base + n0 + lane] : __float2half_rn(0.f);
              }
            }
            // -0 leaves base's own zeros as they are where nothing is added
            const float zero = rank > 0 ? 0.f : -0.f;
            float acc[4][4];
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e >> 2][e & 3] = zero;
            uint4 bv[2];                                   // VEC: base of 8 columns of each token
            auto read_base = [&](int h) { bv[h] = *reinterpret_cast<const uint4*>(bases + ring * C::EXPAND_BASE + (half * 2 + h) * 512); };
            if (VEC && kBaseFirst) read_base(0), read_base(1);
            const bool whole = FULL || col + 8 <= p.N;
#pragma unroll
            for (int s = 0; s < RS; ++s) {
              if (s * 32 >= rank) break;
              uint4 b[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const uint4*>(bs + (half * 32 + 2 * j) * LD + s * 32);
              if (rank & 7) {
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = below_rank(b[j], s * 32 + 8 * q, rank);
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {                // neighbouring mma's add to different accumulators
                const uint4 u0 = u[h][2 * s], u1 = u[h][2 * s + 1];
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_16816(acc[j], u0.x, u0.y, u0.z, u0.w, b[j].x, b[j].y);
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_16816(acc[j], u1.x, u1.y, u1.z, u1.w, b[j].z, b[j].w);
              }
            }
            if (VEC) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (tok[h] < 0) continue;
                if (whole) {
                  if (!kBaseFirst) read_base(h);
                  const uint32_t from[4] = {bv[h].x, bv[h].y, bv[h].z, bv[h].w};
                  uint32_t o[4];
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&from[j]));
                    const __half2 r = __float22half2_rn(fma_pair(acc[j][2 * h], acc[j][2 * h + 1], down[h], f));
                    o[j] = *reinterpret_cast<const uint32_t*>(&r);
                  }
                  *reinterpret_cast<uint4*>(dst[h] + off) = make_uint4(o[0], o[1], o[2], o[3]);
                } else {
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    if (col + e < p.N)
                      dst[h][off + e] = __float2half_rn(fmaf(acc[e >> 1][2 * h + (e & 1)], down[h], __half2float(src[h][off + e])));
                }
              }
            } else {
              // rows of any alignment: through a patch of [16 tokens][32 columns], a lane a column
              float* const patch = reinterpret_cast<float*>(smem + kExpandStages * C::EXPAND_B + warp * 2048);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  *reinterpret_cast<float2*>(patch + (h * 8 + g) * 32 + 8 * q + 2 * j) =
                      make_float2(acc[j][2 * h] * down[h], acc[j][2 * h + 1] * down[h]);
              __syncwarp();
#pragma unroll
              for (int t = 0; t < 16; ++t) {
                const int tk = __shfl_sync(0xffffffffu, tok[t >> 3], (t & 7) * 4);
                if (tk >= 0 && n0 + lane < p.N)
                  p.out[tk * p.ldo + n0 + lane] = __float2half_rn(__half2float(plain[t]) + patch[t * 32 + lane]);
              }
              __syncwarp();
            }
          }
        };
        if ((st + 1) * kExpandCols <= p.N) columns(std::true_type());
        else columns(std::false_type());
      }
      ring = ring + 1 == kExpandStages ? 0 : ring + 1;
    }
    cp_async_wait<0>();
  }
}

struct LoraLayout {
  int R;                                 // rank the kernels are built for
  int64_t rows, max_tiles;
  int64_t tiles, row, slot, hi, lo, down, bytes;
};

LoraLayout lora_layout(int64_t T, int64_t r, int64_t n) {
  LoraLayout m;
  std::memset(&m, 0, sizeof(m));
  m.R = r <= 32 ? 32 : r <= 64 ? 64 : 128;
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

// Whether two sets of `rows` rows of fp16 elements share any: row strides ld, row lengths len.  Rows of one stride
// may lie between one another (column slices of one buffer); with two strides, ranges that meet count as shared.
bool rows_meet(const void* a, int64_t lda, int64_t lena, const void* b, int64_t ldb, int64_t lenb, int64_t rows) {
  const int64_t d = (static_cast<const char*>(b) - static_cast<const char*>(a)) / 2;
  if (d >= (rows - 1) * lda + lena || -d >= (rows - 1) * ldb + lenb) return false;
  if (rows == 1 || lda != ldb) return true;
  const int64_t m = (d % lda + lda) % lda;       // where b's rows begin within a's
  return m < lena || m + lenb > lda;
}

int lora_check(int64_t T, int64_t r, int64_t n) {
  if (T < 0 || T > (1 << 24)) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: need 0..2^24 tokens");
  if (r < 16 || r > kLoraMaxRank || r % 16) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: the largest rank must be a multiple of 16 up to %d", kLoraMaxRank);
  if (n < 1 || n > kLoraMaxAdapters) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: 1..%d adapters", kLoraMaxAdapters);
  return NVFP4_OK;
}

// CTAs a cluster for few tokens: 8 read an item's matrices sooner, but where more items than clusters are to be expected
// smaller clusters take them in fewer rounds.  The items are in GPU memory; `T` tokens that choose among n adapters at
// random take n (1 - (1 - 1/n)^T) of them, in eights.  fit: clusters of 1, 2, 4, 8 that run at once.  Returns the size's log2.
// us with 8, 4, 2 and 1 (K = N = 4096): 16 tokens of 300 adapters of rank 16 6.6, 7.0, 8.2, 10.6; 100 of 100 of rank 16 12.7, 9.7, 12.7,
// 17.0; 256 of 200 of rank 64 52.8, 40.0, 37.4, 48.8; 256 of 256 (1024 x 1024) 24.8, 16.1, 13.2, 11.2.  A batch of one adapter
// among many would rather have 8 (200 tokens, 300 adapters of rank 64: 12.0, where this takes 2 and 16.6).
int decode_cluster(int T, int n, const int (&fit)[4]) {
  const double used = n * (1 - std::pow(1 - 1.0 / n, T));
  const double items = used * std::max(1.0, (T / used + 3.5) / 8);
  int size = 3;
  while (size > 0 && items > fit[size]) --size;
  return size;
}

template <int RT>
int lora_run(const LoraArgs& p, const LoraLayout& m, uint8_t* ws, cudaStream_t stream) {
  using C = LoraCfg<RT>;
  static OncePerDevice once;
  static int fits[kMaxDevices][4];       // clusters of 1, 2, 4, 8 for few tokens that run at once
  constexpr int kWide = RT <= 4 ? 2 : 1, kSlots = RT <= 4 ? 2 : 1;   // m tiles a warp, CTAs an SM, of the first product
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return fail(NVFP4_ERR_UNSUPPORTED, "device index out of range");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kDecodeWarps * 32);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int rc = once.run(dev, [&] {
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<RT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<RT>::smem(8));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(decode_kernel<RT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<RT>::smem(8));
    for (int size = 0; size < 4 && e == cudaSuccess; ++size) {
      int with = 0, without = 0;
      attr[0].val.clusterDim.x = 1u << size;
      cfg.gridDim = dim3(1u << size);
      cfg.dynamicSmemBytes = DecodeCfg<RT>::smem(1 << size);
      e = cudaOccupancyMaxActiveClusters(&with, decode_kernel<RT, true>, &cfg);
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&without, decode_kernel<RT, false>, &cfg);
      fits[dev][size] = std::max(1, std::min(with, without));
    }
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(shrink_kernel<RT, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, ShrinkCfg<RT, 1>::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(shrink_kernel<RT, kWide>, cudaFuncAttributeMaxDynamicSharedMemorySize, ShrinkCfg<RT, kWide>::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(expand_kernel<RT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::EXPAND_SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(expand_kernel<RT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::EXPAND_SMEM);
    return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "cudaFuncSetAttribute(low-rank products)");
  });
  if (rc) return rc;
  if (p.T <= kDecodeTokens) {
    const int size = decode_cluster(p.T, p.n, fits[dev]);
    const int ncta = 1 << size;
    attr[0].val.clusterDim.x = (unsigned)ncta;
    cfg.dynamicSmemBytes = DecodeCfg<RT>::smem(ncta);
    const int64_t most = (int64_t)p.T * decode_parts(p.N, ncta);
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(most, fits[dev][size]) * ncta));
    cudaError_t e = cudaLaunchKernelEx(&cfg, p.vec ? decode_kernel<RT, true> : decode_kernel<RT, false>, p);
    return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "cudaLaunchKernelEx(decode)");
  }
  const Plan plan = {reinterpret_cast<int*>(ws), reinterpret_cast<PlanTile*>(ws + m.tiles),
                     reinterpret_cast<int*>(ws + m.row), reinterpret_cast<int*>(ws + m.slot)};
  // tokens without an adapter become adapter n's, which only copies; in place they are left out
  rc = launch_plan(p.adapters, p.T, p.n, p.in_place ? -1 : p.n, kTile, kTile, plan, stream);
  if (rc) return rc;
  const LoraRows rows = {plan.head, plan.tiles, plan.slot, reinterpret_cast<__half*>(ws + m.hi),
                         reinterpret_cast<__half*>(ws + m.lo), reinterpret_cast<float*>(ws + m.down)};
  // 64 tokens a CTA read A half as often, which pays once they fill the SMs (K = 4096, us a call, 32 and 64 tokens: 2048
  // tokens 32.6 and 33.2, 3000 33.0 and 32.0, 16384 103.3 and 92.7).  CTAs per tile: as many as fill the slots, each
  // with at least two stages (300 tokens, K = 1024, the product: 6.7 us with four, 5.7 with two).  One CTA a tile and as many
  // as this, the product alone at K = 4096, r = 64: 300 tokens 23.0 and 7.4, 1024 tokens 25.9 and 14.4, 8192 37.7 and 32.9.
  const bool twice = kWide > 1 && p.T >= 2560;
  const int tokens = twice ? 32 * kWide : 32;
  const int64_t items = (p.T + tokens - 1) / tokens;
  int share = 1;
  while (share < 8 && items * share * 2 <= sm_count() * kSlots && p.K > (share * 2 * 2 - 1) * kShrinkK) share *= 2;
  {
    cudaLaunchAttribute both[2] = {attr[0], attr[0]};
    both[0].val.clusterDim.x = (unsigned)share;
    both[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    both[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(m.max_tiles * (kTile / tokens), std::max(1, sm_count() * 2 / share)) * share));
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = twice ? ShrinkCfg<RT, kWide>::SMEM : ShrinkCfg<RT, 1>::SMEM;
    cfg.attrs = both;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, twice ? shrink_kernel<RT, kWide> : shrink_kernel<RT, 1>, p, rows);
    if (e != cudaSuccess) return cuda_fail(e, "cudaLaunchKernelEx(shrink)");
  }
  const int64_t steps = (p.N + kExpandCols - 1) / kExpandCols;
  return launch_after(p.vec ? expand_kernel<RT, true> : expand_kernel<RT, false>, "expand_kernel",
                      (unsigned)std::min<int64_t>(m.max_tiles * steps, (int64_t)sm_count() * 2), kLoraThreads,
                      C::EXPAND_SMEM, stream, p, rows);
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
  if (rows_meet(x, ldx, K, out, ldo, N, T)) return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: out overlaps x");
  if (base != out && rows_meet(base, ld_base, N, out, ldo, N, T))
    return fail(NVFP4_ERR_INVALID, "nvfp4_lora_add: out overlaps base without being it");
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
    case 32: return lora_run<2>(p, m, ws, st);
    case 64: return lora_run<4>(p, m, ws, st);
    default: return lora_run<8>(p, m, ws, st);
  }
}
