// The experts' SiLU-gated MLP on NVFP4 weights, for tokens that each chose
// their experts (nvfp4_route_experts or any other ids):
//
//   xq = nvfp4(x[t]);  h = silu(xq . Wg_e^T) * (xq . Wu_e^T);  hq = nvfp4(h)
//   out[t] = fp16( sum_j weights[t, j] * (hq . Wd_e^T) ),  e = ids[t, j], slots in order of j
//
// The plan (plan.cuh), quantising the tokens into their rows (each token once,
// stored for each of its experts; one launch with the plan for few slots),
// the two expert products (moe_gemm.cuh) and the sum over a token's slots.  h never leaves the first
// product but as NVFP4.  y = weight * product stays in fp32 between the second
// product and the sum: the sum then rounds once, and a product beyond fp16's
// range does no harm.
#include <cuda_fp16.h>
#include <algorithm>
#include <cstring>
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "common.h"
#include "tmap.h"
#include "gemm_cfg.cuh"
#include "moe_gemm.cuh"

namespace nvfp4 {
namespace {

constexpr int kMoeMaxExperts = kPlanMaxIndexes, kMoeMaxTopK = 32;

struct ScatterArgs {
  const __half* x;
  int64_t ldx, T;
  int k, D;
  const float* weights;
  uint8_t* codes;
  uint8_t* sf;
  float* row_weight;
};

// Quantises token t and stores it for each of its slots: a thread takes one 16-element block.
__device__ __forceinline__ void scatter_token(const ScatterArgs& a, int64_t t, const int* rows) {
  const int kb = a.D / 16, lane = threadIdx.x & 31;
  for (int c0 = threadIdx.x & ~31; c0 < kb; c0 += blockDim.x) {
    const int c = c0 + lane;
    const bool live = c < kb;
    uint32_t w[8], packed[2], sbyte = 0;
    if (live) {
      load_block(a.x + t * a.ldx + (int64_t)c * 16, w);
      sbyte = quant_halves(w, packed);
    }
    const uint32_t b1 = __shfl_down_sync(0xffffffffu, sbyte, 1);
    const uint32_t b2 = __shfl_down_sync(0xffffffffu, sbyte, 2);
    const uint32_t b3 = __shfl_down_sync(0xffffffffu, sbyte, 3);
    if (!live) continue;
    for (int j = 0; j < a.k; ++j) {
      const int r = rows[j];
      if (r < 0) continue;
      *reinterpret_cast<uint2*>(a.codes + (int64_t)r * (a.D / 2) + c * 8) = make_uint2(packed[0], packed[1]);
      if ((lane & 3) == 0)             // D is a multiple of 64: whole words of four blocks
        *reinterpret_cast<uint32_t*>(a.sf + blocked_at(r, c, a.D / 64)) = sbyte | (b1 << 8) | (b2 << 16) | (b3 << 24);
    }
  }
  if ((int)threadIdx.x < a.k && rows[threadIdx.x] >= 0)
    a.row_weight[rows[threadIdx.x]] = a.weights[t * a.k + threadIdx.x];
}

__global__ void __launch_bounds__(256) scatter_kernel(const int* rows, ScatterArgs a) {
  griddep_launch();
  griddep_wait();
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) scatter_token(a, t, rows + t * a.k);
}

// Plan and scatter in one launch, for few slots: every CTA (one per token) counts all of them for itself and
// finds the rows of its own token's, a warp a slot: its expert's first row plus the number of equal ids before
// it.  CTA 0 lists the tiles.  Every CTA counts all slots, which pays while the CTAs run at once.  Calls, us, so and with
// the two kernels one after the other (64 experts of 2048 x 1024): 1 token of 8 slots 20.1 and 21.4, 256 of 8 64.7 and
// 66.1, 384 of 5 62.5 and 63.2, 512 of 2 56.7 and 57.8, 512 of 4 63.7 and 64.3; 682 of 3 64.3 and 63.9, 1024 of 1 59.7 and
// 56.8, 1000 of 2 68.3 and 64.8, 2000 of 1 75.6 and 66.7.  Few tokens of many slots are as fast either way (64 of 32:
// 75.1 and 74.6).
constexpr int kFusedSlots = 2048, kFewTokens = 512;

__global__ void __launch_bounds__(256) plan_scatter_kernel(const int32_t* __restrict__ ids, int n, int experts, int align,
                                                           int tile, Plan p, ScatterArgs a) {
  __shared__ int id[kFusedSlots];
  __shared__ int count[kPlanMaxIndexes], row0[kPlanMaxIndexes];
  __shared__ int mine[kMoeMaxTopK], sums[8][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t = blockIdx.x;
  griddep_launch();
  for (int e = tid; e < kPlanMaxIndexes; e += 256) count[e] = 0;
  __syncthreads();
  for (int s = tid; s < n; s += 256) {
    const int e = ids[s];
    id[s] = (unsigned)e < (unsigned)experts ? e : -1;
    if (id[s] >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  // thread i: experts 4i .. 4i + 3
  int span = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = count[4 * tid + j];
    span += (c + align - 1) / align * align;
    tiles += (c + tile - 1) / tile;
  }
  int r = span, m = tiles;                       // inclusive scans
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, r, o), v = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) r += u, m += v;
  }
  if (lane == 31) sums[warp][0] = r, sums[warp][1] = m;
  __syncthreads();
  int first = m - tiles, from = r - span, all = 0;
  for (int w = 0; w < 8; ++w) {
    if (w < warp) from += sums[w][0], first += sums[w][1];
    all += sums[w][1];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = 4 * tid + j, c = count[e], here = (c + tile - 1) / tile;
    row0[e] = from;
    if (t == 0)
      for (int i = 0; i < here; ++i) {
        PlanTile q;
        q.index = e; q.row0 = from; q.first = first; q.tiles = here; q.rows = c;
        q.pad[0] = q.pad[1] = q.pad[2] = 0;
        p.tiles[first + i] = q;
      }
    from += (c + align - 1) / align * align;
    first += here;
  }
  if (t == 0 && tid == 0) p.head[0] = all;
  __syncthreads();
  for (int j = warp; j < a.k; j += 8) {
    const int s = (int)t * a.k + j, e = id[s];
    int before = 0;
    for (int o = lane; o < s; o += 32) before += id[o] == e;
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) {
      mine[j] = e >= 0 ? row0[e] + before : -1;
      p.row[s] = mine[j];
    }
  }
  __syncthreads();
  scatter_token(a, t, mine);
}

// out[t] = sum of its slots' rows of y, in slot order (and of the parts of each); eight columns a thread.
// 4096 tokens of 4096 columns in 2 slots each: it ends 38 us after the down product, 4.4 TB/s of y (fp32) and out.
// No __restrict__: y is still being written when this kernel starts, so it is not read-only for the kernel's lifetime.
__global__ void __launch_bounds__(256) combine_kernel(const float* y, int parts, int64_t part_stride, const int* rows,
                                                      int64_t T, int k, int D, __half* out, int64_t ldo, int vec) {
  griddep_launch();
  griddep_wait();
  const int per = D / 8;
  const int64_t total = T * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per;
    const int c = (int)(i - t * per) * 8;
    float acc[8] = {};
    for (int j = 0; j < k; ++j) {
      const int r = rows[t * k + j];
      if (r < 0) continue;
      for (int s = 0; s < parts; ++s) {
        const float4* src = reinterpret_cast<const float4*>(y + s * part_stride + (int64_t)r * D + c);
        const float4 a = src[0], b = src[1];
        acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
        acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
      }
    }
    const uint4 piece = make_uint4(pack_h2(acc[0], acc[1]), pack_h2(acc[2], acc[3]), pack_h2(acc[4], acc[5]),
                                   pack_h2(acc[6], acc[7]));
    __half* dst = out + t * ldo + c;
    if (vec) *reinterpret_cast<uint4*>(dst) = piece;
    else store_piece(dst, piece, 8);
  }
}

// Where the pieces of the workspace begin.
struct MoeLayout {
  bool trans;           // few tokens per expert: weights as the MMA's first operand
  int tile;             // token rows per tile, and the alignment of an expert's rows
  int parts;            // of the down product's inner dimension
  int64_t rows, max_tiles;
  int64_t tiles, row, row_weight, xq, xs, hq, hs, y, bytes;
};

// Into how many parts the down product of few tokens cuts its inner dimension where its tiles would leave SMs
// idle: the count with the fewest stages on the busiest SM, if every expert that can be active is.  A part more
// costs a y to write and to read again, which is counted at half a stage (32 KB of weights).
int down_parts(int64_t n, int64_t E, int64_t D, int64_t F, int tile) {
  const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(std::min(n, E) + n / tile, n)) * ((D + 127) / 128);
  const int64_t stages = (F + 511) / 512, sms = sm_count();
  int best = 1;
  double least = 1e30;
  for (int64_t s = 1; s <= std::min<int64_t>(8, stages) && (s == 1 || tiles < sms); ++s) {
    const double cost = (double)((tiles * s + sms - 1) / sms) * ((stages + s - 1) / s) + 0.5 * (s - 1);
    if (cost < least - 1e-9) {
      least = cost;
      best = (int)s;
    }
  }
  return best;
}

MoeLayout moe_layout(int64_t T, int64_t k, int64_t E, int64_t D, int64_t F) {
  MoeLayout m;
  const int64_t n = T * k;
  // 16-token tiles up to 16 rows an expert, 128-row tiles above.  64 experts of 2048 x 1024, us: 16 rows an expert
  // 58.9 and 57.9, 8 rows 51.5 and 54.8, 32 rows 78 and 66; 8 experts of 4096 x 14336: 4 rows 124 and 135, 16 rows 146
  // and 149, 24 rows 172 and 139.  Tiles of 32 and 64 tokens are slower than one or the other everywhere.
  m.trans = n <= 16 * E;
  m.tile = m.trans ? 16 : 128;
  m.parts = m.trans ? down_parts(n, E, D, F, m.tile) : 1;
  m.rows = (plan_max_rows(n, E, m.tile) + 127) / 128 * 128;
  m.max_tiles = plan_max_tiles(n, E, m.tile);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 1023) / 1024 * 1024;
    return here;
  };
  take(256);
  m.tiles = take(m.max_tiles * (int64_t)sizeof(PlanTile));
  m.row = take(n * 4);
  m.row_weight = take(m.rows * 4);
  m.xq = take(m.rows * D / 2);
  m.xs = take(m.rows * D / 16);
  m.hq = take(m.rows * F / 2);
  m.hs = take(m.rows * F / 16);
  m.y = take(m.parts * m.rows * D * 4);
  m.bytes = at;
  return m;
}

int moe_check(int64_t T, int64_t k, int64_t E, int64_t D, int64_t F) {
  if (T < 0 || k < 1 || k > kMoeMaxTopK || E < 1 || E > kMoeMaxExperts)
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: need T >= 0, 1..%d slots per token and 1..%d experts", kMoeMaxTopK, kMoeMaxExperts);
  if (D < 64 || D % 64 || F < 64 || F % 64 || D > (1 << 20) || F > (1 << 20))
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: both widths must be positive multiples of 64 (at most 2^20)");
  if (T > (int64_t)(1 << 24) / k) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: more than 2^24 slots");
  return NVFP4_OK;
}

int check_weights(const char* name, const void* w, const void* sf, int64_t E, int64_t K, int64_t ld, int64_t es,
                  int64_t sfe) {
  if (!w || !sf) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: %s: null pointer", name);
  if (ld < K / 2 || (E > 1 && (es <= 0 || sfe <= 0)))
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: %s: row stride below K/2, or an expert stride that is not positive", name);
  if (!aligned16(w) || !aligned16(sf) || ld % 16 || (E > 1 && (es % 16 || sfe % 16)))
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_moe_mlp: %s: pointers and strides must be multiples of 16 bytes", name);
  return NVFP4_OK;
}

int weight_maps(CUtensorMap* tw, CUtensorMap* tsw, const void* w, const void* sf, int64_t E, int64_t N, int64_t K,
                int64_t ld, int64_t es, int64_t sfe, int box_rows, int kps) {
  if (E == 1) es = N * ld, sfe = (N + 127) / 128 * (K / 64) * 512;
  const uint64_t dims[3] = {(uint64_t)(K / 2), (uint64_t)N, (uint64_t)E};
  const uint64_t str[2] = {(uint64_t)ld, (uint64_t)es};
  const uint32_t box[3] = {KSTEP_BYTES, (uint32_t)box_rows, 1};
  int rc = encode_tmap(tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, w, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  const uint64_t nk64 = (uint64_t)(K / 64);
  const uint64_t sdims[4] = {128, nk64, (uint64_t)((N + 127) / 128), (uint64_t)E};
  const uint64_t sstr[3] = {512, nk64 * 512, (uint64_t)sfe};
  const uint32_t sbox[4] = {128, (uint32_t)kps, (uint32_t)(box_rows / 128), 1};
  return encode_tmap(tsw, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, sf, sdims, sstr, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
}

int token_maps(ExpertParams& P, const void* codes, const void* sf, int64_t rows, int64_t K, int box_rows, int kps) {
  const uint64_t dims[2] = {(uint64_t)(K / 2), (uint64_t)rows};
  const uint64_t str[1] = {(uint64_t)(K / 2)};
  const uint32_t box[2] = {KSTEP_BYTES, (uint32_t)box_rows};
  int rc = encode_tmap(&P.tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, TmapOf::kWorkspace);
  if (rc) return rc;
  const uint64_t nk64 = (uint64_t)(K / 64);
  const uint64_t sdims[3] = {128, nk64, (uint64_t)(rows / 128)};
  const uint64_t sstr[2] = {512, nk64 * 512};
  const uint32_t sbox[3] = {128, (uint32_t)kps, 1};
  return encode_tmap(&P.tst, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, sf, sdims, sstr, sbox, CU_TENSOR_MAP_SWIZZLE_NONE,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, TmapOf::kWorkspace);
}

struct MoeCall {
  const __half* x;
  int64_t ldx;
  const int32_t* ids;
  const float* weights;
  __half* out;
  int64_t ldo, T, k;
  const void *wg, *wu, *wd, *sg, *su, *sd;
  int64_t E, D, F;
  int64_t ld_in, es_in, sfe_in, ld_down, es_down, sfe_down;   // byte strides: rows, experts, scales of an expert
  MoeLayout m;
  uint8_t* ws;
  uint32_t* err;
  cudaStream_t stream;
  int dev;
};

// Everything of a product's launch that can be refused, before the first launch of the call.
template <class C>
int expert_params(const MoeCall& c, ExpertParams& P) {
  std::memset(&P, 0, sizeof(P));
  const MoeLayout& m = c.m;
  int rc;
  if (C::DUAL) {
    if ((rc = token_maps(P, c.ws + m.xq, c.ws + m.xs, m.rows, c.D, C::T_ROWS, C::KPS)) ||
        (rc = weight_maps(&P.tw[0], &P.tsw[0], c.wg, c.sg, c.E, c.F, c.D, c.ld_in, c.es_in, c.sfe_in, C::W_ROWS, C::KPS)) ||
        (rc = weight_maps(&P.tw[1], &P.tsw[1], c.wu, c.su, c.E, c.F, c.D, c.ld_in, c.es_in, c.sfe_in, C::W_ROWS, C::KPS)))
      return rc;
  } else {
    if ((rc = token_maps(P, c.ws + m.hq, c.ws + m.hs, m.rows, c.F, C::T_ROWS, C::KPS)) ||
        (rc = weight_maps(&P.tw[0], &P.tsw[0], c.wd, c.sd, c.E, c.D, c.F, c.ld_down, c.es_down, c.sfe_down, C::W_ROWS, C::KPS)))
      return rc;
  }
  P.tiles = reinterpret_cast<const PlanTile*>(c.ws + m.tiles);
  P.ntiles = reinterpret_cast<const int*>(c.ws);
  P.N = (int)(C::DUAL ? c.F : c.D);
  P.K = (int)(C::DUAL ? c.D : c.F);
  P.wtiles = (P.N + C::W_ROWS - 1) / C::W_ROWS;
  P.codes = c.ws + m.hq;
  P.sf = c.ws + m.hs;
  P.y = reinterpret_cast<float*>(c.ws + m.y);
  P.row_weight = reinterpret_cast<const float*>(c.ws + m.row_weight);
  P.parts = m.parts;
  P.part_stride = m.rows * c.D;
  P.err = c.err;
  if (m.max_tiles * P.wtiles * m.parts > INT32_MAX / 2) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: too many tiles");
  static OncePerDevice once;
  return once.run(c.dev, [] {
    cudaError_t e = cudaFuncSetAttribute(expert_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "cudaFuncSetAttribute(expert product)");
  });
}

template <class C>
int launch_product(const MoeCall& c, const ExpertParams& P) {
  const int64_t most = c.m.max_tiles * P.wtiles * (C::TRANS && !C::DUAL ? P.parts : 1);
  return launch_after(expert_kernel<C>, "expert_kernel", (unsigned)std::min<int64_t>(sm_count(), most), C::THREADS,
                      C::SMEM, c.stream, P);
}

template <class In, class Down>
int moe_run(const MoeCall& c) {
  ExpertParams in, down;
  int rc;
  if ((rc = expert_params<In>(c, in)) || (rc = expert_params<Down>(c, down))) return rc;
  const MoeLayout& m = c.m;
  int* const rows = reinterpret_cast<int*>(c.ws + m.row);
  const Plan plan = {reinterpret_cast<int*>(c.ws), reinterpret_cast<PlanTile*>(c.ws + m.tiles), rows, nullptr};
  const ScatterArgs a = {c.x, c.ldx, c.T, (int)c.k, (int)c.D, c.weights, c.ws + m.xq, c.ws + m.xs,
                         reinterpret_cast<float*>(c.ws + m.row_weight)};
  const int64_t n = c.T * c.k;
  if (n <= kFusedSlots && c.T <= kFewTokens) {
    plan_scatter_kernel<<<(unsigned)c.T, 256, 0, c.stream>>>(c.ids, (int)n, (int)c.E, m.tile, m.tile, plan, a);
    if ((rc = check_launch("plan_scatter_kernel"))) return rc;
  } else {
    if ((rc = launch_plan(c.ids, n, c.E, -1, m.tile, m.tile, plan, c.stream))) return rc;
    if ((rc = launch_after(scatter_kernel, "scatter_kernel", (unsigned)std::min<int64_t>(c.T, (int64_t)sm_count() * 8),
                           256, 0, c.stream, (const int*)rows, a)))
      return rc;
  }
  if ((rc = launch_product<In>(c, in)) || (rc = launch_product<Down>(c, down))) return rc;
  const int64_t pieces = c.T * (c.D / 8);
  return launch_after(combine_kernel, "combine_kernel",
                      (unsigned)std::min<int64_t>((pieces + 255) / 256, (int64_t)sm_count() * 8), 256, 0, c.stream,
                      (const float*)(c.ws + m.y), m.parts, m.rows * c.D, (const int*)rows, c.T, (int)c.k, (int)c.D,
                      c.out, c.ldo, (int)(aligned16(c.out) && (c.ldo % 8 == 0 || c.T == 1)));
}

}  // namespace
}  // namespace nvfp4

extern "C" int nvfp4_moe_workspace(int64_t T, int64_t k, int64_t E, int64_t D, int64_t F, int64_t* bytes) {
  using namespace nvfp4;
  if (!bytes) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_workspace: null output");
  const int rc = moe_check(T, k, E, D, F);
  if (rc) return rc;
  *bytes = T == 0 ? 0 : moe_layout(T, k, E, D, F).bytes;
  return NVFP4_OK;
}

extern "C" int nvfp4_moe_mlp(const void* x, int64_t ldx, const int32_t* ids, const float* weights, int64_t T, int64_t k,
                             int64_t E, int64_t D, int64_t F, const void* w_gate, const void* w_up, const void* sf_gate,
                             const void* sf_up, int64_t ld_in, int64_t es_in, int64_t sfe_in, const void* w_down,
                             const void* sf_down, int64_t ld_down, int64_t es_down, int64_t sfe_down, void* out,
                             int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace nvfp4;
  int rc = moe_check(T, k, E, D, F);
  if (rc) return rc;
  if (T == 0) return NVFP4_OK;
  if (!x || !ids || !weights || !out || !workspace) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: null pointer");
  if ((T > 1 && (ldx < D || ldo < D))) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: a row stride is below the row length");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 1)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_moe_mlp: fp16 pointer not 2-byte aligned");
  if ((reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) & 3)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_moe_mlp: ids and weights must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_moe_mlp: workspace not 256-byte aligned");
  MoeCall c = {static_cast<const __half*>(x), ldx, ids, weights, static_cast<__half*>(out), ldo, T, k,
               w_gate, w_up, w_down, sf_gate, sf_up, sf_down, E, D, F, ld_in, es_in, sfe_in, ld_down, es_down, sfe_down,
               moe_layout(T, k, E, D, F), static_cast<uint8_t*>(workspace), nullptr, static_cast<cudaStream_t>(stream), 0};
  const MoeLayout& m = c.m;
  if (workspace_bytes < m.bytes)
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)m.bytes);
  if ((rc = check_weights("gate", w_gate, sf_gate, E, D, ld_in, es_in, sfe_in)) ||
      (rc = check_weights("up", w_up, sf_up, E, D, ld_in, es_in, sfe_in)) ||
      (rc = check_weights("down", w_down, sf_down, E, F, ld_down, es_down, sfe_down)))
    return rc;
  cudaGetDevice(&c.dev);
  if (c.dev < 0 || c.dev >= kMaxDevices) return fail(NVFP4_ERR_UNSUPPORTED, "device index out of range");
  c.err = device_error_word();
  if (!c.err) return fail(NVFP4_ERR_CUDA, "nvfp4_moe_mlp: cannot resolve the device error word");
  using Up = ExpertCfg<false, true, 128, 1, 4>;
  // The down product's tiles: 128 weight rows where its sums are short (F), so that the boundaries between tiles weigh
  // and the accumulators of two tiles, which fit then, hide them; else 256, which read the tokens half as often.  Calls,
  // us, with 256 and with 128: F = 1024, D = 2048, 1000 tokens of 8 of 64 experts 113.2 and 105.3, D = 4096, 3000 of 4 of 32
  // 254 and 237; D = 4096, 1024 tokens of 2 of 8: F = 2048 79.4 and 76.3, 4096 106.2 and 106.6, 8192 180 and 189.
  if (!m.trans && F <= 2048) return moe_run<Up, ExpertCfg<false, false, 128, 1, 6>>(c);
  if (!m.trans) return moe_run<Up, ExpertCfg<false, false, 256, 1, 4>>(c);
  return moe_run<ExpertCfg<true, true, 16, 1, 5>, ExpertCfg<true, false, 16, 2, 5>>(c);
}
