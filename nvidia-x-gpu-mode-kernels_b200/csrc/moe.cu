// The experts' SiLU-gated MLP on NVFP4 weights, for tokens that each chose
// their experts (nvfp4_route_experts or any other ids):
//
//   xq = nvfp4(x[t]);  h = silu(xq . Wg_e^T) * (xq . Wu_e^T);  hq = nvfp4(h)
//   out[t] = fp16( sum_j weights[t, j] * (hq . Wd_e^T) ),  e = ids[t, j], slots in order of j
//
// Five launches: the plan (plan.cuh), quantising the tokens into their rows
// (each token once, stored for each of its experts), the two expert products
// (moe_gemm.cuh) and the sum over a token's slots.  h never leaves the first
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

// Each CTA takes whole tokens: a thread quantises one 16-element block and
// stores it for each of the token's slots.
__global__ void __launch_bounds__(256) scatter_quantize_kernel(const __half* __restrict__ x, int64_t ldx, int64_t T,
                                                               int k, int D, const int* __restrict__ rows,
                                                               const float* __restrict__ weights, uint8_t* codes,
                                                               uint8_t* sf, float* row_weight) {
  const int kb = D / 16, lane = threadIdx.x & 31;
  griddep_launch();
  griddep_wait();
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    for (int c0 = threadIdx.x & ~31; c0 < kb; c0 += blockDim.x) {
      const int c = c0 + lane;
      const bool live = c < kb;
      uint32_t w[8], packed[2], sbyte = 0;
      if (live) {
        load_block(x + t * ldx + (int64_t)c * 16, w);
        sbyte = quant_halves(w, packed);
      }
      const uint32_t b1 = __shfl_down_sync(0xffffffffu, sbyte, 1);
      const uint32_t b2 = __shfl_down_sync(0xffffffffu, sbyte, 2);
      const uint32_t b3 = __shfl_down_sync(0xffffffffu, sbyte, 3);
      if (!live) continue;
      for (int j = 0; j < k; ++j) {
        const int r = rows[t * k + j];
        if (r < 0) continue;
        *reinterpret_cast<uint2*>(codes + (int64_t)r * (D / 2) + c * 8) = make_uint2(packed[0], packed[1]);
        if ((lane & 3) == 0)             // D is a multiple of 64: whole words of four blocks
          *reinterpret_cast<uint32_t*>(sf + blocked_at(r, c, D / 64)) = sbyte | (b1 << 8) | (b2 << 16) | (b3 << 24);
      }
    }
    if ((int)threadIdx.x < k) {
      const int r = rows[t * k + threadIdx.x];
      if (r >= 0) row_weight[r] = weights[t * k + threadIdx.x];
    }
  }
}

// out[t] = sum of its slots' rows of y, in slot order; eight columns a thread.
__global__ void __launch_bounds__(256) combine_kernel(const float* __restrict__ y, const int* __restrict__ rows,
                                                      int64_t T, int k, int D, __half* __restrict__ out, int64_t ldo,
                                                      int vec) {
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
      const float4* src = reinterpret_cast<const float4*>(y + (int64_t)r * D + c);
      const float4 a = src[0], b = src[1];
      acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
      acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
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
  int64_t rows, max_tiles;
  int64_t tiles, row, row_weight, xq, xs, hq, hs, y, bytes;
};

MoeLayout moe_layout(int64_t T, int64_t k, int64_t E, int64_t D, int64_t F) {
  MoeLayout m;
  const int64_t n = T * k;
  m.trans = n <= 64 * E;
  m.tile = !m.trans ? 128 : n <= 8 * E ? 16 : n <= 16 * E ? 32 : 64;
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
  m.y = take(m.rows * D * 4);
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

int weight_maps(const char* name, CUtensorMap* tw, CUtensorMap* tsw, const void* w, const void* sf, int64_t E,
                int64_t N, int64_t K, int64_t ld, int64_t es, int64_t sfe, int box_rows, int kps) {
  if (!w || !sf) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: %s: null pointer", name);
  if (ld < K / 2 || (E > 1 && (es <= 0 || sfe <= 0)))
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: %s: row stride below K/2, or an expert stride that is not positive", name);
  if (E == 1) es = N * ld, sfe = (N + 127) / 128 * (K / 64) * 512;
  if (!aligned16(w) || !aligned16(sf) || ld % 16 || es % 16 || sfe % 16)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_moe_mlp: %s: pointers and strides must be multiples of 16 bytes", name);
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
  int rc = encode_tmap(&P.tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  const uint64_t nk64 = (uint64_t)(K / 64);
  const uint64_t sdims[3] = {128, nk64, (uint64_t)(rows / 128)};
  const uint64_t sstr[2] = {512, nk64 * 512};
  const uint32_t sbox[3] = {128, (uint32_t)kps, 1};
  return encode_tmap(&P.tst, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, sf, sdims, sstr, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct MoeCall {
  const void *wg, *wu, *wd, *sg, *su, *sd;
  int64_t E, D, F;
  int64_t ld_in, es_in, sfe_in, ld_down, es_down, sfe_down;   // byte strides: rows, experts, scales of an expert
  MoeLayout m;
  uint8_t* ws;
  uint32_t* err;
  cudaStream_t stream;
};

template <class C>
int expert_product(const MoeCall& c) {
  ExpertParams P;
  std::memset(&P, 0, sizeof(P));
  const MoeLayout& m = c.m;
  int rc;
  if (C::DUAL) {
    if ((rc = token_maps(P, c.ws + m.xq, c.ws + m.xs, m.rows, c.D, C::T_ROWS, C::KPS)) ||
        (rc = weight_maps("gate", &P.tw[0], &P.tsw[0], c.wg, c.sg, c.E, c.F, c.D, c.ld_in, c.es_in, c.sfe_in, C::W_ROWS, C::KPS)) ||
        (rc = weight_maps("up", &P.tw[1], &P.tsw[1], c.wu, c.su, c.E, c.F, c.D, c.ld_in, c.es_in, c.sfe_in, C::W_ROWS, C::KPS)))
      return rc;
  } else {
    if ((rc = token_maps(P, c.ws + m.hq, c.ws + m.hs, m.rows, c.F, C::T_ROWS, C::KPS)) ||
        (rc = weight_maps("down", &P.tw[0], &P.tsw[0], c.wd, c.sd, c.E, c.D, c.F, c.ld_down, c.es_down, c.sfe_down, C::W_ROWS, C::KPS)))
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
  P.err = c.err;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(NVFP4_ERR_UNSUPPORTED, "device index out of range");
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(expert_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(expert product)");
    attr_set[dev] = true;
  }
  const int64_t most = m.max_tiles * P.wtiles;
  if (most > INT32_MAX / 2) return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: too many tiles");
  return launch_after(expert_kernel<C>, "expert_kernel", (unsigned)std::min<int64_t>(sm_count(), most), C::THREADS,
                      C::SMEM, c.stream, P);
}

template <int BN, int STAGES_IN, int STAGES_DOWN>
int expert_products_trans(const MoeCall& c) {
  const int rc = expert_product<ExpertCfg<true, true, BN, 1, STAGES_IN>>(c);
  return rc ? rc : expert_product<ExpertCfg<true, false, BN, 2, STAGES_DOWN>>(c);
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
  MoeCall c = {w_gate, w_up, w_down, sf_gate, sf_up, sf_down, E, D, F, ld_in, es_in, sfe_in, ld_down, es_down, sfe_down,
               moe_layout(T, k, E, D, F), static_cast<uint8_t*>(workspace), nullptr, static_cast<cudaStream_t>(stream)};
  const MoeLayout& m = c.m;
  if (workspace_bytes < m.bytes)
    return fail(NVFP4_ERR_INVALID, "nvfp4_moe_mlp: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)m.bytes);
  {
    // everything that can be refused is refused before the first launch
    CUtensorMap a, b;
    if ((rc = weight_maps("gate", &a, &b, w_gate, sf_gate, E, F, D, ld_in, es_in, sfe_in, 128, 4)) ||
        (rc = weight_maps("up", &a, &b, w_up, sf_up, E, F, D, ld_in, es_in, sfe_in, 128, 4)) ||
        (rc = weight_maps("down", &a, &b, w_down, sf_down, E, D, F, ld_down, es_down, sfe_down, 128, 4)))
      return rc;
  }
  c.err = device_error_word();
  if (!c.err) return fail(NVFP4_ERR_CUDA, "nvfp4_moe_mlp: cannot resolve the device error word");
  int* const rows = reinterpret_cast<int*>(c.ws + m.row);
  const Plan plan = {reinterpret_cast<int*>(c.ws), reinterpret_cast<PlanTile*>(c.ws + m.tiles), rows, nullptr};
  if ((rc = launch_plan(ids, T * k, E, -1, m.tile, m.tile, plan, c.stream))) return rc;
  const int threads = (int)std::min<int64_t>(256, (D / 16 + 31) / 32 * 32);
  if ((rc = launch_after(scatter_quantize_kernel, "scatter_quantize_kernel",
                         (unsigned)std::min<int64_t>(T, (int64_t)sm_count() * 8), threads, 0, c.stream,
                         static_cast<const __half*>(x), ldx, T, (int)k, (int)D, (const int*)rows, weights, c.ws + m.xq,
                         c.ws + m.xs, reinterpret_cast<float*>(c.ws + m.row_weight))))
    return rc;
  if (!m.trans) {
    if ((rc = expert_product<ExpertCfg<false, true, 128, 2, 2>>(c)) || (rc = expert_product<ExpertCfg<false, false, 256, 1, 4>>(c)))
      return rc;
  } else {
    rc = m.tile == 16   ? expert_products_trans<16, 5, 5>(c)
         : m.tile == 32 ? expert_products_trans<32, 4, 4>(c)
                        : expert_products_trans<64, 4, 4>(c);
    if (rc) return rc;
  }
  const int64_t pieces = T * (D / 8);
  return launch_after(combine_kernel, "combine_kernel",
                      (unsigned)std::min<int64_t>((pieces + 255) / 256, (int64_t)sm_count() * 8), 256, 0, c.stream,
                      (const float*)(c.ws + m.y), (const int*)rows, T, (int)k, (int)D, static_cast<__half*>(out), ldo,
                      (int)(aligned16(out) && (ldo % 8 == 0 || T == 1)));
}
