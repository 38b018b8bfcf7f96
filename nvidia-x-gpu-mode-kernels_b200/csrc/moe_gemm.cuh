// The experts' products on the tcgen05 tensor cores: for every row tile of the
// plan (rows of one expert, ordered by expert) and every tile of the expert's
// weight rows,
//
//   gate and up (DUAL):  h = silu(x . Wg^T) * (x . Wu^T), quantised to NVFP4 in the epilogue
//   down:                y = weight[row] * (h . Wd^T), in fp32
//
// The walk over tiles reads the plan from device memory, so one launch serves
// any split of the tokens over the experts, known to the host or not.  Weights
// are [experts, rows, K/2] codes (3-D tensor map) with blocked scales
// [experts][row tiles][K/64][512 bytes] (4-D map).
//
// TRANS 0: the tokens are the MMA's 128-row operand, BN weight rows its other
// one; an epilogue thread holds one token's row.  TRANS 1, for few tokens per
// expert: 128 weight rows are the MMA's first operand and BN = 16 tokens the
// other, so the tensor cores' work shrinks with the tokens and the weights
// stream; an epilogue lane holds one weight row of every token.
//
// Warp roles: warp 0 TMA producer of the operands, warp 1 MMA, then the
// epilogue's warps, four that copy the scales into tensor memory, and the
// scales' own TMA producer (a thread needs about 50 ns to issue a box).  The
// MMA thread waits for one barrier a stage, which the operands' bytes and the
// scale warps complete: the tensor pipe holds about two MMAs ahead, so what
// the thread does between two stages must fit into their time.  Every wait is
// bounded.
//
// TRANS 0 has an epilogue warp for every 64 columns of a lane quarter of tensor memory
// (16 for 256 columns): each drains its columns into registers (64 a thread) and
// releases them, and the SiLU, quantisation and stores run under the next
// tile's products (4096 tokens, 2 of 8 experts of 4096 x 14336, gate and up:
// 547 us with 4 warps that worked their way through the columns before
// releasing them, 485 with 16; 446 with one 256-column MMA for both matrices
// and one barrier a stage).  What bounds a stage of 256 elements then is the
// round trip of the ring: 4 slots of 54 KB, all of shared memory, each taking
// 0.3 us from the MMAs' end to its refill, 1.4 us until the operands land and
// 0.28 us of MMAs.  Stages of 512 elements, two of them: 468 us.  CTA pairs (38 KB
// a stage, 5 slots; before the one MMA for both): 935 us a call against 954, the
// gate and up product alone slower (516 against 481).  Prefetching weights into
// L2: no gain.  Under minutes of such work the power
// limit takes its share, too (772 us a call before it sets in, 909 after).
#pragma once
#include "plan.cuh"
#include "quant.cuh"

namespace nvfp4 {
namespace {

struct ExpertParams {
  CUtensorMap tt, tst;              // tokens: codes [rows][K/2], scales [row tiles][K/64][128 x u32]
  CUtensorMap tw[2], tsw[2];        // weights (gate and up, or down) and their scales
  const PlanTile* tiles;
  const int* ntiles;
  int N, K;                         // weight rows of one matrix, inner dimension
  int wtiles;                       // tiles of weight rows
  int parts;                        // TRANS down: the inner dimension is cut into so many parts, each with a y of its own
  int64_t part_stride;              // of y, in elements
  uint8_t* codes;                   // DUAL: h [rows][N/2] and its blocked scales
  uint8_t* sf;
  float* y;                         // down: [rows][N]
  const float* row_weight;
  uint32_t* err;
};

template <bool TRANS_, bool DUAL_, int BN_, int KA_, int STAGES_>
struct ExpertCfg {
  static constexpr bool TRANS = TRANS_, DUAL = DUAL_;
  static constexpr int BN = BN_, KA = KA_, STAGES = STAGES_;
  static constexpr int KPS = 4 * KA;                       // 64-element K blocks per stage
  static constexpr int NW = DUAL ? 2 : 1;                  // weight matrices
  static constexpr int T_ROWS = TRANS ? BN : BM;           // tokens per tile
  static constexpr int W_ROWS = TRANS ? BM : BN;           // weight rows per tile
  static constexpr int NBW = W_ROWS / 128;                 // scale blocks of a weight tile
  static_assert(W_ROWS % 128 == 0, "weight tiles are whole scale blocks");
  static_assert(!TRANS || BN == 16, "token tiles");
  // One MMA does it where the weights are its second operand: the gate rows and the up rows of a K atom lie one
  // after the other, as its N = 2 BN rows.
  static constexpr int MMA_N = TRANS ? BN : NW * BN;
  static_assert(MMA_N <= 256, "N of an MMA");
  static constexpr int T_ATOM = T_ROWS * KSTEP_BYTES, W_ATOM = W_ROWS * KSTEP_BYTES;
  static constexpr int T_BYTES = KA * T_ATOM, W_BYTES = KA * W_ATOM;
  static constexpr int OFF_W = T_BYTES;                    // [K atom][matrix][rows]
  static constexpr int SFT_BYTES = KPS * 512;
  static constexpr int SFW_BYTES = NBW * KPS * 512;        // per weight matrix
  static constexpr int OFF_SFT = OFF_W + NW * W_BYTES;
  static constexpr int OFF_SFW = OFF_SFT + SFT_BYTES;
  static constexpr int STAGE_BYTES = (OFF_SFW + NW * SFW_BYTES + 1023) / 1024 * 1024;
  static constexpr int OFF_BAR = STAGES * STAGE_BYTES;
  static constexpr int OFF_BUF = OFF_BAR + 512;            // TRANS && DUAL: a 16 x 36 float patch per epilogue warp
  static constexpr int BUF_BYTES = TRANS && DUAL ? 4 * 16 * 36 * 4 : 0;
  static constexpr int SMEM = OFF_BUF + BUF_BYTES;
  static_assert((3 * STAGES + 4) * 8 + 4 <= 512, "barriers");
  static constexpr uint32_t OP_BYTES = T_BYTES + NW * W_BYTES;
  static constexpr uint32_t SF_BYTES = SFT_BYTES + NW * SFW_BYTES;
  // tensor memory columns
  static constexpr int BUFS = TRANS || NW * BN <= 128 ? 2 : 1;   // accumulators of two tiles where they fit
  static constexpr int ACC_COLS = NW * BN;
  static constexpr int SF_BASE = BUFS * ACC_COLS;          // the accumulators come first
  static constexpr int SFT_COLS = 4 * KPS;
  static constexpr int SFW_COLS = KPS * NW * NBW * 4;      // [K block][matrix][128 rows]
  static constexpr int SF_STAGE_COLS = SFT_COLS + SFW_COLS;
  static constexpr int TMEM_COLS = 512;
  static_assert(SF_BASE + STAGES * SF_STAGE_COLS <= TMEM_COLS, "tensor memory budget");
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert(SMEM < (1 << 18), "descriptor address field");
  static constexpr int EPI_WARPS = TRANS ? 4 : NW * BN / 16;   // 64 accumulator values a thread
  static constexpr int THREADS = 32 * (2 + EPI_WARPS + 4 + 1);   // producer, MMA, epilogue, scales, scales' producer
  static constexpr uint32_t IDESC = tc::idesc_mxf4nvf4(BM, MMA_N);
};

template <class C>
__device__ __forceinline__ void expert_mma(uint32_t tmem, uint64_t dt, uint64_t dw, uint32_t sft, uint32_t sfw,
                                           int kk, uint32_t accum) {
  const uint64_t ot = (uint64_t)((kk >> 2) * (C::T_ATOM >> 4) + 2 * (kk & 3));
  const uint64_t ow = (uint64_t)((kk >> 2) * (C::NW * C::W_ATOM >> 4) + 2 * (kk & 3));
  if (C::TRANS) {
#pragma unroll
    for (int m = 0; m < C::NW; ++m)
      tc::mma_mxf4nvf4(tmem + m * C::BN, dw + (uint64_t)(m * (C::W_ATOM >> 4)) + ow, dt + ot, C::IDESC,
                       sfw + (kk * C::NW + m) * 4, sft + 4 * kk, accum);
  } else {
    tc::mma_mxf4nvf4(tmem, dt + ot, dw + ow, C::IDESC, sft + 4 * kk, sfw + kk * C::NW * C::NBW * 4, accum);
  }
}

// silu(g) * u.  An h that lies beside the border of two 4-bit codes is decided by its last digits: the approximations
// that an fp16 result can do with (off by 2^-20 at g = -16) put outputs up to 5 times as far from the definition as 32-bit
// functions do.  e^-g = 2^t * e^d with t = -g log2(e) as rounded and d = -g - t ln(2), which a fused step gets without
// cancellation; |d| < 2^-18, so e^d is 1 + d.  The quotient gets one step of its residual.  Off by at most 12 units of
// 2^-24: 4 of ex2.approx, 4 of ln(2) at |t| = 115, one each of the product, 1 + e, the quotient and the product with u.
// Calls, us, with the approximations, with this and with CUDA's exponential and quotient: 4096 tokens of 2 of 8 experts
// of 4096 x 14336 874, 884 and 942; 333 of 4 of 16 of 1984 x 1344 45.2, 45.2 and 54.7; 64 of 8 of 64 112.7, 112.9 and 115.0.
__device__ __forceinline__ float silu_mul_32(float g, float u) {
  const float a = fmaxf(g, -80.f);         // below, |g|, |u| < 2^20 (6 * 448)^2 leave nothing that a scale of 2^-9 holds
  const float t = a * -1.4426950408889634f;
  float p, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
  const float d = fmaf(t, -0.6931471805599453f, -a);
  const float n = 1.f + fmaf(p, d, p);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(n));
  const float q = g * r;
  return fmaf(fmaf(-q, n, g), r, q) * u;
}

// Through L2: the down product's early reads come before its griddep_wait.
__device__ __forceinline__ PlanTile load_tile(const PlanTile* p) {
  const int4 a = __ldcg(reinterpret_cast<const int4*>(p));
  PlanTile q;
  q.index = a.x; q.row0 = a.y; q.first = a.z; q.tiles = a.w;
  q.rows = __ldcg(&p->rows);
  return q;
}

// Byte of the blocked scale layout that belongs to (row, 16-element block).
__device__ __forceinline__ int64_t blocked_at(int row, int block, int64_t nk64) {
  return ((int64_t)(row >> 7) * nk64 + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1) expert_kernel(const __grid_constant__ ExpertParams P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (sbase & 1023u) {  // the swizzled tiles need a 1024-aligned base; the launch guarantees it
    if (threadIdx.x == 0) atomicOr(P.err, kDevErrTimeoutMma);
    griddep_wait();
    return;
  }
  const uint32_t bar_full = sbase + C::OFF_BAR;             // operand boxes landed and scales staged in tensor memory
  const uint32_t bar_empty = bar_full + 8 * C::STAGES;      // stage consumed by the MMAs
  const uint32_t bar_sff = bar_empty + 8 * C::STAGES;       // scale boxes landed
  const uint32_t bar_accf = bar_sff + 8 * C::STAGES;        // accumulators finished, one barrier a buffer
  const uint32_t bar_acce = bar_accf + 8 * C::BUFS;         // and read
  const uint32_t tmem_slot = bar_acce + 8 * C::BUFS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 5);                       // the producer with its bytes, four scale warps
      mbar_init(bar_empty + 8 * s, 1);
      mbar_init(bar_sff + 8 * s, 1);
    }
    for (int b = 0; b < C::BUFS; ++b) {
      mbar_init(bar_accf + 8 * b, 1);
      mbar_init(bar_acce + 8 * b, C::EPI_WARPS);
    }
    fence_mbar_init();
    prefetch_tmap(&P.tt);
    prefetch_tmap(&P.tst);
#pragma unroll
    for (int m = 0; m < C::NW; ++m) {
      prefetch_tmap(&P.tw[m]);
      prefetch_tmap(&P.tsw[m]);
    }
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - sbase));
  // The down product's producer starts on weights before its predecessor, the gate and up product, has ended:
  // that one lets its dependents start only after the plan was written (below).
  const bool scales = warp == C::THREADS / 32 - 1;          // the producer of scales
  const bool early = !C::DUAL && (warp == 0 || scales);
  if (!early) {
    griddep_wait();                                         // the plan and the operands are written
    griddep_launch();
  }
  const int parts = C::TRANS && !C::DUAL ? P.parts : 1;
  const int wtiles = P.wtiles * parts;
  const int total = __ldcg(P.ntiles) * wtiles;
  const int nk64 = P.K / 64;
  const int nks = (nk64 + C::KPS - 1) / C::KPS;             // stages of a whole product
  // the stages of item t (all but the TRANS down product: all of them): parts are the fastest index
  auto from_stage = [&](int t) { return parts == 1 ? 0 : nks * (t % parts) / parts; };
  auto to_stage = [&](int t) { return parts == 1 ? nks : nks * (t % parts + 1) / parts; };

  if (warp == 0 || scales) {
    // ------------------- producers: operands, scales -------------------
    if (lane == 0) {
      const uint64_t pol_t = policy_evict_last();    // token tiles are re-read by every weight tile
      const uint64_t pol_w = policy_evict_first();
      // Stage `it` (of item t's stage ks): its weights, its tokens.  Boxes always count in full (what lies past
      // the end of a matrix or of K reads as zeros).
      auto ask_weights = [&](uint32_t it, int ks, int index, int w0) {
        const int s = it % C::STAGES;
        const uint32_t st = sbase + s * C::STAGE_BYTES;
        if (scales) {
          const uint32_t sb = bar_sff + 8 * s;
          mbar_arrive_expect_tx(sb, C::SF_BYTES);
#pragma unroll
          for (int m = 0; m < C::NW; ++m)
            tma_load_4d(st + C::OFF_SFW + m * C::SFW_BYTES, &P.tsw[m], sb, 0, C::KPS * ks, w0 / 128, index, pol_w);
        } else {
          const uint32_t fb = bar_full + 8 * s;
          mbar_arrive_expect_tx(fb, C::OP_BYTES);
#pragma unroll
          for (int a = 0; a < C::KA; ++a)
#pragma unroll
            for (int m = 0; m < C::NW; ++m)
              tma_load_3d(st + C::OFF_W + (a * C::NW + m) * C::W_ATOM, &P.tw[m], fb, (ks * C::KA + a) * KSTEP_BYTES, w0, index, pol_w);
        }
      };
      auto ask_tokens = [&](uint32_t it, int ks, int row) {
        const int s = it % C::STAGES;
        const uint32_t st = sbase + s * C::STAGE_BYTES;
        if (scales) {
          tma_load_3d(st + C::OFF_SFT, &P.tst, bar_sff + 8 * s, 0, C::KPS * ks, row / 128, pol_t);
        } else {
#pragma unroll
          for (int a = 0; a < C::KA; ++a)
            tma_load_2d(st + a * C::T_ATOM, &P.tt, bar_full + 8 * s, (ks * C::KA + a) * KSTEP_BYTES, row, pol_t);
        }
      };
      // calls body(it, ks, expert, first weight row, first token row) for every stage of this CTA until it says no
      auto walk = [&](auto body) {
        uint32_t it = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x) {
          const PlanTile q = load_tile(P.tiles + t / wtiles);
          const int local = t / parts - q.first * P.wtiles;
          const int row = q.row0 + local % q.tiles * C::T_ROWS, w0 = local / q.tiles * C::W_ROWS;
          for (int ks = from_stage(t); ks < to_stage(t); ++ks, ++it)
            if (!body(it, ks, q.index, w0, row)) return;
        }
      };
      if (early) {
        walk([&](uint32_t it, int ks, int index, int w0, int) {
          if (it == C::STAGES) return false;
          ask_weights(it, ks, index, w0);                   // the ring is empty
          return true;
        });
        griddep_wait();                                     // h is written
        griddep_launch();
      }
      walk([&](uint32_t it, int ks, int index, int w0, int row) {
        const int s = it % C::STAGES;
        if (!early || it >= C::STAGES) {
          if (!mbar_wait(bar_empty + 8 * s, ((it / C::STAGES) & 1) ^ 1, P.err, kDevErrTimeoutEmpty)) return false;
          ask_weights(it, ks, index, w0);
        }
        ask_tokens(it, ks, row);
        return true;
      });
    } else if (early) {
      griddep_wait();
      griddep_launch();
    }
  } else if (warp == 1) {
    // ------------------------------ MMA -------------------------------
    if (lane == 0) {
      const uint64_t dt0 = tc::desc_sw128(sbase), dw0 = tc::desc_sw128(sbase + C::OFF_W);
      uint32_t it = 0, tile_it = 0;
      for (int t = blockIdx.x; t < total; t += gridDim.x, ++tile_it) {
        const uint32_t buf = tile_it % C::BUFS, acc = tmem + buf * C::ACC_COLS;
        if (!mbar_wait(bar_acce + 8 * buf, ((tile_it / C::BUFS) & 1) ^ 1, P.err, kDevErrTimeoutMma)) goto done;
        tc::fence_after_sync();
        const int first = from_stage(t), last = to_stage(t);
        bool ready = false;                                 // the stage is known to be there
        for (int ks = first; ks < last; ++ks, ++it) {
          const int s = it % C::STAGES;
          const uint32_t par = (it / C::STAGES) & 1;
          if (!ready && !mbar_wait(bar_full + 8 * s, par, P.err, kDevErrTimeoutFull)) goto done;
          tc::fence_after_sync();
          const uint64_t soff = (uint64_t)((s * C::STAGE_BYTES) >> 4);
          const uint32_t sf = tmem + C::SF_BASE + s * C::SF_STAGE_COLS;
          const int nch = min(C::KPS, nk64 - C::KPS * ks);
          ready = false;
          if (nch == C::KPS) {   // a compile-time count: straight-line MMA issues
#pragma unroll
            for (int kk = 0; kk < C::KPS; ++kk) {
              // A look at the next stage while MMAs are queued: the wait, when there is nothing to wait for, costs
              // the pipe nothing.
              if (kk == C::KPS - 1 && ks + 1 < last)
                ready = mbar_test(bar_full + 8 * ((it + 1) % C::STAGES), ((it + 1) / C::STAGES) & 1);
              expert_mma<C>(acc, dt0 + soff, dw0 + soff, sf, sf + C::SFT_COLS, kk, (ks > first || kk > 0) ? 1u : 0u);
            }
          } else {
            for (int kk = 0; kk < nch; ++kk)
              expert_mma<C>(acc, dt0 + soff, dw0 + soff, sf, sf + C::SFT_COLS, kk, (ks > first || kk > 0) ? 1u : 0u);
          }
          tc::commit(bar_empty + 8 * s);
        }
        tc::commit(bar_accf + 8 * buf);
      }
    }
  } else if (warp >= 2 + C::EPI_WARPS) {
    // --------------------------- scale warps ---------------------------
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t it = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      // A narrow token tile starts anywhere in its 128-row scale block, but the MMA reads a tile's scales from
      // an aligned group of columns and from lane 0 on: they are moved there on the way to tensor memory.
      // `from`: byte of this lane's first word in a 512-byte block.
      int from = lane * 16;
      if (C::TRANS) {
        const PlanTile q = load_tile(P.tiles + t / wtiles);
        const int off = (q.row0 + (t / parts - q.first * P.wtiles) % q.tiles * C::T_ROWS) % 128;
        from = (lane + off) % 32 * 16 + off / 32 * 4;
      }
      for (int ks = from_stage(t); ks < to_stage(t); ++ks, ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(bar_sff + 8 * s, (it / C::STAGES) & 1, P.err, kDevErrTimeoutFull)) goto done;
        const uint8_t* st = smem_raw + s * C::STAGE_BYTES;
        const uint32_t sf = tmem + lane_base + C::SF_BASE + s * C::SF_STAGE_COLS;
#pragma unroll
        for (int kk = 0; kk < C::KPS; ++kk) {
          uint4 v;
          if constexpr (!C::TRANS) {
            v = *reinterpret_cast<const uint4*>(st + C::OFF_SFT + kk * 512 + from);
            tc::st_32x32b_x4(sf + 4 * kk, v.x, v.y, v.z, v.w);
          } else {                                       // one column of 16 tokens
            const uint32_t u = *reinterpret_cast<const uint32_t*>(st + C::OFF_SFT + kk * 512 + from);
            tc::st_32x32b_x2(sf + 4 * kk, u, u);
          }
#pragma unroll
          for (int m = 0; m < C::NW; ++m)
#pragma unroll
            for (int nb = 0; nb < C::NBW; ++nb) {
              v = *reinterpret_cast<const uint4*>(st + C::OFF_SFW + m * C::SFW_BYTES + (nb * C::KPS + kk) * 512 + lane * 16);
              tc::st_32x32b_x4(sf + C::SFT_COLS + ((kk * C::NW + m) * C::NBW + nb) * 4, v.x, v.y, v.z, v.w);
            }
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_full + 8 * s);
      }
    }
  } else {
    // ---------------------------- epilogue ----------------------------
    const int sub = warp & 3;                 // tensor-memory lane quarter of this warp
    uint32_t tile_it = 0;
    auto release = [&] {                      // the accumulators are read: the next tile's MMAs may start
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_acce + 8 * (tile_it % C::BUFS));
    };
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++tile_it) {
      const PlanTile q = load_tile(P.tiles + t / wtiles);
      const int local = t / parts - q.first * P.wtiles;
      const int t0 = local % q.tiles * C::T_ROWS, w0 = local / q.tiles * C::W_ROWS;
      const uint32_t acc = tmem + ((uint32_t)(sub * 32) << 16) + tile_it % C::BUFS * C::ACC_COLS;
      if (!mbar_wait(bar_accf + 8 * (tile_it % C::BUFS), (tile_it / C::BUFS) & 1, P.err, kDevErrTimeoutMma)) break;
      tc::fence_after_sync();
      if constexpr (C::TRANS && C::DUAL) {
        // lane = weight row, column = token: through a patch of shared memory, so that a lane gets one
        // token's block of 16 weight rows
        float* buf = reinterpret_cast<float*>(smem_raw + C::OFF_BUF) + sub * 16 * 36;
        const int blk = (w0 + sub * 32) / 16 + (lane & 1);
        uint32_t g[32], u[32];
        tc::ld_32x32b_x16(acc, g);
        tc::ld_32x32b_x16(acc + C::BN, u);
        tc::wait_ld();
        release();
#pragma unroll
        for (int j = 0; j < 16; ++j) buf[j * 36 + lane] = silu_mul_32(__uint_as_float(g[j]), __uint_as_float(u[j]));
        __syncwarp();
        float v[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 f = *reinterpret_cast<const float4*>(buf + (lane >> 1) * 36 + (lane & 1) * 16 + 4 * j);
          v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
        __syncwarp();
        const int tok = t0 + (lane >> 1);
        if (tok < q.rows && blk * 16 < P.N) {
          const int row = q.row0 + tok;
          uint32_t packed[2];
          const uint32_t sbyte = quant_floats(v, packed);
          *reinterpret_cast<uint2*>(P.codes + (int64_t)row * (P.N / 2) + blk * 8) = make_uint2(packed[0], packed[1]);
          P.sf[blocked_at(row, blk, P.N / 64)] = (uint8_t)sbyte;
        }
      } else if constexpr (C::TRANS) {
        const int col = w0 + sub * 32 + lane;
        float* const y = P.y + t % parts * P.part_stride;
        uint32_t v[32];
        tc::ld_32x32b_x16(acc, v);
        tc::wait_ld();
        release();
        if (col < P.N) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (t0 + j < q.rows)
              y[(int64_t)(q.row0 + t0 + j) * P.N + col] = P.row_weight[q.row0 + t0 + j] * __uint_as_float(v[j]);
        }
      } else {
        // thread = token row, warp = a quarter of the columns: all of them into registers first
        constexpr int COLS = C::NW * C::BN / (C::EPI_WARPS / 4);
        static_assert(COLS == 64, "accumulator values per thread");
        const int part = (warp - 2) >> 2;
        const int tok = t0 + sub * 32 + lane, row = q.row0 + tok;
        uint32_t v[32], u[32];
        tc::ld_32x32b_x32(acc + part * (C::DUAL ? 32 : 64), v);
        tc::ld_32x32b_x32(acc + (C::DUAL ? C::BN + part * 32 : part * 64 + 32), u);
        tc::wait_ld();
        release();
        const bool live = tok < q.rows;
        if constexpr (C::DUAL) {
          // 32 columns: two blocks of 16
          const int col0 = w0 + part * 32;           // N is a multiple of 64
          uint32_t codes[4], scales = 0;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            float h[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) h[j] = silu_mul_32(__uint_as_float(v[16 * b + j]), __uint_as_float(u[16 * b + j]));
            uint32_t packed[2];
            scales |= quant_floats(h, packed) << (8 * b);
            codes[2 * b] = packed[0];
            codes[2 * b + 1] = packed[1];
          }
          if (live && col0 < P.N) {
            *reinterpret_cast<uint4*>(P.codes + (int64_t)row * (P.N / 2) + col0 / 2) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            *reinterpret_cast<uint16_t*>(P.sf + blocked_at(row, col0 / 16, P.N / 64)) = (uint16_t)scales;
          }
        } else {
          const int col0 = w0 + part * 64;
          if (live && col0 < P.N) {
            const float weight = P.row_weight[row];
            float4* dst = reinterpret_cast<float4*>(P.y + (int64_t)row * P.N + col0);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint32_t* w = j < 8 ? v + 4 * j : u + 4 * (j - 8);
              dst[j] = make_float4(weight * __uint_as_float(w[0]), weight * __uint_as_float(w[1]),
                                   weight * __uint_as_float(w[2]), weight * __uint_as_float(w[3]));
            }
          }
        }
      }
    }
  }
done:
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

}  // namespace
}  // namespace nvfp4
