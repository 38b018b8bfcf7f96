// Routing of tokens to experts: scores, limit to the best groups, top-k and
// weights, one warp per token.
//
//   s_e = softmax(x)_e  or  1 / (1 + exp(-x_e))
//   c_e = s_e + bias_e                      (the choice; without a bias the experts rank by x itself,
//                                            the same order in exact arithmetic)
//   group score = sum of the group's `group_top` largest c; experts outside the `top_groups` best groups are off
//   ids = the k largest c, ties to the lowest index;  w_j = s_j / sum_j s_j * scale
//
// An expert whose logit or bias is -inf or NaN is off; +inf counts as the largest float.  Slots that no
// expert fills get id -1 and weight 0.
//
// The ids are those of 64-bit arithmetic.  Scores are evaluated in 32 bits first; each comparison that
// decides (the last group in against the first one out, and every neighbouring pair of the k + 1 best)
// must differ by more than the 32-bit evaluation can be off, otherwise the warp repeats the row in 64
// bits (256 experts with a bias, normal logits: 0.4 to 0.5 % of the rows with sigmoid, 1 % with softmax).
// Comparisons of logits alone are exact.  The same holds for a row whose chosen scores fall below the normal numbers of
// 32 bits although its weights do not (`faint`).
//
// Three forms of the 32-bit pass:
//   quick_row    rows without surprises: the lowest bits of a value carry its place, batches of rows;
//   careful_row  with a bias, any row;
//   route_row    without a bias, any row: values as unsigned keys that order like the numbers (0 = off), each maximum
//                with its lowest index; also the 64-bit pass, over double.
//
// The bytes (a row read once) are 5 us at 32768 x 256; what bounds the kernel is the issue of comparisons and
// selections: 575 instructions a row of 256 experts with a bias in 8 groups, two of three cycles issue one (41 us in a
// graph).  Keys for every row took 88 us, comparing floats 58, the short form for rows without surprises 48; weights and
// stores of several rows together and groups as runs of lanes followed.  top_k = 8 of a softmax without a bias: 17 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include "common.h"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 32;
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  int64_t T, ld;
  int E, k, groups, top_groups, group_top, group_size;
  int dtype;               // of the logits: 0 float, 1 half, 2 bfloat16
  int vec;                 // 16-byte aligned rows
  int group_lanes;         // quick_row: lanes per group, 0 where groups are no power-of-two runs of lanes
  int batch;               // rows a warp takes at a time
  int renorm;
  float scale;
};

// Order-preserving keys.  0 is below every number's key and means "off".
template <typename R> struct KeyOf;
template <> struct KeyOf<float> {
  using U = uint32_t;
  static __device__ __forceinline__ U key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);   // -0 and +0 are one value
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  }
  static __device__ __forceinline__ float value(U k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
  }
  static __device__ __forceinline__ U warp_max(U v) { return __reduce_max_sync(kAll, v); }
  static __device__ __forceinline__ float exponential(float v) { return expf(v); }
  // for the screen alone: a sigmoid of these is within 1e-6 of the exact one
  static __device__ __forceinline__ float rough_exponential(float v) { return __expf(v); }
  static __device__ __forceinline__ float rough_quotient(float a, float b) { return __fdividef(a, b); }
};
template <> struct KeyOf<double> {
  using U = unsigned long long;
  static __device__ __forceinline__ U key(double v) {
    const U b = (U)__double_as_longlong(v + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
  }
  static __device__ __forceinline__ double value(U k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
  }
  static __device__ __forceinline__ U warp_max(U v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const U w = __shfl_xor_sync(kAll, v, o);
      v = w > v ? w : v;
    }
    return v;
  }
  static __device__ __forceinline__ double exponential(double v) { return exp(v); }
  static __device__ __forceinline__ double rough_exponential(double v) { return exp(v); }
  static __device__ __forceinline__ double rough_quotient(double a, double b) { return a / b; }
};

template <typename R>
__device__ __forceinline__ R warp_sum(R v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// How far two 32-bit choices together may be off.  An approximate exponential of v is within
// (2 + 1.5 |v|) * 2^-23 relative, an approximate quotient within 2^-22; a score of 1/(1 + e^-x) or e^(x-m)/z moves
// by that times at most 1/4 (|v| s (1 - s) < 0.23) or 1 (|v| e^v < 0.37), a softmax's sum of up to 1024 terms by 16
// roundings more, the bias rounds once: 1.5e-6 for one choice, 3e-6 for two, 4e-6 with room.  A group's
// score is a sum of two.
__device__ __forceinline__ bool too_near(float hi, float lo) {
  return !(hi - lo > 4e-6f * fmaxf(1.0f, fmaxf(fabsf(hi), fabsf(lo))));
}

// Whether a chosen score s has too few digits in 32 bits: it lies below the normal numbers (0 among them), and the
// weight made of it, scale / total times as large, is more than the 64 times that leave it below 1e-36 anyway.  So it is for sigmoids
// of logits that are all below -88, and for softmaxes whose bias prefers experts far below the row's maximum.
__device__ __forceinline__ bool faint(float s, float scale, float total) {
  return s < FLT_MIN && !(fabsf(scale) <= 64.f * total);
}

// One row in R arithmetic.  x: this lane's logits (expert i * 32 + lane), -inf where off.  Returns whether
// a comparison was too near to be trusted, or a chosen score too small (R = float only); else lane j holds slot j's id and
// weight.
template <typename R, int VPL, bool SOFTMAX, bool BIAS, bool GROUPS>
__device__ bool route_row(const RouteArgs& p, const float (&x)[VPL], const float (&bias)[VPL],
                          int lane, int& id, float& weight) {
  using K = KeyOf<R>;
  using U = typename K::U;
  constexpr bool kScreen = sizeof(R) == 4;
  bool near = false;
  R m = 0, z = 0;
  if (SOFTMAX) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) mx = fmaxf(mx, x[i]);
    const uint32_t mk = __reduce_max_sync(kAll, KeyOf<float>::key(mx));
    m = (R)KeyOf<float>::value(mk);
    if (BIAS || GROUPS || !p.renorm) {
      R part = 0;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (x[i] > -INFINITY) part += K::exponential((R)x[i] - m);
      z = warp_sum(part);
    }
  }
  auto score = [&](float v) -> R {      // of an expert that is on
    if (SOFTMAX) return K::exponential((R)v - m) / z;
    return (R)1 / ((R)1 + K::exponential(-(R)v));
  };
  auto rough_score = [&](float v) -> R {
    if (SOFTMAX) return K::rough_quotient(K::rough_exponential((R)v - m), z);
    return K::rough_quotient((R)1, (R)1 + K::rough_exponential(-(R)v));
  };
  U key[VPL];
  if (BIAS || GROUPS) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      key[i] = 0;
      if (x[i] > -INFINITY) {
        const R c = BIAS ? rough_score(x[i]) + (R)bias[i] : rough_score(x[i]);
        key[i] = K::key(c);
      }
    }
  }
  if (GROUPS) {
    U mine = 0;                          // lane g: group g's score
    // top, next: this lane's two largest of the group
    auto group_score = [&](int g, U top, U next) {
      const U first = K::warp_max(top);
      R sum = K::value(first);
      if (p.group_top == 2) {
        // the second largest: the (lowest) lane that holds the largest offers its next
        const unsigned holders = __ballot_sync(kAll, top == first);
        if (lane == __ffs(holders) - 1) top = next;
        const U second = K::warp_max(top);
        if (second) sum += K::value(second);
      }
      if (lane == g && first) mine = K::key(sum);
    };
    // groups of 32, 64 or 128 experts are 1, 2 or 4 whole registers: compile-time loops, whose warp-wide
    // maxima overlap
    auto by_registers = [&](auto regs) {
      constexpr int RPG = decltype(regs)::value;
#pragma unroll
      for (int g = 0; g * RPG < VPL; ++g) {
        U top = 0, next = 0;
#pragma unroll
        for (int i = g * RPG; i < (g + 1) * RPG && i < VPL; ++i) {
          next = key[i] > top ? top : (key[i] > next ? key[i] : next);
          top = key[i] > top ? key[i] : top;
        }
        group_score(g, top, next);
      }
    };
    if (kScreen && p.group_size == 32) {
      by_registers(std::integral_constant<int, 1>());
    } else if (kScreen && p.group_size == 64) {
      by_registers(std::integral_constant<int, 2>());
    } else if (kScreen && p.group_size == 128) {
      by_registers(std::integral_constant<int, 4>());
    } else {
      for (int g = 0; g < p.groups; ++g) {
        U top = 0, next = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const int e = i * 32 + lane - g * p.group_size;
          if (e < 0 || e >= p.group_size) continue;
          next = key[i] > top ? top : (key[i] > next ? key[i] : next);
          top = key[i] > top ? key[i] : top;
        }
        group_score(g, top, next);
      }
    }
    unsigned chosen = 0;
    U last = 0;
    for (int q = 0; q < p.top_groups; ++q) {
      const U best = K::warp_max((chosen >> lane) & 1 ? 0 : mine);
      if (best == 0) break;
      const unsigned at = __ballot_sync(kAll, mine == best && !((chosen >> lane) & 1));
      chosen |= at & (0u - at);
      last = best;
    }
    if (kScreen && last) {
      const U out = K::warp_max((chosen >> lane) & 1 ? 0 : mine);
      if (out) near = near || too_near((float)K::value(last) * 0.5f, (float)K::value(out) * 0.5f);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i * 32 + lane < p.E && !((chosen >> ((i * 32 + lane) / p.group_size)) & 1)) key[i] = 0;
  }
  if (!BIAS) {                           // experts rank by their logits, exactly
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      key[i] = (x[i] > -INFINITY && (!GROUPS || key[i])) ? K::key((R)x[i]) : 0;
  }
  // Each lane keeps its DEPTH largest in order; a lane whose DEPTH have all been taken looks for the next
  // ones below the last taken (rare: of 256 experts' 8 best, 3 share a lane in one row of twenty).
  constexpr int DEPTH = VPL < 3 ? VPL : 3;
  U top[DEPTH];
  unsigned at[DEPTH];
  auto refill = [&](U below, unsigned after) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) top[d] = 0, at[d] = ~0u;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const unsigned e = i * 32 + lane;
      U v = key[i] < below || (key[i] == below && e > after) ? key[i] : 0;
      unsigned w = e;
      // strictly larger goes first and moves all that follow down by one: equal ones stay in index order
      bool up = false;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        up = up || v > top[d];
        const U tv = top[d];
        const unsigned tw = at[d];
        top[d] = up ? v : tv;
        at[d] = up ? w : tw;
        v = up ? tv : v;
        w = up ? tw : w;
      }
    }
  };
  refill(~(U)0, ~0u);
  int taken = 0;
  id = -1;
  U before = 0;
  const int rounds = kScreen && BIAS ? p.k + 1 : p.k;   // the screen also looks at the first one left out
  for (int j = 0; j < rounds; ++j) {
    const U best = K::warp_max(top[0]);
    if (best == 0) break;
    if (kScreen && BIAS) {
      if (j) near = near || too_near((float)K::value(before), (float)K::value(best));
      before = best;
    }
    if (j == p.k) break;
    const unsigned e = __reduce_min_sync(kAll, top[0] == best ? at[0] : ~0u);
    if (lane == j) id = (int)e;
    if (lane == (int)(e & 31)) {
#pragma unroll
      for (int d = 0; d + 1 < DEPTH; ++d) top[d] = top[d + 1], at[d] = at[d + 1];
      top[DEPTH - 1] = 0;
      if (VPL > DEPTH && ++taken == DEPTH) {
        taken = 0;
        refill(best, e);
      }
    }
  }
  if (kScreen && near) return true;
  // weights: lane j fetches its expert's logit from the lane that holds it
  float lx = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float v = __shfl_sync(kAll, x[i], id & 31);
    if (id >= 0 && (id >> 5) == i) lx = v;
  }
  R w = 0;
  if (id >= 0) {
    if (SOFTMAX) {
      w = K::exponential((R)lx - m);
      if (!p.renorm) w /= z;
    } else {
      w = score(lx);
    }
  }
  const R total = p.renorm ? warp_sum(w) : (R)1;
  if (kScreen && __any_sync(kAll, id >= 0 && faint((float)w, p.scale, (float)total))) return true;
  if (p.renorm) w = total > 0 ? w / total : (R)0;
  weight = (float)(w * (R)p.scale);
  return false;
}

// Row t's logits as they are, expert i * 32 + lane in x[i]; -inf past the last expert.
template <int VPL>
__device__ __forceinline__ void load_raw(const RouteArgs& p, int64_t t, int lane, float (&x)[VPL]) {
  const bool full = p.E == VPL * 32;
#pragma unroll
  for (int i = 0; i < VPL; ++i) x[i] = -INFINITY;
  if (p.dtype == 0) {
    const float* row = static_cast<const float*>(p.logits) + t * p.ld + lane;
    if (full) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) x[i] = row[i * 32];
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i * 32 + lane < p.E) x[i] = row[i * 32];
    }
  } else if (p.dtype == 1) {
    const __half* row = static_cast<const __half*>(p.logits) + t * p.ld + lane;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i * 32 + lane < p.E) x[i] = __half2float(row[i * 32]);
  } else {
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.logits) + t * p.ld + lane;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (i * 32 + lane < p.E) x[i] = __bfloat162float(row[i * 32]);
  }
}

// The same, -inf where the expert is off, at most the largest float.
template <int VPL, bool BIAS>
__device__ __forceinline__ void load_row(const RouteArgs& p, int64_t t, int lane, const float (&bias)[VPL],
                                         float (&x)[VPL]) {
  load_raw<VPL>(p, t, lane, x);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    x[i] = x[i] > -INFINITY ? fminf(x[i], FLT_MAX) : -INFINITY;       // NaN is off
    if (BIAS && !(bias[i] > -INFINITY)) x[i] = -INFINITY;
  }
}

template <int VPL, bool BIAS>
__device__ __forceinline__ void load_bias(const RouteArgs& p, int lane, float (&bias)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    bias[i] = BIAS && i * 32 + lane < p.E ? p.bias[i * 32 + lane] : 0.f;
    bias[i] = bias[i] > -INFINITY ? bias[i] : -INFINITY;     // NaN: off, too
  }
}

__device__ __forceinline__ void store_row(const RouteArgs& p, int64_t t, int lane, int id, float w) {
  if (lane < p.k) {
    p.ids[t * p.k + lane] = id;
    p.weights[t * p.k + lane] = w;
  }
}

// A row that 32 bits could not decide, from the start: a function of its own, so that the common path keeps
// none of it in registers.
template <int VPL, bool SOFTMAX, bool BIAS, bool GROUPS>
__device__ __noinline__ void route_row_in_64_bits(const RouteArgs& p, int64_t t, int lane) {
  float bias[VPL], x[VPL];
  load_bias<VPL, BIAS>(p, lane, bias);
  load_row<VPL, BIAS>(p, t, lane, bias, x);
  int id;
  float w;
  route_row<double, VPL, SOFTMAX, BIAS, GROUPS>(p, x, bias, lane, id, w);
  store_row(p, t, lane, id, w);
}

__device__ __forceinline__ float warp_max_float(float v) {      // no NaN among the values
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The 32-bit pass over a row with a bias, where every choice is approximate anyway: floats instead of keys
// (-inf: off), and the lowest bits of a choice replaced by its place in the lane, so that a lane's choices
// differ and carry their index.  That moves a choice by less than VPL units of 2^-23 relative.  Two forms of it:
// quick_row for rows without surprises, careful_row for all.
enum RowState { kDone, kOdd, kNear };   // kOdd: not for quick_row; kNear: a comparison is too near or a score too small, 64 bits must decide

constexpr float kLog2e = 1.4426950408889634f;

template <int VPL>
__device__ __forceinline__ bool near_choices(float hi, float lo) {
  constexpr float kTol = 4e-6f + 2 * VPL * 1.2e-7f;
  return !(hi - lo > kTol * fmaxf(1.f, fmaxf(fabsf(hi), fabsf(lo))));
}

__device__ __forceinline__ float raw_logit(const RouteArgs& p, int64_t t, int e) {
  const int64_t from = t * p.ld + e;
  return p.dtype == 0   ? static_cast<const float*>(p.logits)[from]
         : p.dtype == 1 ? __half2float(static_cast<const __half*>(p.logits)[from])
                        : __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[from]);
}
// Of an expert that is on (so not NaN), as the passes see it.
__device__ __forceinline__ float logit_at(const RouteArgs& p, int64_t t, int e) { return fminf(raw_logit(p, t, e), FLT_MAX); }

// Any row, expert i * 32 + lane in register i.
template <int VPL, bool SOFTMAX, bool GROUPS>
__device__ __noinline__ RowState careful_row(const RouteArgs& p, int64_t t, int lane, float2* slots) {
  constexpr uint32_t kPlace = VPL - 1;
  float bias[VPL], c[VPL];
  load_bias<VPL, true>(p, lane, bias);
  load_row<VPL, true>(p, t, lane, bias, c);
  float m = 0.f;
  if (SOFTMAX) {
    float mx = c[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) mx = fmaxf(mx, c[i]);
    m = warp_max_float(mx);
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {      // a row that is off as a whole has NaN here, and no expert that is on
      const float e = exp2_approx((c[i] - m) * kLog2e);
      z += c[i] > -INFINITY ? e : 0.f;
      c[i] = c[i] > -INFINITY ? e : -INFINITY;
    }
    z = reciprocal_approx(warp_sum(z));
#pragma unroll
    for (int i = 0; i < VPL; ++i) c[i] *= z;
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float s = reciprocal_approx(1.f + exp2_approx(c[i] * -kLog2e));
      c[i] = c[i] > -INFINITY ? s : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float v = c[i] + fminf(bias[i], FLT_MAX);
    c[i] = c[i] > -INFINITY ? __uint_as_float((__float_as_uint(v) & ~kPlace) | (kPlace - i)) : -INFINITY;
  }
  if (GROUPS) {
    float mine = -INFINITY;              // lane g: group g's score
    for (int g = 0; g < p.groups; ++g) {
      float top = -INFINITY, next = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = i * 32 + lane - g * p.group_size;
        const float v = e >= 0 && e < p.group_size ? c[i] : -INFINITY;
        next = fmaxf(next, fminf(top, v));
        top = fmaxf(top, v);
      }
      const float first = warp_max_float(top);
      float sum = first;
      if (p.group_top == 2) {
        // the second largest: the lowest lane that holds the largest offers its next
        if (lane == __ffs(__ballot_sync(kAll, top == first)) - 1) top = next;
        const float second = warp_max_float(top);
        if (second > -INFINITY) sum += second;
      }
      if (lane == g) mine = sum;
    }
    unsigned chosen = 0;
    float last = -INFINITY;
    for (int q = 0; q < p.top_groups; ++q) {
      const bool open = !((chosen >> lane) & 1);
      const float best = warp_max_float(open ? mine : -INFINITY);
      if (best == -INFINITY) break;
      const unsigned at = __ballot_sync(kAll, open && mine == best);
      chosen |= at & (0u - at);
      last = best;
    }
    const float out = warp_max_float((chosen >> lane) & 1 ? -INFINITY : mine);
    if (out > -INFINITY && near_choices<VPL>(0.5f * last, 0.5f * out)) return kNear;
#pragma unroll
    for (int i = 0; i < VPL; ++i) c[i] = (chosen >> min((i * 32 + lane) / p.group_size, 31)) & 1 ? c[i] : -INFINITY;
  }
  // Each lane keeps its DEPTH largest in order; a lane whose DEPTH have all been taken looks for the next ones
  // below the last taken.
  constexpr int DEPTH = VPL < 3 ? VPL : 3;
  float top[DEPTH];
  auto fill = [&](float limit) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) top[d] = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      float v = c[i] < limit ? c[i] : -INFINITY;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const float lower = fminf(top[d], v);
        top[d] = fmaxf(top[d], v);
        v = lower;
      }
    }
  };
  fill(INFINITY);
  int taken = 0;
  unsigned all_taken = 0;
  if (lane < p.k) slots[lane] = make_float2(-INFINITY, 0.f);
  __syncwarp();
  for (int j = 0; j < p.k; ++j) {
    const float best = warp_max_float(top[0]);
    if (best == -INFINITY) break;
    if (top[0] == best) {                // one lane; two where choices are equal, found below
      slots[j] = make_float2(best, __int_as_float(lane));
#pragma unroll
      for (int d = 0; d + 1 < DEPTH; ++d) top[d] = top[d + 1];
      top[DEPTH - 1] = -INFINITY;
      ++all_taken;
      if (VPL > DEPTH && ++taken == DEPTH) {
        taken = 0;
        fill(best);
      }
    }
  }
  const float left_out = warp_max_float(top[0]);
  __syncwarp();
  const float2 slot = lane < p.k ? slots[lane] : make_float2(-INFINITY, 0.f);
  const float mine = slot.x;
  const bool on = mine > -INFINITY;
  if ((int)__reduce_add_sync(kAll, all_taken) != __popc(__ballot_sync(kAll, on))) return kNear;      // equal choices
  const float up = __shfl_up_sync(kAll, mine, 1);
  bool bad = on && lane > 0 && near_choices<VPL>(up, mine);
  if (lane == p.k - 1 && left_out > -INFINITY) bad = bad || near_choices<VPL>(mine, left_out);
  if (__any_sync(kAll, bad)) return kNear;
  const int id = on ? (int)(kPlace - (__float_as_uint(mine) & kPlace)) * 32 + __float_as_int(slot.y) : -1;
  float w = 0.f;
  if (on) {
    const float x = logit_at(p, t, id);
    w = SOFTMAX ? expf(x - m) : 1.f / (1.f + expf(-x));
  }
  const float total = p.renorm ? warp_sum(w) : 1.f;
  if (__any_sync(kAll, on && faint(w, p.scale, total))) return kNear;
  if (p.renorm) w = total > 0.f ? w / total : 0.f;
  store_row(p, t, lane, id, w * p.scale);
  return kDone;
}

// A row none of whose experts is off or has a logit below -88, without equal maxima, and with at most DEPTH of the
// k best in one lane (kOdd where that does not hold).  Such rows are bound by the ALU pipe (comparisons and
// selections, half the rate of the others), so the form has few of them: expert lane * VPL + i is in register
// i, a group then is a run of lanes, and all groups' scores come from one pass over the registers and log2(lanes)
// exchanges (25 instructions a group as maxima over the warp before).  The choices (without a bias the logits
// themselves, which are only as approximate as the place in their lowest bits makes them) go to slots[0..k) as
// (value, lane); `m` is the row's maximum (SOFTMAX with BIAS or GROUPS), left_out the best choice that is left.
template <int VPL>
__device__ __forceinline__ void load_run(const RouteArgs& p, int64_t t, int lane, float (&x)[VPL]) {
  const int64_t from = t * p.ld + lane * VPL;
  if (p.E != VPL * 32) {                 // zeros past the last expert
#pragma unroll
    for (int i = 0; i < VPL; ++i) x[i] = lane * VPL + i < p.E ? raw_logit(p, t, lane * VPL + i) : 0.f;
  } else if (p.dtype == 0) {
    const float* row = static_cast<const float*>(p.logits) + from;
    if (VPL % 4 == 0 && p.vec) {
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const float4 v = reinterpret_cast<const float4*>(row)[i];
        x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) x[i] = row[i];
    }
  } else {
    const uint16_t* row = static_cast<const uint16_t*>(p.logits) + from;
    auto value = [&](uint32_t bits) {
      return p.dtype == 1 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
    };
    if (VPL % 8 == 0 && p.vec) {
#pragma unroll
      for (int i = 0; i < VPL / 8; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(row)[i];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[8 * i + j] = value(w[j / 2] >> (16 * (j & 1)) & 0xffffu);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) x[i] = value(row[i]);
    }
  }
}

template <int VPL, bool SOFTMAX, bool BIAS, bool GROUPS>
__device__ __forceinline__ RowState quick_row(const RouteArgs& p, int lane, float (&c)[VPL], const float (&bias)[VPL],
                                              float2* slots, float& m, float& left_out) {
  constexpr uint32_t kPlace = VPL - 1;
  float x[VPL];                          // what ranks without a bias
  if (!BIAS) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) x[i] = c[i];
  }
  if (BIAS || GROUPS) {
    if (SOFTMAX) {
      float mx = c[0];
#pragma unroll
      for (int i = 1; i < VPL; ++i) mx = fmaxf(mx, lane * VPL + i < p.E ? c[i] : mx);
      m = warp_max_float(lane * VPL < p.E ? mx : -INFINITY);
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        // NaN from a logit of NaN or an infinity, 1/0 * 0 from one too far below (its exponential is 0)
        const float e = exp2_approx((c[i] - m) * kLog2e);
        z += lane * VPL + i < p.E ? e : 0.f;
        c[i] = fmaf(reciprocal_approx(e), 0.f, e);
      }
      z = reciprocal_approx(warp_sum(z));
#pragma unroll
      for (int i = 0; i < VPL; ++i) c[i] = fmaf(c[i], z, BIAS ? bias[i] : 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        // a logit of +inf scores 1; NaN from a logit of NaN, inf * 0 from one that is -inf or below -88
        const float e = exp2_approx(c[i] * -kLog2e);
        c[i] = fmaf(e, 0.f, reciprocal_approx(1.f + e) + (BIAS ? bias[i] : 0.f));
      }
    }
  }
  float any = 0.f;                       // NaN if one of them is, or if a logit that ranks is infinite
#pragma unroll
  for (int i = 0; i < VPL; ++i) any = fmaf(c[i], 0.f, any);
  if (!BIAS && GROUPS) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) any = fmaf(x[i], 0.f, any);
  }
  if (__any_sync(kAll, !(any == 0.f))) return kOdd;
  if (BIAS || !GROUPS) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) c[i] = __uint_as_float((__float_as_uint(c[i]) & ~kPlace) | (kPlace - i));
  }
  if (p.E != VPL * 32) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) c[i] = lane * VPL + i < p.E ? c[i] : -INFINITY;
  }
  if (GROUPS) {
    float top = c[0], next = -INFINITY;
#pragma unroll
    for (int i = 1; i < VPL; ++i) {
      next = fmaxf(next, fminf(top, c[i]));
      top = fmaxf(top, c[i]);
    }
    for (int o = 1; o < p.group_lanes; o <<= 1) {
      const float t2 = __shfl_xor_sync(kAll, top, o), n2 = __shfl_xor_sync(kAll, next, o);
      next = fmaxf(fmaxf(next, n2), fminf(top, t2));
      top = fmaxf(top, t2);
    }
    // every lane holds its group's score; -inf once the group is chosen
    float mine = p.group_top == 2 && p.group_size > 1 ? top + next : top;
    bool chosen = false;
    float last = 0.f;
    for (int q = 0; q < p.top_groups; ++q) {
      last = warp_max_float(mine);
      if (mine == last) {                // one group; more where scores are equal, found below
        chosen = true;
        mine = -INFINITY;
      }
    }
    const float out = warp_max_float(mine);
    if (__popc(__ballot_sync(kAll, chosen)) != p.top_groups * p.group_lanes) return kNear;
    if (out > -INFINITY && near_choices<VPL>(0.5f * last, 0.5f * out)) return kNear;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (!BIAS) c[i] = __uint_as_float((__float_as_uint(x[i]) & ~kPlace) | (kPlace - i));
      c[i] = chosen ? c[i] : -INFINITY;
    }
  }
  constexpr int DEPTH = VPL < 4 ? VPL : 4;
  float top[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) top[d] = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float v = c[i];
#pragma unroll
    for (int d = 0; d < DEPTH && d <= i; ++d) {
      const float lower = fminf(top[d], v);
      top[d] = fmaxf(top[d], v);
      v = lower;
    }
  }
  unsigned taken = 0;
  for (int j = 0; j < p.k; ++j) {
    const float best = warp_max_float(top[0]);
    if (top[0] == best) {                // one lane; more where choices are equal or have run out, found below
      slots[j] = make_float2(best, __int_as_float(lane));
#pragma unroll
      for (int d = 0; d + 1 < DEPTH; ++d) top[d] = top[d + 1];
      top[DEPTH - 1] = -INFINITY;
      ++taken;
    }
  }
  left_out = warp_max_float(top[0]);
  // an exhausted lane may hold more of the best than it offered
  if (VPL > DEPTH && __any_sync(kAll, taken >= DEPTH)) return kOdd;
  return __reduce_add_sync(kAll, taken) == (unsigned)p.k ? kDone : kNear;
}

// A row that quick_row left, without a bias: keys, exact in 32 bits but for the groups' scores.
template <int VPL, bool SOFTMAX, bool BIAS, bool GROUPS>
__device__ __noinline__ void keyed_row(const RouteArgs& p, int64_t t, int lane) {
  float bias[VPL], x[VPL];
  load_bias<VPL, BIAS>(p, lane, bias);
  load_row<VPL, BIAS>(p, t, lane, bias, x);
  int id;
  float w;
  if (route_row<float, VPL, SOFTMAX, BIAS, GROUPS>(p, x, bias, lane, id, w))
    route_row_in_64_bits<VPL, SOFTMAX, BIAS, GROUPS>(p, t, lane);
  else
    store_row(p, t, lane, id, w);
}

// A warp takes `batch` neighbouring rows at a time: quick_row one after the other, then the weights and stores of
// all of them together, row b's slot j in lane b * width + j; then the rows that quick_row left.
template <int VPL, bool SOFTMAX, bool BIAS, bool GROUPS>
__global__ void __launch_bounds__(256, VPL <= 8 ? 4 : VPL == 16 ? 2 : 1) route_kernel(const __grid_constant__ RouteArgs p) {
  constexpr uint32_t kPlace = VPL - 1;
  __shared__ float2 all_slots[8][kMaxTopK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5), me = (int64_t)blockIdx.x * (blockDim.x >> 5) + warp;
  float2* const slots = all_slots[warp];
  float bias[VPL];
  // softmax weights as they are want an accurate sum over all experts, which the keyed pass has
  const bool keyed = !BIAS || (SOFTMAX && !p.renorm);
  // 16-bit logits that rank by themselves are often equal, and a row is then tried in vain: it counts where a warp has no
  // other row, and for bfloat16 the more of the best there are.  us with the short form first and without it:
  //   one row a warp    4097 x 60 fp16 5.1 and 4.4, bf16 5.2 and 4.6; 64 x 256 5.5 and 4.4, 5.6 and 4.5
  //   fp16, batches     32768 x 256, k = 8 22.9 and 33.7, k = 16 36.6 and 41.7; x 60, k = 4 13.9 and 21.8; 9500 x 256 10.6 and 13.8
  //   bf16, k = 4       32768 x 256 24.6 and 33.4, x 60 16.9 and 23.7; 12000 x 256 13.4 and 13.9, x 128 11.3 and 11.1
  //   bf16, k = 6, 8    32768 x 256 35.1 and 34.3, x 32 17.6 and 19.6; 12000 x 60 11.9 and 10.3, x 128 14.8 and 13.1
  //   bf16, 8 groups    32768 x 256, k = 8 67.1 and 82.8, k = 12 95.4 and 81.6; 12000 x 256, k = 8 33.3 and 39.2
  const bool ties = !BIAS && p.dtype != 0 && (p.batch == 1 || (p.dtype == 2 && p.k > (GROUPS ? 8 : 4)));
  bool odd = ties || (GROUPS && p.group_lanes == 0) || (SOFTMAX && !p.renorm);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    bias[i] = BIAS && lane * VPL + i < p.E ? p.bias[lane * VPL + i] : 0.f;
    odd = odd || !(bias[i] > -INFINITY);                 // off by its bias
    bias[i] = fminf(bias[i], FLT_MAX);                   // the 64-bit pass tells it from +inf
  }
  odd = __any_sync(kAll, odd);
  const int shift = p.k <= 4 ? 2 : p.k <= 8 ? 3 : p.k <= 16 ? 4 : 5, width = 1 << shift;
  for (int64_t t0 = me * p.batch; t0 < p.T; t0 += warps * p.batch) {
    const int rows = (int)min((int64_t)p.batch, p.T - t0);
    unsigned odd_rows = odd ? (1u << rows) - 1 : 0, near_rows = 0;
    if (!odd) {
      float m = 0.f, left_out = -INFINITY;               // of this lane's row below
      float c[VPL], ahead[VPL];
      load_run<VPL>(p, t0, lane, ahead);
      for (int b = 0; b < rows; ++b) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] = ahead[i];
        if (b + 1 < rows) load_run<VPL>(p, t0 + b + 1, lane, ahead);
        float row_m = 0.f, row_out = -INFINITY;
        const RowState state = quick_row<VPL, SOFTMAX, BIAS, GROUPS>(p, lane, c, bias, slots + b * width, row_m, row_out);
        if (state == kOdd) odd_rows |= 1u << b;
        if (state == kNear) near_rows |= 1u << b;
        if (lane >> shift == b) m = row_m, left_out = row_out;
      }
      __syncwarp();
      const int b = lane >> shift, j = lane & (width - 1);
      const bool on = j < p.k && b < rows && !(((odd_rows | near_rows) >> b) & 1);
      const float2 slot = on ? slots[lane] : make_float2(0.f, 0.f);
      const float mine = slot.x;
      const float up = __shfl_up_sync(kAll, mine, 1);
      bool bad = on && ((j > 0 && near_choices<VPL>(up, mine)) ||
                        (j == p.k - 1 && left_out > -INFINITY && near_choices<VPL>(mine, left_out)));
      const int id = (int)(__float_as_int(slot.y) * VPL + (kPlace - (__float_as_uint(mine) & kPlace)));
      const float x = on ? logit_at(p, t0 + b, id) : 0.f;
      if (SOFTMAX && !BIAS && !GROUPS) m = __shfl_sync(kAll, x, b << shift);      // the best of all
      float w = !on ? 0.f : SOFTMAX ? expf(x - m) : 1.f / (1.f + expf(-x));
      float total = 1.f;
      if (p.renorm) {
        total = w;
        for (int o = width / 2; o; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
      }
      bad = bad || (on && faint(w, p.scale, total));
      if (p.renorm) w = total > 0.f ? w / total : 0.f;
      const unsigned bad_lanes = __ballot_sync(kAll, bad);
      const unsigned first_row = width == 32 ? kAll : (1u << width) - 1;
      if (on && !(bad_lanes & (first_row << (b << shift)))) {
        p.ids[(t0 + b) * p.k + j] = id;
        p.weights[(t0 + b) * p.k + j] = w * p.scale;
      }
      for (int r = 0; r < rows; ++r)
        if (bad_lanes & (first_row << (r << shift))) near_rows |= 1u << r;
      __syncwarp();
    }
    if (keyed) {
      for (unsigned left = odd_rows | near_rows; left; left &= left - 1)
        keyed_row<VPL, SOFTMAX, BIAS, GROUPS>(p, t0 + __ffs(left) - 1, lane);
    } else if constexpr (BIAS) {
      for (unsigned left = odd_rows; left; left &= left - 1) {
        const int r = __ffs(left) - 1;
        if (careful_row<VPL, SOFTMAX, GROUPS>(p, t0 + r, lane, slots) == kNear) near_rows |= 1u << r;
        __syncwarp();
      }
      for (unsigned left = near_rows; left; left &= left - 1)
        route_row_in_64_bits<VPL, SOFTMAX, BIAS, GROUPS>(p, t0 + __ffs(left) - 1, lane);
    }
  }
}

template <int VPL>
int launch_route(const RouteArgs& p, bool softmax, cudaStream_t stream) {
  using Fn = void (*)(const RouteArgs);
  const bool b = p.bias != nullptr, g = p.groups > 1;
  static const Fn table[8] = {
      route_kernel<VPL, false, false, false>, route_kernel<VPL, false, false, true>,
      route_kernel<VPL, false, true, false>,  route_kernel<VPL, false, true, true>,
      route_kernel<VPL, true, false, false>,  route_kernel<VPL, true, false, true>,
      route_kernel<VPL, true, true, false>,   route_kernel<VPL, true, true, true>};
  RouteArgs q = p;
  const int lanes = p.group_size / VPL;
  q.group_lanes = g && p.group_size % VPL == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  // as many rows a batch as its lanes hold, if that leaves every SM its 32 warps
  const int most = p.k <= 4 ? 8 : p.k <= 8 ? 4 : p.k <= 16 ? 2 : 1;
  q.batch = (int)std::max<int64_t>(1, std::min<int64_t>(most, p.T / ((int64_t)sm_count() * 32)));
  const int64_t ctas = std::min<int64_t>((p.T + 8 * q.batch - 1) / (8 * q.batch), (int64_t)sm_count() * 8);
  table[softmax * 4 + b * 2 + g]<<<(unsigned)ctas, 256, 0, stream>>>(q);
  return check_launch("route_kernel");
}

}  // namespace
}  // namespace nvfp4
