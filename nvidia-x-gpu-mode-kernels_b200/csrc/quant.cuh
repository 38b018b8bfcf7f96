// NVFP4 quantisation of one 16-element block in registers, shared by the
// quantiser and the experts' kernels: s = e4m3(amax / 6), q = e2m1(x * fl32(1/s)),
// both round-to-nearest-even with saturation; a block whose s is 0 gets zeros.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "ptx.cuh"

namespace nvfp4 {
namespace {

__device__ __forceinline__ uint32_t e2m1x2_from_f32(float lo, float hi) {
  uint32_t r;
  asm("{\n .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n cvt.u32.u8 %0, t;\n}\n"
      : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ uint32_t e4m3_from_f32(float v) {
  uint32_t r;
  asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %1, %1;\n cvt.u32.u16 %0, t;\n}\n" : "=r"(r) : "f"(v));
  return r & 0xFFu;
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  float lo, hi;
  h2_to_f2(cvt_e4m3x2(byte), lo, hi);
  return lo;
}

__device__ __forceinline__ void load_block(const __half* xp, uint32_t (&w)[8]) {
  if ((reinterpret_cast<uintptr_t>(xp) & 15u) == 0) {
    const uint4 u0 = reinterpret_cast<const uint4*>(xp)[0];
    const uint4 u1 = reinterpret_cast<const uint4*>(xp)[1];
    w[0] = u0.x; w[1] = u0.y; w[2] = u0.z; w[3] = u0.w;
    w[4] = u1.x; w[5] = u1.y; w[6] = u1.z; w[7] = u1.w;
  } else {   // any 2-byte alignment
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j] = (uint32_t)__half_as_ushort(xp[2 * j]) | ((uint32_t)__half_as_ushort(xp[2 * j + 1]) << 16);
  }
}

// Quantises one 16-element block held as 8 packed half2 words: its 16 codes in
// `packed`, element 0 in the lowest nibble; returns the scale byte.
__device__ __forceinline__ uint32_t quant_halves(const uint32_t (&w)[8], uint32_t (&packed)[2]) {
  // amax in half2: |x| and max are exact in fp16; starting from zero,
  // __hmax2 (like fmaxf) ignores NaN inputs
  __half2 m = __float2half2_rn(0.f);
#pragma unroll
  for (int j = 0; j < 8; ++j) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&w[j])));
  const float amax = fmaxf(__low2float(m), __high2float(m));
  const uint32_t sbyte = e4m3_from_f32(__fdiv_rn(amax, 6.0f));
  const float s = e4m3_to_f32(sbyte);
  packed[0] = packed[1] = 0u;
  if (s > 0.f) {
    const float inv = __fdiv_rn(1.0f, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[j]);
      const uint32_t b = e2m1x2_from_f32(__fmul_rn(__low2float(h), inv), __fmul_rn(__high2float(h), inv));
      packed[j / 4] |= b << (8 * (j % 4));
    }
  }
  return sbyte;
}

// The same for a block of 16 floats.
__device__ __forceinline__ uint32_t quant_floats(const float (&v)[16], uint32_t (&packed)[2]) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(v[j]));
  const uint32_t sbyte = e4m3_from_f32(__fdiv_rn(amax, 6.0f));
  const float s = e4m3_to_f32(sbyte);
  packed[0] = packed[1] = 0u;
  if (s > 0.f) {
    const float inv = __fdiv_rn(1.0f, s);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      packed[j / 4] |= e2m1x2_from_f32(__fmul_rn(v[2 * j], inv), __fmul_rn(v[2 * j + 1], inv)) << (8 * (j % 4));
  }
  return sbyte;
}

}  // namespace
}  // namespace nvfp4
