// What the attention kernels share: one-instruction exponential and maximum, packing of two fp32 values to 16 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ascdev {

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two values on the FMA and integer pipes, for kernels whose exponentials fill the special-function unit (16 a
// clock and SM).  x = n + f with n the nearest integer (by adding 1.5 * 2^23, whose low bits then hold n), 2^f by the
// polynomial of degree 4 with the least relative error on [-1/2, 1/2] (Remez exchange: 2.6e-6), n added to the exponent.
// x is at most 127; below -126 the result is 2^-126, which no sum next to 1 sees.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
  const float2 magic = make_float2(12582912.f, 12582912.f);
  const float2 r = __fadd2_rn(x, magic);
  const float2 n = __fadd2_rn(r, make_float2(-12582912.f, -12582912.f));
  const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  float2 p = __ffma2_rn(f, make_float2(0.009570102f, 0.009570102f), make_float2(0.05591786f, 0.05591786f));
  p = __ffma2_rn(p, f, make_float2(0.24024744f, 0.24024744f));
  p = __ffma2_rn(p, f, make_float2(0.6931218f, 0.6931218f));
  p = __ffma2_rn(p, f, make_float2(0.9999993f, 0.9999993f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (kBf16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

}  // namespace ascdev
