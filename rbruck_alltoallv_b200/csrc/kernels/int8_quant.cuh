// Rows of bf16 as 8-bit integers: the steps that the quantiser and the linear of a few rows share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rbv {
namespace quant {

// Largest magnitudes of the even and the odd ones of eight values; a NaN stays.
__device__ __forceinline__ __nv_bfloat162 vec_max(uint4 v, __nv_bfloat162 m) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  #pragma unroll
  for (int j = 0; j < 4; j++) m = __hmax2_nan(m, __habs2(h[j]));
  return m;
}
__device__ __forceinline__ float no_nan(float m) { return m == m ? m : INFINITY; }

// What a row with the largest magnitude m (an infinity also for a NaN) is divided by.
struct RowScale {
  float scale, s, inv;                     // what the row's integers stand for; the divisor and its reciprocal
  bool zero;                               // the integers are all zero
  __device__ __forceinline__ explicit RowScale(float m) {
    const bool bad = m == INFINITY;
    zero = bad || m < 0x1p-100f;
    s = zero ? 1.0f : __fdiv_rn(m, 127.0f);
    inv = zero ? 0.0f : __frcp_rn(s);
    scale = bad ? __int_as_float(0x7fffffff) : s;
  }
};

__device__ __forceinline__ unsigned quantize_slowly(float x, float s) {
  return (unsigned)max(-127, min(127, __float2int_rn(__fdiv_rn(x, s))));
}

// Two 32-bit numbers in one register pair: a * b + c of both with one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}

// t = x * inv is within 2^-22 of x / s, relatively, and |t| <= 127.01: where t is further than 2^-14 from a half both round alike.
// Adding 1.5 * 2^23 (to the exact product, in one fused step) rounds t to an integer, which then stands in the low byte.
__device__ __forceinline__ uint2 quantize_vec(uint4 v, const RowScale& row) {
  const float s = row.s, inv = row.inv;
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  constexpr float kMagic = 12582912.0f;
  const float2 magic = make_float2(kMagic, kMagic), inv2 = make_float2(inv, inv), minus = make_float2(-1.0f, -1.0f);
  unsigned u[8];
  float far = 0.0f;                        // largest distance from the integer next to it
  #pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 f = __bfloat1622float2(h[j]), up = fma2(f, inv2, magic), d = fma2(f, inv2, fma2(up, minus, magic));
    far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
    u[2 * j] = __float_as_uint(up.x);
    u[2 * j + 1] = __float_as_uint(up.y);
  }
  if (far > 0.5f - 6.2e-5f) {              // one in a thousand
    #pragma unroll
    for (int j = 0; j < 4; j++) {
      const float2 f = __bfloat1622float2(h[j]);
      u[2 * j] = quantize_slowly(f.x, s);
      u[2 * j + 1] = quantize_slowly(f.y, s);
    }
  }
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

}  // namespace quant
}  // namespace rbv
