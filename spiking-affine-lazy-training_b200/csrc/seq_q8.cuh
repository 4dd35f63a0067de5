// Scales of 8-bit values (e4m3), shared by the norm's 8-bit form and the quantisation.
#pragma once
#include <cuda_fp8.h>

#include "sequence.cuh"

namespace salt {

constexpr float kE4m3Max = 448.f;

// The scale of a group whose largest magnitude is m: the float32 quotient m / 448 (at least float32's
// smallest value; 1 for a group of zeros), and what divides the group's values by it.  fmaxf leaves NaNs out of m: they become e4m3's
// own, beside the other elements' scale.
//
// A product with one rounded inverse may bring a value near the middle of two 8-bit ones to the other
// side than the quotient.  So the scale is the product m (1/448) with its remainder added (P.
// Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990): m /
// 448 rounded, for every m.  The inverse of the scale has two parts, y and y (1 - scale y); the sum of
// a value's products with them is rounded once, and off by less than 2^-44 of itself before that.
// Against the one product: 16384 rows of 5120 in bf16 with a residual, by groups of 128, take 128
// us instead of 123.
// Far from 1 the parts or products would underflow: `lift` moves both operands by a power of two.  An
// infinity as the largest value leaves 0 for all finite ones.
struct E4m3Scale {
  float scale, lift;
  f32x2 high, low;
  // the four numbers of one, to be kept in shared memory
  __device__ __forceinline__ float4 packed() const {
    return make_float4(scale, lift, halves(high).x, halves(low).x);
  }
  __device__ __forceinline__ explicit E4m3Scale(const float4& p)
      : scale(p.x), lift(p.y), high(both(p.z)), low(both(p.w)) {}
  __device__ __forceinline__ explicit E4m3Scale(float m) : lift(1.f) {
    float divisor;
    if (m >= 0x1p-60f && m < 0x1p60f) {
      constexpr float by = 1.f / kE4m3Max;
      const float q = m * by;
      divisor = scale = fmaf(fmaf(-q, kE4m3Max, m), by, q);
    } else {
      scale = m == 0.f ? 1.f : fmaxf(m / kE4m3Max, 0x1p-149f);  // a scale of 0 would divide by it
      lift = m < 1.f ? 0x1p64f : 0x1p-64f;
      divisor = scale * lift;
    }
    const float y = rcp_fast(divisor);
    high = both(y);
    low = both(divisor < INFINITY ? fmaf(-divisor, y, 1.f) * y : 0.f);
  }
  // the values' quotients by the scale
  template <int H>
  __device__ __forceinline__ void divide(f32x2 (&v)[H]) const {
    if (lift != 1.f) {
#pragma unroll
      for (int k = 0; k < H; ++k) v[k] = mul2(v[k], both(lift));
    }
#pragma unroll
    for (int k = 0; k < H; ++k) v[k] = fma2(v[k], high, mul2(v[k], low));
  }
};

}  // namespace salt
