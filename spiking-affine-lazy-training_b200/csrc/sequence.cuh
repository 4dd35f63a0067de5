// Shared device helpers and launch declarations of the sequence operators (root-mean-square norm,
// short causal convolution, selective state space scan).
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/salt_b200.h"

namespace salt {

constexpr int kVec = 8;  // elements a thread moves at once: 16 bytes of a 16-bit type

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N neighbouring elements as they lie in memory; loads and stores are 16 (or 8, 4) bytes wide.
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// p[0 .. n) of N elements, zero behind; n outside [0, N] is clipped.  Without `vec` (the pointer
// may be unaligned) or with n < N every element is loaded by itself.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p, int n, bool vec) {
  Pack<T, N> r;
  if (vec && n >= N) {
    r = *reinterpret_cast<const Pack<T, N>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
  return r;
}
// The same where packs are whole (the pointer is aligned, and `at` or the end lies on a pack): p[at
// .. at + N), or p[0 .. N) if at is not under `end`, for the caller to leave out where it uses
// them.  A branch around a load, or a choice behind it, would make the thread wait for the load
// there and then, and not where its values are used.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_whole(const T* p, int64_t at, int64_t end) {
  return *reinterpret_cast<const Pack<T, N>*>(p + (at < end ? at : 0));
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float* f, int n, bool vec) {
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(f[i]);
  if (vec && n >= N) {
    *reinterpret_cast<Pack<T, N>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

// N neighbouring weights that hold T or float32; n as in load_pack.
template <typename T, int N>
__device__ __forceinline__ void load_weights(float (&f)[N], const void* w, int64_t at, int n,
                                             bool is_f32, bool vec) {
  if (is_f32) {
    const Pack<float, N> p = load_pack<float, N>(static_cast<const float*>(w) + at, n, vec);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = p.v[i];
  } else {
    const Pack<T, N> p = load_pack<T, N>(static_cast<const T*>(w) + at, n, vec);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(p.v[i]);
  }
}

// A weight that holds T or float32.
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int64_t i, bool is_f32) {
  return is_f32 ? static_cast<const float*>(w)[i] : to_f32(static_cast<const T*>(w)[i]);
}

constexpr float kLog2e = 1.4426950408889634f;

// 2^x to about 2 ulp in one instruction; results below the normal range become 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }

// 1 / (1 + e^-x).  e^-x overflows to infinity for x < -88; the quotient is then 0.
__device__ __forceinline__ float sigmoid(float x) {
  return __fdividef(1.f, 1.f + exp_fast(-x));
}


__device__ __forceinline__ int32_t row_tokens(const int32_t* n_real, int b, int32_t len) {
  if (!n_real) return len;
  const int32_t n = n_real[b];
  return n < 0 ? 0 : (n < len ? n : len);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two float32 side by side: one instruction does both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 exp2_fast2(f32x2 v) {
  const float2 h = halves(v);
  return pair(exp2_fast(h.x), exp2_fast(h.y));
}

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log(1 + e^x) = max(x, 0) + log1p(u) with u = e^-|x| in (0, 1].  log1p keeps its relative
// precision at small u (a step of 1e-3 is an ordinary value, and 1 + u would drop 4 of its
// digits) through log1p(u) = 2 atanh(q), q = u / (2 + u) <= 1/3: 2 atanh(q) / q is interpolated at
// the Chebyshev nodes of q^2 in [0, 1/9] by a polynomial of degree 4, within 8e-9 of itself.  A NaN
// stays one: fmaxf drops it, u keeps it.
__device__ __forceinline__ f32x2 softplus2(f32x2 x) {
  const float2 v = halves(x);
  const f32x2 u = pair(exp2_fast(fabsf(v.x) * -kLog2e), exp2_fast(fabsf(v.y) * -kLog2e));
  const float2 w = halves(add2(u, pair(2.f, 2.f)));
  const f32x2 q = mul2(u, pair(rcp_fast(w.x), rcp_fast(w.y))), s = mul2(q, q);
  f32x2 p = pair(0.2815778f, 0.2815778f);
  p = fma2(p, s, pair(0.27965158f, 0.27965158f));
  p = fma2(p, s, pair(0.40024596f, 0.40024596f));
  p = fma2(p, s, pair(0.6666632f, 0.6666632f));
  p = fma2(p, s, pair(2.f, 2.f));
  return fma2(p, q, pair(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
}
__device__ __forceinline__ float softplus_f(float x) { return halves(softplus2(pair(x, x))).x; }

// 1 / (1 + e^-x) of both.
__device__ __forceinline__ f32x2 sigmoid2(f32x2 x) {
  const f32x2 e = exp2_fast2(mul2(x, pair(-kLog2e, -kLog2e)));
  const float2 d = halves(add2(e, pair(1.f, 1.f)));
  return pair(rcp_fast(d.x), rcp_fast(d.y));
}

// Elements k and k + 1 of a pack.
template <typename T, int N>
__device__ __forceinline__ f32x2 pair_of(const Pack<T, N>& p, int k) {
  return pair(to_f32(p.v[k]), to_f32(p.v[k + 1]));
}
template <int N>
__device__ __forceinline__ f32x2 pair_of(const Pack<__nv_bfloat16, N>& p, int k) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&p.v[k]);  // k is even
  return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// Elements 2 k and 2 k + 1 of a pack; a pack of one has a zero behind it.
template <typename T, int V>
__device__ __forceinline__ f32x2 pair_in(const Pack<T, V>& p, int k) {
  if constexpr (V == 1)
    return pair(to_f32(p.v[0]), 0.f);
  else
    return pair_of(p, 2 * k);
}
__device__ __forceinline__ f32x2 both(float v) { return pair(v, v); }
// d/dx of x * sigmoid(x), of both.
__device__ __forceinline__ f32x2 silu_slope2(f32x2 x, f32x2 p) {
  return mul2(p, fma2(x, fma2(p, both(-1.f), both(1.f)), both(1.f)));
}

// Launches (argument checks are the caller's; each returns the launch's status).
cudaError_t rms_norm_launch(const salt_rms_norm_args& a, cudaStream_t st, int* launches);
size_t rms_norm_backward_bytes(const salt_rms_norm_backward_args& a);
cudaError_t rms_norm_backward_launch(const salt_rms_norm_backward_args& a, void* ws,
                                     cudaStream_t st, int* launches);
cudaError_t causal_conv_launch(const salt_causal_conv_args& a, cudaStream_t st, int* launches);
cudaError_t causal_conv_step_launch(const salt_causal_conv_step_args& a, cudaStream_t st,
                                    int* launches);
size_t causal_conv_backward_bytes(const salt_causal_conv_backward_args& a);
cudaError_t causal_conv_backward_launch(const salt_causal_conv_backward_args& a, void* ws,
                                        cudaStream_t st, int* launches);
size_t selective_scan_bytes(const salt_selective_scan_args& a);
cudaError_t selective_scan_launch(const salt_selective_scan_args& a, void* ws, cudaStream_t st,
                                  int* launches);
cudaError_t selective_scan_step_launch(const salt_selective_scan_step_args& a, cudaStream_t st,
                                       int* launches);
size_t selective_scan_backward_bytes(const salt_selective_scan_backward_args& a);
cudaError_t selective_scan_backward_launch(const salt_selective_scan_backward_args& a, void* ws,
                                           cudaStream_t st, int* launches);

// The second stage of every weight gradient: sums `parts` partial arrays of float32, part p at
// in + p * n, in an order that their number alone decides.  A part holds up to three gradients of
// n0, n1 and n2 elements one after the other (n is their sum; an out that is NULL is left out).
// With width set, the first is (width, n0 / width) there and comes out transposed.
struct PartSums {
  int64_t n0, n1, n2;
  float *out0, *out1, *out2;
  int width;
};
cudaError_t sum_parts_launch(const float* in, int64_t parts, const PartSums& to, cudaStream_t st);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Whether rows at p with these strides (in elements) start on boundaries of `bytes`.
inline bool packed_rows(const void* p, int64_t bytes, size_t size, int64_t s0, int64_t s1) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (int64_t)(s0 * size) % bytes == 0 &&
         (int64_t)(s1 * size) % bytes == 0;
}
inline size_t type_size(int32_t type) { return type == SALT_F32 ? 4 : 2; }
// Whether rows at p can be moved in packs of `n` elements.
inline bool pack_rows(const void* p, int n, size_t size, int64_t s0, int64_t s1 = 0) {
  return !p || packed_rows(p, std::min<int64_t>(16, n * size), size, s0, s1);
}

// Calls F<T>(...) for the C type that `type` names.
#define SALT_WITH_TYPE(type, T, ...)          \
  do {                                        \
    if ((type) == SALT_F32) {                 \
      using T = float;                        \
      __VA_ARGS__;                            \
    } else if ((type) == SALT_F16) {          \
      using T = __half;                       \
      __VA_ARGS__;                            \
    } else {                                  \
      using T = __nv_bfloat16;                \
      __VA_ARGS__;                            \
    }                                         \
  } while (0)

}  // namespace salt
