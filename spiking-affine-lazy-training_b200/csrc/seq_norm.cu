// Root-mean-square norm with the residual's addition, its 8-bit form and its gradient.
//
// One pass over the data: a row is held in registers between the sum of squares and the scaling.
// What bounds both directions is memory: 2 to 4 arrays of the row's size against about ten
// operations an element.
#include <cuda_fp8.h>

#include <algorithm>

#include "sequence.cuh"

namespace salt {

namespace {

constexpr int kWarpRowMost = 1024;  // widest row that one warp takes (4 packs a lane)
constexpr int kRowThreadsMost = 512;  // at 4 packs a thread: rows of up to 16384 elements
constexpr float kE4m3Max = 448.f;

// Sums v over the threads of one row: a warp (threads == 32), or the whole block.  `red` has a
// place per warp and is free again when this returns and the next call has passed its barrier.
__device__ __forceinline__ float row_sum(float v, int threads, float* red) {
  v = warp_sum(v);
  if (threads == 32) return v;
  const int warps = threads >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ float row_max(float v, int threads, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threads == 32) return v;
  const int warps = threads >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s = fmaxf(s, red[i]);
  return s;
}

// A thread holds PER packs of 8 neighbouring elements, pack i of the row's thread t at element
// 8 * (i * threads + t).  Rows of up to 1024 elements take a warp each, 4 to a block; wider ones a
// block.
template <typename T, typename R, int PER>
__global__ void __launch_bounds__(kRowThreadsMost)
rms_norm_kernel(salt_rms_norm_args a, int threads, bool vec, bool w_f32) {
  __shared__ float red[32];
  const int t = threads == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = threads == 32 ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)
                                    : (int64_t)blockIdx.x;
  if (row >= a.rows) return;  // a whole warp, or no thread of the block
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* res = static_cast<const R*>(a.residual);
  float r[PER][kVec];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = kVec * (i * threads + t), n = a.dim - at;
    const Pack<T, kVec> px = load_pack<T, kVec>(x + at, n, vec);
#pragma unroll
    for (int k = 0; k < kVec; ++k) r[i][k] = to_f32(px.v[k]);
    if (res) {
      const Pack<R, kVec> pr = load_pack<R, kVec>(res + row * a.residual_stride + at, n, vec);
#pragma unroll
      for (int k = 0; k < kVec; ++k) r[i][k] += to_f32(pr.v[k]);
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k) sq = fmaf(r[i][k], r[i][k], sq);
  }
  const float rstd = rsqrtf(row_sum(sq, threads, red) / (float)a.dim + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = rstd;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = kVec * (i * threads + t), n = a.dim - at;
    if (a.residual_out)
      store_pack<R, kVec>(static_cast<R*>(a.residual_out) + row * a.residual_out_stride + at, r[i],
                          n, vec);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const float w = k < n ? weight_at<T>(a.weight, at + k, w_f32) : 0.f;
      r[i][k] *= rstd * w;
      most = fmaxf(most, fabsf(r[i][k]));
    }
    if (!a.scale) {
      store_pack<T, kVec>(static_cast<T*>(a.out) + row * a.out_stride + at, r[i], n, vec);
    } else if (a.group) {
      // group / 8 neighbouring lanes hold a group (4 to 32 of them, so never across warps)
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < kVec; ++k) m = fmaxf(m, fabsf(r[i][k]));
      for (int o = a.group / kVec / 2; o; o >>= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = m > 0.f ? m / kE4m3Max : 1.f;
      if (n > 0 && at % a.group == 0)
        a.scale[row * ((a.dim + a.group - 1) / a.group) + at / a.group] = scale;
#pragma unroll
      for (int k = 0; k < kVec; ++k) r[i][k] /= scale;
    }
  }
  if (!a.scale) return;
  if (!a.group) {
    const float m = row_max(most, threads, red), scale = m > 0.f ? m / kE4m3Max : 1.f;
    if (t == 0) a.scale[row] = scale;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int k = 0; k < kVec; ++k) r[i][k] /= scale;
  }
  uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.out_stride;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 7) == 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = kVec * (i * threads + t), n = a.dim - at;
    alignas(8) uint8_t q[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      q[k] = __nv_cvt_float_to_fp8(r[i][k], __NV_SATFINITE, __NV_E4M3);
    if (wide && n >= kVec)
      *reinterpret_cast<uint2*>(out + at) = *reinterpret_cast<const uint2*>(q);
    else
      for (int k = 0; k < kVec; ++k)
        if (k < n) out[at + k] = q[k];
  }
}

// The gradient.  Blocks walk over rows with a fixed set of columns for each thread, so that the
// weight's gradient stays in registers; each block (each warp, for narrow rows) writes one partial
// row of it, which sum_parts adds up in order.
template <typename T, typename R, int PER>
__global__ void __launch_bounds__(kRowThreadsMost)
rms_norm_backward_kernel(salt_rms_norm_backward_args a, int threads, bool vec, bool w_f32,
                         float* parts) {
  __shared__ float red[32];
  const bool by_warp = threads == 32;
  const int t = by_warp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t worker = by_warp ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)
                                 : (int64_t)blockIdx.x;
  const int64_t workers = by_warp ? (int64_t)gridDim.x * (blockDim.x >> 5) : (int64_t)gridDim.x;
  float w[PER][kVec], dw[PER][kVec];
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const int at = kVec * (i * threads + t) + k;
      w[i][k] = at < a.dim ? weight_at<T>(a.weight, at, w_f32) : 0.f;
      dw[i][k] = 0.f;
    }
  for (int64_t row = worker; row < a.rows; row += workers) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const R* x = static_cast<const R*>(a.x) + row * a.x_stride;
    const R* dres = static_cast<const R*>(a.dresidual);
    const float rstd = a.rstd[row];
    float h[PER][kVec], g[PER][kVec];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = kVec * (i * threads + t), n = a.dim - at;
      const Pack<T, kVec> pdy = load_pack<T, kVec>(dy + at, n, vec);
      const Pack<R, kVec> px = load_pack<R, kVec>(x + at, n, vec);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        h[i][k] = to_f32(px.v[k]) * rstd;
        const float d = to_f32(pdy.v[k]);
        dw[i][k] = fmaf(d, h[i][k], dw[i][k]);
        g[i][k] = d * w[i][k];
        dot = fmaf(g[i][k], h[i][k], dot);
      }
    }
    const float mean = row_sum(dot, threads, red) / (float)a.dim;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = kVec * (i * threads + t), n = a.dim - at;
      Pack<R, kVec> pr;
      if (dres) pr = load_pack<R, kVec>(dres + row * a.dresidual_stride + at, n, vec);
      float dx[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        dx[k] = rstd * fmaf(-h[i][k], mean, g[i][k]);
        if (dres) dx[k] += to_f32(pr.v[k]);
      }
      store_pack<R, kVec>(static_cast<R*>(a.dx) + row * a.dx_stride + at, dx, n, vec);
    }
  }
  if (!parts) return;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = kVec * (i * threads + t);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (at + k < a.dim) parts[worker * a.dim + at + k] = dw[i][k];
  }
}

__global__ void sum_parts_kernel(const float* __restrict__ in, int64_t parts, int64_t n,
                                 float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int64_t p = 0; p < parts; ++p) s += in[p * n + i];
  out[i] = s;
}

struct NormPlan {
  int threads, per, block;
  int64_t blocks;
};

NormPlan norm_plan(int32_t rows, int32_t dim) {
  NormPlan p;
  const int packs = (dim + kVec - 1) / kVec;
  if (dim <= kWarpRowMost) {
    p.threads = 32;
    p.block = 128;
    p.blocks = ((int64_t)rows + 3) / 4;
    p.per = packs <= 32 ? 1 : packs <= 64 ? 2 : 4;
  } else {
    p.per = packs <= 512 ? 1 : packs <= 1024 ? 2 : 4;
    p.threads = p.block = (((packs + p.per - 1) / p.per) + 31) / 32 * 32;
    p.blocks = rows;
  }
  return p;
}

constexpr int kNormBackBlocks = 148 * 4;

// Workers (blocks, or warps of narrow rows) of the gradient: one partial weight gradient each.
void norm_back_grid(const NormPlan& p, int32_t rows, int* blocks, int* workers) {
  const int each = p.threads == 32 ? p.block / 32 : 1;
  *blocks = (int)std::max<int64_t>(
      1, std::min<int64_t>(kNormBackBlocks, ((int64_t)rows + each - 1) / each));
  *workers = *blocks * each;
}

}  // namespace

cudaError_t sum_parts_launch(const float* in, int64_t parts, int64_t n, float* out,
                             cudaStream_t st) {
  if (n > 0) sum_parts_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(in, parts, n, out);
  return cudaGetLastError();
}

#define SALT_NORM_PER(kernel, per, T, R, ...)             \
  do {                                                    \
    if ((per) == 1)                                       \
      kernel<T, R, 1> __VA_ARGS__;                        \
    else if ((per) == 2)                                  \
      kernel<T, R, 2> __VA_ARGS__;                        \
    else                                                  \
      kernel<T, R, 4> __VA_ARGS__;                        \
  } while (0)

cudaError_t rms_norm_launch(const salt_rms_norm_args& a, cudaStream_t st, int* launches) {
  if (a.rows == 0) return cudaSuccess;
  const NormPlan p = norm_plan(a.rows, a.dim);
  const size_t ts = type_size(a.type), rs = type_size(a.residual_type);
  const bool vec = vec_rows(a.x, ts, a.x_stride) && vec_rows(a.residual, rs, a.residual_stride) &&
                   vec_rows(a.residual_out, rs, a.residual_out_stride) &&
                   (a.scale || vec_rows(a.out, ts, a.out_stride));
  const bool w_f32 = a.weight_type == SALT_F32;
  SALT_WITH_TYPE(a.type, T, {
    if (a.residual_type == SALT_F32)
      SALT_NORM_PER(rms_norm_kernel, p.per, T, float,
                    <<<(unsigned)p.blocks, p.block, 0, st>>>(a, p.threads, vec, w_f32));
    else
      SALT_NORM_PER(rms_norm_kernel, p.per, T, T,
                    <<<(unsigned)p.blocks, p.block, 0, st>>>(a, p.threads, vec, w_f32));
  });
  ++*launches;
  return cudaGetLastError();
}

size_t rms_norm_backward_bytes(const salt_rms_norm_backward_args& a) {
  if (!a.dweight) return 0;
  int blocks, workers;
  norm_back_grid(norm_plan(a.rows, a.dim), a.rows, &blocks, &workers);
  return (size_t)workers * a.dim * sizeof(float);
}

cudaError_t rms_norm_backward_launch(const salt_rms_norm_backward_args& a, void* ws,
                                     cudaStream_t st, int* launches) {
  const NormPlan p = norm_plan(a.rows, a.dim);
  int blocks, workers;
  norm_back_grid(p, a.rows, &blocks, &workers);
  const size_t ts = type_size(a.type), rs = type_size(a.residual_type);
  const bool vec = vec_rows(a.dy, ts, a.dy_stride) && vec_rows(a.x, rs, a.x_stride) &&
                   vec_rows(a.dresidual, rs, a.dresidual_stride) &&
                   vec_rows(a.dx, rs, a.dx_stride);
  const bool w_f32 = a.weight_type == SALT_F32;
  float* parts = a.dweight ? static_cast<float*>(ws) : nullptr;
  SALT_WITH_TYPE(a.type, T, {
    if (a.residual_type == SALT_F32)
      SALT_NORM_PER(rms_norm_backward_kernel, p.per, T, float,
                    <<<blocks, p.block, 0, st>>>(a, p.threads, vec, w_f32, parts));
    else
      SALT_NORM_PER(rms_norm_backward_kernel, p.per, T, T,
                    <<<blocks, p.block, 0, st>>>(a, p.threads, vec, w_f32, parts));
  });
  ++*launches;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !parts) return e;
  ++*launches;
  return sum_parts_launch(parts, workers, a.dim, a.dweight, st);
}

}  // namespace salt
