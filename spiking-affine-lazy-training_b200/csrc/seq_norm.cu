// Root-mean-square norm with the residual's addition, its 8-bit form and its gradient.
//
// One pass over the data: a row is held in registers between the sum of squares and the scaling.
// What bounds both directions is memory: 2 to 4 arrays of the row's size against about ten
// operations an element.
#include <cuda_fp8.h>

#include <algorithm>

#include "seq_q8.cuh"
#include "sequence.cuh"

namespace salt {

namespace {

constexpr int kWarpRowMost = 1024;    // widest row that one warp takes (4 packs a lane)
constexpr int kRowThreadsMost = 512;  // at 4 packs a thread: rows of up to 16384 elements

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

template <typename T, int V>
__device__ __forceinline__ void store_pairs(T* p, const f32x2 (&r)[(V + 1) / 2], int n, bool vec) {
  float f[V + 1];
#pragma unroll
  for (int k = 0; k < (V + 1) / 2; ++k) {
    const float2 v = halves(r[k]);
    f[2 * k] = v.x, f[2 * k + 1] = v.y;
  }
  store_pack<T, V>(p, f, n, vec);
}
template <typename T, int V>
__device__ __forceinline__ void load_weight_pairs(f32x2 (&w)[(V + 1) / 2], const void* from,
                                                  int64_t at, int n, bool is_f32, bool vec) {
  float f[V];
  load_weights<T, V>(f, from, at, n, is_f32, vec);
  if constexpr (V == 1) {
    w[0] = pair(f[0], 0.f);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) w[k] = pair(f[2 * k], f[2 * k + 1]);
  }
}

// r = x + residual; out = r * rsqrt(mean(r^2) + eps) * weight.
//
// A thread holds PER packs of V neighbouring elements, pack i of the row's thread t at element
// V * (i * threads + t); V is the widest that all rows' starts allow.  Rows of up to 1024 elements
// take a warp each, 4 to a block; wider ones a block.  Blocks go on to further rows, with the next
// row's loads on their way while this one is summed and stored (16384 rows of 5120 in bf16 with a
// residual to 8 bits by groups of 128: 143 us against 150 us with a block for each row, 167 us with
// branches around the loads, 123 us without divisions by the group's size, 128 us with exact
// quotients).  Those 128 us are 4.6 TB/s or 71 % of the measured copy rate; an instruction issues in
// two of three cycles, so what is left is shared by instructions and the two barriers of a row's sum.
// Few rows cost the call alone: 10 us from the host.
// The registers are held down for more threads than the grid starts (1024 an SM), and the compiler
// spills: 36 to 536 bytes a thread for packs of 8, 36 to 604 for packs of 4 and 532 to 824 for packs of
// 1.  Those take 144 us for 8192 rows of 2501 in bf16, where rows of 4096 take 52 us.
template <typename T, typename R, int V, int PER, bool VEC>
__global__ void __launch_bounds__(kRowThreadsMost, V * PER <= 8 ? 3 : V * PER <= 16 ? 2 : 1)
rms_norm_kernel(salt_rms_norm_args a, int threads, bool w_f32, int group_bits, int groups) {
  constexpr bool vec = VEC;
  __shared__ float red[32];
  const int t = threads == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int each = threads == 32 ? blockDim.x >> 5 : 1;  // rows of the block at a time
  const int64_t step = (int64_t)gridDim.x * each;
  int64_t row = (int64_t)blockIdx.x * each + (threads == 32 ? threadIdx.x >> 5 : 0);
  const R* res = static_cast<const R*>(a.residual);
  Pack<T, V> px[PER];
  Pack<R, V> pr[PER];
  auto load = [&](int64_t at_row) {
    const T* x = static_cast<const T*>(a.x) + at_row * a.x_stride;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = V * (i * threads + t), n = a.dim - at;
      px[i] = VEC ? load_whole<T, V>(x, at, a.dim) : load_pack<T, V>(x + at, n, false);
      if (res) {
        const R* from = res + at_row * a.residual_stride;
        pr[i] = VEC ? load_whole<R, V>(from, at, a.dim) : load_pack<R, V>(from + at, n, false);
      }
    }
  };
  constexpr int H = (V + 1) / 2;  // pairs of a pack; the one element of V = 1 has a zero beside it
  if (row < a.rows) load(row);
  f32x2 w[PER][H];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = V * (i * threads + t);
    load_weight_pairs<T, V>(w[i], a.weight, at, a.dim - at, w_f32, vec);
  }
  for (; row < a.rows; row += step) {  // the same for a whole warp, or a whole block
    f32x2 r[PER][H], sq = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
      for (int k = 0; k < H; ++k) {
        r[i][k] = pair_in(px[i], k);
        if (res) r[i][k] = add2(r[i][k], pair_in(pr[i], k));
        if (V * (i * threads + t) >= a.dim) r[i][k] = 0;
        sq = fma2(r[i][k], r[i][k], sq);
      }
    }
    if (row + step < a.rows) load(row + step);  // on its way while this row is summed and stored
    const float2 both_sq = halves(sq);
    const float rstd =
        rsqrtf(row_sum(both_sq.x + both_sq.y, threads, red) / (float)a.dim + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rstd;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = V * (i * threads + t), n = a.dim - at;
      if (a.residual_out)
        store_pairs<R, V>(static_cast<R*>(a.residual_out) + row * a.residual_out_stride + at, r[i],
                          n, vec);
#pragma unroll
      for (int k = 0; k < H; ++k) r[i][k] = mul2(mul2(r[i][k], both(rstd)), w[i][k]);
      if (!a.scale) {
        store_pairs<T, V>(static_cast<T*>(a.out) + row * a.out_stride + at, r[i], n, vec);
        continue;
      }
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const float2 v = halves(r[i][k]);
        m = fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
      most = fmaxf(most, m);
      if (a.group) {
        // group / V neighbouring lanes hold a group (at V = 8, which 8 bits always take: 4 to 32,
        // never across warps)
        for (int o = a.group / V / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const E4m3Scale by(m);
        // a division by the group's size would cost as much as the rest of the pack
        if (n > 0 && (at & (a.group - 1)) == 0)
          a.scale[row * groups + (at >> group_bits)] = by.scale;
        by.divide(r[i]);
      }
    }
    if (!a.scale) continue;
    if (!a.group) {
      const E4m3Scale by(row_max(most, threads, red));
      if (t == 0) a.scale[row] = by.scale;
#pragma unroll
      for (int i = 0; i < PER; ++i) by.divide(r[i]);
    }
    uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.out_stride;
    const bool wide = V == 8 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = V * (i * threads + t), n = a.dim - at;
      uint16_t q[H];
#pragma unroll
      for (int k = 0; k < H; ++k)
        q[k] = __nv_cvt_float2_to_fp8x2(halves(r[i][k]), __NV_SATFINITE, __NV_E4M3);
      if (V == 8 && wide && n >= V) {
        *reinterpret_cast<uint2*>(out + at) =
            make_uint2(q[0] | (uint32_t)q[1 % H] << 16, q[2 % H] | (uint32_t)q[3 % H] << 16);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k < n) out[at + k] = (uint8_t)(q[k / 2] >> (k % 2 * 8));
      }
    }
  }
}

// dx = rstd (w dy - h mean(w dy h)) + dresidual with h = x rstd; dweight = sum over rows of dy h.
//
// Blocks walk over rows with a fixed set of columns for each thread, so that the
// weight's gradient stays in registers; each block (each warp, for narrow rows) writes one partial
// row of it, which sum_parts adds up in order.  All three arrays' loads of a row go out before the
// barriers of its sum: 59 us against 77 us with branches between them, for 8190 rows of 2500 (packs
// of 4) in bf16 with a 32-bit residual, sum_parts' 7 us included: 4.9 TB/s, 75 % of the copy rate.
// Rows over 8192 wide spill 416 to 1956 bytes a thread (8192 rows of 12288 in bf16: 254 us, those of
// 4096 80 us).
template <typename T, typename R, int V, int PER, bool VEC>
__global__ void __launch_bounds__(kRowThreadsMost)
rms_norm_backward_kernel(salt_rms_norm_backward_args a, int threads, bool w_f32, float* parts) {
  constexpr bool vec = VEC;
  __shared__ float red[32];
  const bool by_warp = threads == 32;
  const int t = by_warp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t worker = by_warp ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)
                                 : (int64_t)blockIdx.x;
  const int64_t workers = by_warp ? (int64_t)gridDim.x * (blockDim.x >> 5) : (int64_t)gridDim.x;
  float w[PER][V], dw[PER][V];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = V * (i * threads + t);
    load_weights<T, V>(w[i], a.weight, at, a.dim - at, w_f32, vec);
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = 0.f;
  }
  for (int64_t row = worker; row < a.rows; row += workers) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const R* x = static_cast<const R*>(a.x) + row * a.x_stride;
    const R* dres = static_cast<const R*>(a.dresidual);
    const float rstd = a.rstd[row];
    // all of a row's loads before the barriers of its sum
    Pack<T, V> pdy[PER];
    Pack<R, V> px[PER], pr[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = V * (i * threads + t), n = a.dim - at;
      pdy[i] = VEC ? load_whole<T, V>(dy, at, a.dim) : load_pack<T, V>(dy + at, n, false);
      px[i] = VEC ? load_whole<R, V>(x, at, a.dim) : load_pack<R, V>(x + at, n, false);
      if (dres) {
        const R* from = dres + row * a.dresidual_stride;
        pr[i] = VEC ? load_whole<R, V>(from, at, a.dim) : load_pack<R, V>(from + at, n, false);
      }
    }
    float h[PER][V], g[PER][V];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const bool in = V * (i * threads + t) < a.dim;
        h[i][k] = in ? to_f32(px[i].v[k]) * rstd : 0.f;
        const float d = in ? to_f32(pdy[i].v[k]) : 0.f;
        dw[i][k] = fmaf(d, h[i][k], dw[i][k]);
        g[i][k] = d * w[i][k];
        dot = fmaf(g[i][k], h[i][k], dot);
      }
    }
    const float mean = row_sum(dot, threads, red) / (float)a.dim;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = V * (i * threads + t), n = a.dim - at;
      float dx[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dx[k] = rstd * fmaf(-h[i][k], mean, g[i][k]);
        if (dres) dx[k] += to_f32(pr[i].v[k]);
      }
      store_pack<R, V>(static_cast<R*>(a.dx) + row * a.dx_stride + at, dx, n, vec);
    }
  }
  if (!parts) return;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = V * (i * threads + t);
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (at + k < a.dim) parts[worker * a.dim + at + k] = dw[i][k];
  }
}

// A block takes 32 elements; thread row y adds the parts y, y + rows, ... and the first row adds
// the rows' sums in order.
template <int ROWS>
__global__ void __launch_bounds__(32 * ROWS)
sum_parts_kernel(const float* __restrict__ in, int64_t parts, int64_t n, PartSums to) {
  __shared__ float red[ROWS][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int64_t p = threadIdx.y; p < parts; p += ROWS) s += in[p * n + i];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || i >= n) return;
#pragma unroll
  for (int r = 1; r < ROWS; ++r) s += red[r][threadIdx.x];
  if (i < to.n0) {
    const int64_t dim = to.width ? to.n0 / to.width : 1;
    if (to.out0) to.out0[to.width ? i % dim * to.width + i / dim : i] = s;
  } else if (i < to.n0 + to.n1) {
    if (to.out1) to.out1[i - to.n0] = s;
  } else if (to.out2) {
    to.out2[i - to.n0 - to.n1] = s;
  }
}

struct NormPlan {
  int v, threads, per, block;
  int64_t blocks;
};

NormPlan norm_plan(int32_t rows, int32_t dim, int v) {
  NormPlan p;
  p.v = v;
  const int packs = (dim + v - 1) / v, most = 32 / v;  // a thread holds up to 32 elements
  if (dim <= kWarpRowMost) {
    p.threads = 32;
    p.block = 128;
    p.blocks = ((int64_t)rows + 3) / 4;
    p.per = (packs + 31) / 32;
  } else {
    p.per = std::max((packs + kRowThreadsMost - 1) / kRowThreadsMost, 8 / v);
  }
  int per = std::max(1, most / 4);  // 8, 16 or 32 elements
  while (per < p.per) per *= 2;
  p.per = per;
  if (dim > kWarpRowMost) {
    p.threads = p.block = ((packs + per - 1) / per + 31) / 32 * 32;
    p.blocks = rows;
  }
  return p;
}

// Workers (blocks, or warps of narrow rows) of the gradient: one partial weight gradient each.
void norm_back_grid(const NormPlan& p, int32_t rows, int* blocks, int* workers) {
  const int each = p.threads == 32 ? p.block / 32 : 1;
  const int64_t at_once = 148 * std::max(1, 1024 / p.block);
  *blocks = (int)std::max<int64_t>(1, std::min(at_once, ((int64_t)rows + each - 1) / each));
  *workers = *blocks * each;
}

}  // namespace

cudaError_t sum_parts_launch(const float* in, int64_t parts, const PartSums& to, cudaStream_t st) {
  const int64_t n = to.n0 + to.n1 + to.n2;
  if (n == 0) return cudaSuccess;
  const unsigned blocks = (unsigned)((n + 31) / 32);
  if (parts <= 16)
    sum_parts_kernel<4><<<blocks, dim3(32, 4), 0, st>>>(in, parts, n, to);
  else
    sum_parts_kernel<32><<<blocks, dim3(32, 32), 0, st>>>(in, parts, n, to);
  return cudaGetLastError();
}

// Elements per pack by V, packs of a thread by PER.  Packs of one element are always whole; packs
// of 8 may be cut in the 8-bit form alone, whose groups are counted in them.
#define SALT_NORM_SHAPE(p, kernel, T, R, ...)                      \
  do {                                                             \
    if ((p).v == 8) {                                              \
      if ((p).per == 1)                                            \
        kernel<T, R, 8, 1, true> __VA_ARGS__;                      \
      else if ((p).per == 2)                                       \
        kernel<T, R, 8, 2, true> __VA_ARGS__;                      \
      else                                                         \
        kernel<T, R, 8, 4, true> __VA_ARGS__;                      \
    } else if ((p).v == 4) {                                       \
      if ((p).per == 2)                                            \
        kernel<T, R, 4, 2, true> __VA_ARGS__;                      \
      else if ((p).per == 4)                                       \
        kernel<T, R, 4, 4, true> __VA_ARGS__;                      \
      else                                                         \
        kernel<T, R, 4, 8, true> __VA_ARGS__;                      \
    } else {                                                       \
      if ((p).per == 8)                                            \
        kernel<T, R, 1, 8, true> __VA_ARGS__;                      \
      else if ((p).per == 16)                                      \
        kernel<T, R, 1, 16, true> __VA_ARGS__;                     \
      else                                                         \
        kernel<T, R, 1, 32, true> __VA_ARGS__;                     \
    }                                                              \
  } while (0)
#define SALT_NORM_CUT(p, kernel, T, R, ...)                        \
  do {                                                             \
    if ((p).per == 1)                                              \
      kernel<T, R, 8, 1, false> __VA_ARGS__;                       \
    else if ((p).per == 2)                                         \
      kernel<T, R, 8, 2, false> __VA_ARGS__;                       \
    else                                                           \
      kernel<T, R, 8, 4, false> __VA_ARGS__;                       \
  } while (0)

cudaError_t rms_norm_launch(const salt_rms_norm_args& a, cudaStream_t st, int* launches) {
  if (a.rows == 0) return cudaSuccess;
  const size_t ts = type_size(a.type), rs = type_size(a.residual_type);
  const bool w_f32 = a.weight_type == SALT_F32;
  auto fits = [&](int v) {
    return a.dim % v == 0 && pack_rows(a.x, v, ts, a.x_stride) &&
           pack_rows(a.residual, v, rs, a.residual_stride) &&
           pack_rows(a.residual_out, v, rs, a.residual_out_stride) &&
           pack_rows(a.weight, v, w_f32 ? 4 : ts, 0) &&
           (a.scale || pack_rows(a.out, v, ts, a.out_stride));
  };
  const bool cut = a.scale && !fits(8);
  int bits = 0;
  while (a.group > (1 << bits)) ++bits;
  const int groups = a.group ? (a.dim + a.group - 1) / a.group : 1;
  const NormPlan p = norm_plan(a.rows, a.dim, cut || fits(8) ? 8 : fits(4) ? 4 : 1);
  // as many blocks as the GPU holds at once: each goes on to further rows
  const int64_t at_once = 148 * std::max(1, 1024 / p.block);
  const unsigned blocks = (unsigned)std::min<int64_t>(p.blocks, at_once);
  SALT_WITH_TYPE(a.type, T, {
    using Wide = float;
    if (a.residual_type == SALT_F32) {
      if (cut)
        SALT_NORM_CUT(p, rms_norm_kernel, T, Wide,
                      <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, bits, groups));
      else
        SALT_NORM_SHAPE(p, rms_norm_kernel, T, Wide,
                        <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, bits, groups));
    } else {
      if (cut)
        SALT_NORM_CUT(p, rms_norm_kernel, T, T,
                      <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, bits, groups));
      else
        SALT_NORM_SHAPE(p, rms_norm_kernel, T, T,
                        <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, bits, groups));
    }
  });
  ++*launches;
  return cudaGetLastError();
}

namespace {
NormPlan norm_back_plan(const salt_rms_norm_backward_args& a) {
  const size_t ts = type_size(a.type), rs = type_size(a.residual_type);
  auto fits = [&](int v) {
    return a.dim % v == 0 && pack_rows(a.dy, v, ts, a.dy_stride) &&
           pack_rows(a.x, v, rs, a.x_stride) &&
           pack_rows(a.dresidual, v, rs, a.dresidual_stride) &&
           pack_rows(a.dx, v, rs, a.dx_stride) &&
           pack_rows(a.weight, v, a.weight_type == SALT_F32 ? 4 : ts, 0);
  };
  return norm_plan(a.rows, a.dim, fits(8) ? 8 : fits(4) ? 4 : 1);
}
}  // namespace

size_t rms_norm_backward_bytes(const salt_rms_norm_backward_args& a) {
  if (!a.dweight) return 0;
  int blocks, workers;
  norm_back_grid(norm_back_plan(a), a.rows, &blocks, &workers);
  return (size_t)workers * a.dim * sizeof(float);
}

cudaError_t rms_norm_backward_launch(const salt_rms_norm_backward_args& a, void* ws,
                                     cudaStream_t st, int* launches) {
  const NormPlan p = norm_back_plan(a);
  int blocks, workers;
  norm_back_grid(p, a.rows, &blocks, &workers);
  const bool w_f32 = a.weight_type == SALT_F32;
  float* parts = a.dweight ? static_cast<float*>(ws) : nullptr;
  SALT_WITH_TYPE(a.type, T, {
    if (a.residual_type == SALT_F32)
      SALT_NORM_SHAPE(p, rms_norm_backward_kernel, T, float,
                      <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, parts));
    else
      SALT_NORM_SHAPE(p, rms_norm_backward_kernel, T, T,
                      <<<blocks, p.block, 0, st>>>(a, p.threads, w_f32, parts));
  });
  ++*launches;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !parts) return e;
  ++*launches;
  return sum_parts_launch(parts, workers, PartSums{a.dim, 0, 0, a.dweight, nullptr, nullptr, 0},
                          st);
}

}  // namespace salt
