// Quantisation to 8 bits with a scale for every 128 values.
#include <type_traits>

#include "seq_q8.cuh"
#include "sequence.cuh"

namespace salt {
namespace {

constexpr int kGroup = SALT_Q8_GROUP;

template <int H>
__device__ __forceinline__ void to_e4m3(uint16_t (&q)[H], const f32x2 (&v)[H]) {
#pragma unroll
  for (int k = 0; k < H; ++k)
    q[k] = __nv_cvt_float2_to_fp8x2(halves(v[k]), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ void store8(uint8_t* p, const uint16_t (&q)[4], int n, bool vec) {
  if (vec && n >= 8) {
    *reinterpret_cast<uint2*>(p) =
        make_uint2(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)(q[i / 2] >> (i % 2 * 8));
  }
}

// The largest magnitudes of a pack, NaNs left out.
__device__ __forceinline__ float largest(const Pack<float, 8>& p) {
  float m = fabsf(p.v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(p.v[i]));
  return fmaxf(m, 0.f);
}
template <typename T>
__device__ __forceinline__ float largest(const Pack<T, 8>& p) {
  using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
  const T2* q = reinterpret_cast<const T2*>(&p);
  const T2 m = __hmax2(__hmax2(__habs2(q[0]), __habs2(q[1])), __hmax2(__habs2(q[2]), __habs2(q[3])));
  return fmaxf(fmaxf(to_f32(m.x), to_f32(m.y)), 0.f);
}
// The same of each column of 8 packs.
__device__ __forceinline__ void column_largest(float (&m)[8], const Pack<float, 8> (&p)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    m[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m[j] = fmaxf(m[j], fabsf(p[i].v[j]));
  }
}
template <typename T>
__device__ __forceinline__ void column_largest(float (&m)[8], const Pack<T, 8> (&p)[8]) {
  using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    T2 x = __habs2(reinterpret_cast<const T2*>(&p[0])[j]);
#pragma unroll
    for (int i = 1; i < 8; ++i) x = __hmax2(x, __habs2(reinterpret_cast<const T2*>(&p[i])[j]));
    m[2 * j] = fmaxf(to_f32(x.x), 0.f), m[2 * j + 1] = fmaxf(to_f32(x.y), 0.f);
  }
}
// A pack of a row, zeros where `live` is not: whole ones go out before anything depends on them.
template <typename T, bool VEC>
__device__ __forceinline__ Pack<T, 8> fetch(const T* row, int at, int dim, bool live) {
  if (!VEC) return load_pack<T, 8>(row + at, live ? dim - at : 0, false);
  return load_whole<T, 8>(row, live ? at : dim, dim);
}
template <typename T>
__device__ __forceinline__ void clear(Pack<T, 8>& p) {
#pragma unroll
  for (int i = 0; i < 8; ++i) p.v[i] = from_f32<T>(0.f);
}

// Rows by groups of 128: half a warp a group, 8 elements a lane, four groups' loads on their way at a
// time.  16384 rows of 5120 in bfloat16 take 55 us, 4.5 TB/s (88 us with loads that branch on the rows'
// alignment, magnitudes one by one in 32 bits); what bounds them is instruction issue next to memory.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(salt_quantize_q8_args a, unsigned groups,
                                                            bool vec_out) {
  constexpr int N = sizeof(T) == 4 ? 2 : 4;
  const int64_t n = (int64_t)a.rows * groups;
  const int lane = threadIdx.x & 15;
  const int64_t first = ((int64_t)blockIdx.x * N * 16) + (threadIdx.x >> 4);
  // (a division of 32 bits where the rows allow it: one of 64 would cost as much as the rest)
  Pack<T, 8> p[N];
  int64_t row[N];
  int at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = first + i * 16;
    row[i] = n >> 32 ? g / groups : (unsigned)g / groups;
    at[i] = (int)(g - row[i] * groups) * kGroup + lane * 8;
    p[i] = fetch<T, VEC>(static_cast<const T*>(a.x) + (g < n ? row[i] : 0) * a.x_stride, at[i], a.dim,
                         g < n);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = first + i * 16;
    const bool live = g < n && at[i] < a.dim;
    float most = VEC && !live ? 0.f : largest(p[i]);
#pragma unroll
    for (int o = 8; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const E4m3Scale by(most);
    if (g < n && lane == 0) a.scale[g] = by.scale;
    f32x2 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = pair_of(p[i], 2 * k);
    by.divide(v);
    uint16_t q[4];
    to_e4m3(q, v);
    if (live)
      store8(static_cast<uint8_t*>(a.out) + row[i] * a.out_stride + at[i], q, a.dim - at[i], vec_out);
  }
}

// Tiles of 128 x 128 for scales of whole blocks, for transposed outputs, or both.  A thread holds 8
// neighbouring rows of 8 columns; a transposed tile goes through shared memory, where 8 values of a
// column lie together and their place in the column's 16 is turned by the column's pack, so that
// a half-warp's writes spread over all banks.  Scales are made once a column (or tile) and read from
// shared memory.  4096 x 5120 in bfloat16 by blocks take 13 us (4.7 TB/s), transposed 18 us; 8192 x
// 4096 by columns 29 us (39 us with scales 24 bytes apart, whose reads met in the same banks).
template <typename T, bool VEC, bool BLOCKS, bool TRANSPOSED>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2)
quantize_tile_kernel(salt_quantize_q8_args a, int tiles_x, bool vec_out) {
  __shared__ float red[8][kGroup];
  // a column's scale at place (column % 8) * 16 + column / 8: half a warp reads neighbours
  __shared__ float4 scales[BLOCKS ? 1 : kGroup];
  __shared__ uint2 tile[TRANSPOSED ? kGroup * 16 : 1];
  const int ty = blockIdx.x / tiles_x, tx = blockIdx.x - ty * tiles_x;
  const int cp = threadIdx.x & 15, rg = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int row0 = ty * kGroup + rg * 8, col0 = tx * kGroup + cp * 8;
  const int up = (a.rows + kGroup - 1) / kGroup;
  Pack<T, 8> p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    p[i] = fetch<T, VEC>(static_cast<const T*>(a.x) + (int64_t)min(row0 + i, a.rows - 1) * a.x_stride,
                         col0, a.dim, row0 + i < a.rows);
  if (VEC && (row0 + 8 > a.rows || col0 >= a.dim)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row0 + i >= a.rows || col0 >= a.dim) clear(p[i]);
  }
  float most[8];  // of each column, or (blocks) of each row
  if (BLOCKS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) most[j] = largest(p[j]);
  } else {
    column_largest(most, p);
  }
  if (BLOCKS) {
#pragma unroll
    for (int j = 1; j < 8; ++j) most[0] = fmaxf(most[0], most[j]);
#pragma unroll
    for (int o = 16; o; o >>= 1) most[0] = fmaxf(most[0], __shfl_xor_sync(0xffffffffu, most[0], o));
    if ((threadIdx.x & 31) == 0) red[0][warp] = most[0];
    __syncthreads();
    if (threadIdx.x == 0) {
      float m = 0.f;
      for (int w = 0; w < 8; ++w) m = fmaxf(m, red[0][w]);
      const E4m3Scale by(m);
      scales[0] = by.packed();
      a.scale[TRANSPOSED ? (int64_t)tx * up + ty : (int64_t)ty * tiles_x + tx] = by.scale;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      most[j] = fmaxf(most[j], __shfl_xor_sync(0xffffffffu, most[j], 16));
      if ((threadIdx.x & 16) == 0) red[warp][cp * 8 + j] = most[j];
    }
    __syncthreads();
    if (threadIdx.x < kGroup) {
      float m = 0.f;
      for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w][threadIdx.x]);
      const E4m3Scale by(m);
      scales[(threadIdx.x & 7) * 16 + (threadIdx.x >> 3)] = by.packed();
      const int col = tx * kGroup + threadIdx.x;
      if (col < a.dim) a.scale[(int64_t)col * up + ty] = by.scale;
    }
  }
  __syncthreads();
  if constexpr (!TRANSPOSED) {
    const E4m3Scale by(scales[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f32x2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = pair_of(p[i], 2 * k);
      by.divide(v);
      uint16_t q[4];
      to_e4m3(q, v);
      if (row0 + i < a.rows && col0 < a.dim)
        store8(static_cast<uint8_t*>(a.out) + (int64_t)(row0 + i) * a.out_stride + col0, q,
               a.dim - col0, vec_out);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const E4m3Scale by(scales[BLOCKS ? 0 : j * 16 + cp]);
      f32x2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = pair(to_f32(p[2 * k].v[j]), to_f32(p[2 * k + 1].v[j]));
      by.divide(v);
      uint16_t q[4];
      to_e4m3(q, v);
      tile[(cp * 8 + j) * 16 + (rg ^ cp)] =
          make_uint2(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + rg;  // the tile's column, an output row; cp is its 8 values' place
      const uint2 u = tile[c * 16 + (cp ^ (c >> 3))];
      const uint16_t q[4] = {(uint16_t)u.x, (uint16_t)(u.x >> 16), (uint16_t)u.y,
                             (uint16_t)(u.y >> 16)};
      const int at = ty * kGroup + cp * 8, row = tx * kGroup + c;
      if (row < a.dim && at < a.rows)
        store8(static_cast<uint8_t*>(a.out) + (int64_t)row * a.out_stride + at, q, a.rows - at,
               vec_out);
    }
  }
}

}  // namespace

cudaError_t quantize_q8_launch(const salt_quantize_q8_args& a, cudaStream_t st, int* launches) {
  if (!a.rows) return cudaSuccess;
  const int groups = (a.dim + kGroup - 1) / kGroup;
  const size_t size = type_size(a.type);
  const bool vec_in = a.dim % 8 == 0 && pack_rows(a.x, 8, size, a.x_stride);
  const bool vec_out = packed_rows(a.out, 8, 1, a.out_stride, 0);
  if (!a.blocks && !a.transposed) {
    const int each = 16 * (a.type == SALT_F32 ? 2 : 4);  // groups of a block
    const int64_t blocks = ((int64_t)a.rows * groups + each - 1) / each;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    SALT_WITH_TYPE(a.type, T, {
      const auto kernel = vec_in ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
      kernel<<<(unsigned)blocks, 256, 0, st>>>(a, groups, vec_out);
    });
  } else {
    const int64_t up = (a.rows + (int64_t)kGroup - 1) / kGroup, tiles = up * groups;
    if (tiles > 0x7fffffff) return cudaErrorInvalidConfiguration;
    SALT_WITH_TYPE(a.type, T, {
      const auto kernel =
          vec_in ? (!a.transposed ? quantize_tile_kernel<T, true, true, false>
                    : a.blocks    ? quantize_tile_kernel<T, true, true, true>
                                  : quantize_tile_kernel<T, true, false, true>)
                 : (!a.transposed ? quantize_tile_kernel<T, false, true, false>
                    : a.blocks    ? quantize_tile_kernel<T, false, true, true>
                                  : quantize_tile_kernel<T, false, false, true>);
      kernel<<<(unsigned)tiles, 256, 0, st>>>(a, groups, vec_out);
    });
  }
  ++*launches;
  return cudaGetLastError();
}

}  // namespace salt
