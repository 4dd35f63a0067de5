// Quantisation to 8 bits with a scale for every 128 values.
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

// Rows by groups of 128: half a warp a group, 8 elements a lane, four groups' loads on their way at a
// time.  Bound by memory: type + 1 bytes an element.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(salt_quantize_q8_args a, unsigned groups,
                                                            bool vec_in, bool vec_out) {
  constexpr int N = sizeof(T) == 4 ? 2 : 4;
  const int64_t n = (int64_t)a.rows * groups;
  const int lane = threadIdx.x & 15;
  const int64_t first = ((int64_t)blockIdx.x * N * 16) + (threadIdx.x >> 4);
  // (a product of 32 bits where the rows allow it: a division of 64 would cost as much as the rest)
  Pack<T, 8> p[N];
  int64_t row[N];
  int at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = first + i * 16;
    row[i] = g >> 32 ? g / groups : (unsigned)g / groups;
    at[i] = (int)(g - row[i] * groups) * kGroup + lane * 8;
    p[i] = load_pack<T, 8>(static_cast<const T*>(a.x) + row[i] * a.x_stride + at[i],
                           g < n ? a.dim - at[i] : 0, vec_in);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = first + i * 16;
    f32x2 v[4];
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = pair_of(p[i], 2 * k);
      const float2 h = halves(v[k]);
      most = fmaxf(most, fmaxf(fabsf(h.x), fabsf(h.y)));
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const E4m3Scale by(most);
    if (g < n && lane == 0) a.scale[g] = by.scale;
    by.divide(v);
    uint16_t q[4];
    to_e4m3(q, v);
    if (g < n && at[i] < a.dim)
      store8(static_cast<uint8_t*>(a.out) + row[i] * a.out_stride + at[i], q, a.dim - at[i], vec_out);
  }
}

// Tiles of 128 x 128 for scales of whole blocks, for transposed outputs, or both.  A thread holds 8
// neighbouring rows of 8 columns; a transposed tile goes through shared memory, where 8 values of a
// column lie together and their place in the column's 16 is turned by the column's pack, so that
// a half-warp's writes spread over all banks.  Scales are made once a column (or tile) and read from
// shared memory.  Bound by memory: type + 1 bytes an element.
template <typename T, bool BLOCKS, bool TRANSPOSED>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2)
quantize_tile_kernel(salt_quantize_q8_args a, int tiles_x, bool vec_in, bool vec_out) {
  __shared__ float red[8][kGroup];
  __shared__ E4m3Scale scales[BLOCKS ? 1 : kGroup];
  __shared__ uint2 tile[TRANSPOSED ? kGroup * 16 : 1];
  const int ty = blockIdx.x / tiles_x, tx = blockIdx.x - ty * tiles_x;
  const int cp = threadIdx.x & 15, rg = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int row0 = ty * kGroup + rg * 8, col0 = tx * kGroup + cp * 8;
  const int up = (a.rows + kGroup - 1) / kGroup;
  Pack<T, 8> p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    p[i] = load_pack<T, 8>(static_cast<const T*>(a.x) + (int64_t)(row0 + i) * a.x_stride + col0,
                           row0 + i < a.rows ? a.dim - col0 : 0, vec_in);
  float most[8];  // of each column
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    most[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most[j] = fmaxf(most[j], fabsf(to_f32(p[i].v[j])));
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
      scales[0] = E4m3Scale(m);
      a.scale[TRANSPOSED ? (int64_t)tx * up + ty : (int64_t)ty * tiles_x + tx] = scales[0].scale;
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
      scales[threadIdx.x] = E4m3Scale(m);
      const int col = tx * kGroup + threadIdx.x;
      if (col < a.dim) a.scale[(int64_t)col * up + ty] = scales[threadIdx.x].scale;
    }
  }
  __syncthreads();
  if constexpr (!TRANSPOSED) {
    const E4m3Scale by = scales[0];
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
      const E4m3Scale by = scales[BLOCKS ? 0 : cp * 8 + j];
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
  const bool vec_in = pack_rows(a.x, 8, size, a.x_stride);
  const bool vec_out = packed_rows(a.out, 8, 1, a.out_stride, 0);
  if (!a.blocks && !a.transposed) {
    const int each = 16 * (a.type == SALT_F32 ? 2 : 4);  // groups of a block
    const int64_t blocks = ((int64_t)a.rows * groups + each - 1) / each;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    SALT_WITH_TYPE(a.type, T, quantize_rows_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(
                                  a, groups, vec_in, vec_out));
  } else {
    const int64_t up = (a.rows + (int64_t)kGroup - 1) / kGroup, tiles = up * groups;
    if (tiles > 0x7fffffff) return cudaErrorInvalidConfiguration;
    SALT_WITH_TYPE(a.type, T, {
      const auto kernel = !a.transposed ? quantize_tile_kernel<T, true, false>
                          : a.blocks    ? quantize_tile_kernel<T, true, true>
                                        : quantize_tile_kernel<T, false, true>;
      kernel<<<(unsigned)tiles, 256, 0, st>>>(a, groups, vec_in, vec_out);
    });
  }
  ++*launches;
  return cudaGetLastError();
}

}  // namespace salt
