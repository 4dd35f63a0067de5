// Product of two matrices in 8 bits with a float32 scale for every 128 values of the depth.
#include <cooperative_groups.h>

#include "sequence.cuh"
#include "tc.cuh"

namespace salt {
namespace {

namespace cg = cooperative_groups;

constexpr int kGroup = SALT_Q8_GROUP;
constexpr int kTileA = 128;           // rows of one operand in a block, the accumulators' lanes
constexpr int kSums = 256;             // threads that scale and add up: 8 warps
constexpr int kThreads = kSums + 128;  // behind them a warp for the copies, one for the products and two
                                       // for the scales
constexpr int kMostSplit = 8;
constexpr int kRing = 8;    // groups whose scales are in flight
constexpr int kBehind = 4;  // of them, those whose scales nobody has looked at

// Stages of both operands' tiles in flight.
constexpr int stages(int bn, bool swap) {
  return bn == 256 ? (swap ? 4 : 3) : bn == 128 ? (swap ? 6 : 5) : bn == 64 ? 8 : 9;
}
// Buffers of tensor memory for groups' products.
constexpr int buffers(int bn) { return bn >= 64 ? 512 / bn : 8; }
constexpr int stage_bytes(int bn) { return (kTileA + bn) * kGroup; }
constexpr int shared_bytes(int bn, bool swap) {
  return stages(bn, swap) * stage_bytes(bn) + (swap ? 0 : kSums / 32 * 4096) + 1024;
}

struct Product {
  int64_t rows_a, rows_b;
  int tiles_a, tiles_b, groups, split;
  int shift_a, shift_b;  // rows of a scale, as a power of two
  const float *scale_a, *scale_b;
  void* out;
  int64_t out_stride;
  const void* bias;
  bool bias_f32, vec;
};

// In its upper two bits, whether any of four scales lies outside 2^-47 to 2^17, between which two multiply
// to a normal number.  (Powers that let one instruction look at a scale, on the scale's way from memory.)
__device__ __forceinline__ uint32_t unusual_bits(float4 v) {
  constexpr uint32_t low = (127u - 47u) << 24;
  return ((__float_as_uint(v.x) << 1) - low) | ((__float_as_uint(v.y) << 1) - low) |
         ((__float_as_uint(v.z) << 1) - low) | ((__float_as_uint(v.w) << 1) - low);
}
// a b v where a b may overflow or be subnormal though the whole does not: the larger factor is the
// last one of a large product, the first one of a small.
__device__ __forceinline__ float scaled(float v, float a, float b) {
  const bool a_first = (fabsf(a) < fabsf(b)) == (fabsf(a * b) >= 1.f);
  return v * (a_first ? a : b) * (a_first ? b : a);
}

// out = sum over groups of scale_a scale_b (the group's product of e4m3 values).
//
// The tensor cores add up one group (128 x BN x 128, in 32 bits) into one of two to eight buffers of
// tensor memory; eight warps take it from there, times both scales, to their running sums in registers,
// while the next groups' products go to the other buffers.
//
// SWAP = false: rows of x are the lanes, weight rows the columns, and a warp's columns share one scale
// (blocks of 128).  SWAP = true: weight rows are the lanes, rows of x the columns, each with its own
// scale, which goes through shared memory; a warp's stores are then neighbours in a row of out.
//
// What bounds it: a scale for every 128 of the depth makes the sums a multiplication and an addition of
// every value for each group.  At BN = 256 a group's products take 512 cycles and its sums 360 of every
// scheduler's, next to some 250 of waiting at barriers and taking the values out of tensor memory:
// 16384 x 5120 x 5120 takes 436 us in bfloat16, 1.97 PFLOP/s (350 us without sums and outputs, 268 us
// the library's product with one scale a tensor).  Columns with a scale each take two multiplications a
// value: 2048 x 4096 x 8192 with both operands' scales by rows, to float32, 147 us, 0.94 PFLOP/s.  Few
// rows are bound by what a block waits for: 64 rows of 8192 x 8192 take 28 us, 2.4 TB/s; 16 rows of 2048
// x 4096 9 us, most of it the start, the first copies and the joining.
// The definition has (x scale) (weight scale), and a product of both scales may overflow or be subnormal
// where that does not: from the first group of a tile with such scales on, the values meet the scales one
// after the other.  That loop, with a look at the scales in every group, costs 1 to 3 % (432 -> 436 us
// above, 143 -> 147 us with scales by rows); as a branch beside every 16 values it cost a third.  With scales
// by rows the warps that copy them look, since the sums' warps have no instruction to spare: three
// instructions a scale in there took 162 us.
// Measured and left: two blocks on a tile of 256 x 256 (440 us then, as much as one), sixteen warps of
// sums (455), packed arithmetic for the sums (447), two sets of warps on every other group of narrow
// tiles (24.4 us for 64 rows).
template <int BN, bool SWAP, typename T>
__global__ void __launch_bounds__(kThreads, 1)
matmul_q8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_out, const Product p) {
  constexpr int S = stages(BN, SWAP), B = buffers(BN);
  constexpr int H = BN / 2, PIECE = H < 16 ? H : 16;  // a warp's columns, and those of a load
  constexpr int kCopies = kSums / 32, kProducts = kCopies + 1, kScales = kCopies + 2;  // warps
  extern __shared__ uint8_t raw[];
  uint8_t* tiles = raw + (1024 - tc::shared_at(raw) % 1024) % 1024;
  uint8_t* staged = tiles + S * stage_bytes(BN);  // SWAP = false: 4 KB a warp for rows of out
  __shared__ uint64_t full[S], empty[S], sum_full[B], sum_empty[B];
  __shared__ uint64_t drained;  // every product issued
  __shared__ uint32_t tmem_at, gave_up;  // (by a warp of sums)
  constexpr int kScalesB = SWAP ? BN : 4;  // of each column, or of each block of columns
  __shared__ __align__(16) float scales_a[kRing][kTileA], scales_b[kRing][kScalesB];
  __shared__ uint64_t scales_full[kRing], scales_empty[kRing];
  __shared__ uint2 unusual[kRing];  // SWAP: whether any of a group's scales is, of the lanes, of the columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      tc::barrier_init(&full[i], 1);
      tc::barrier_init(&empty[i], 1);
    }
    for (int i = 0; i < B; ++i) {
      tc::barrier_init(&sum_full[i], 1);
      tc::barrier_init(&sum_empty[i], kSums / 32);
    }
    for (int i = 0; i < kRing; ++i) {
      tc::barrier_init(&scales_full[i], 64);
      tc::barrier_init(&scales_empty[i], kSums / 32);
    }
    tc::barrier_init(&drained, 1);
    gave_up = 0;
    tc::barrier_init_fence();
    tc::prefetch_map(&map_a);
    tc::prefetch_map(&map_b);
  }
  constexpr uint32_t kColumns = B * BN;
  if (warp == kProducts) tc::tmem_alloc(&tmem_at, kColumns);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_at;
  // a worker is one block, or those that share the depth of a tile
  const int rank = blockIdx.x % p.split;
  const int worker = blockIdx.x / p.split, workers = gridDim.x / p.split;
  const int total = p.tiles_a * p.tiles_b;
  const int g0 = (int)((int64_t)p.groups * rank / p.split),
            g1 = (int)((int64_t)p.groups * (rank + 1) / p.split);
  // bands of 16 tiles of a, so that blocks at work at the same time share both operands in L2
  constexpr int kBand = 16;
  auto place = [&](int t, int& ta, int& tb) {
    const int band = t / (kBand * p.tiles_b), in = t - band * kBand * p.tiles_b;
    const int high = min(kBand, p.tiles_a - band * kBand);
    tb = in / high;
    ta = band * kBand + in - tb * high;
  };
  uint32_t tries = tc::kTries;

  if (warp >= kCopies) tc::registers_down<64>();
  if (warp == kCopies) {
    if (tc::one_lane()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int t = worker; tries && t < total; t += workers) {
        int ta, tb;
        place(t, ta, tb);
        for (int g = g0; g < g1; ++g) {
          tc::barrier_wait(&empty[stage], phase ^ 1, tries);
          if (!tries) break;
          uint8_t* a = tiles + stage * stage_bytes(BN);
          tc::barrier_expect(&full[stage], stage_bytes(BN));
          tc::load_box(a, &map_a, g * kGroup, ta * kTileA, &full[stage]);
          tc::load_box(a + kTileA * kGroup, &map_b, g * kGroup, tb * BN, &full[stage]);
          if (++stage == S) stage = 0, phase ^= 1;
        }
      }
      // all copies have to land before the block may end
      uint32_t more = tc::kTries;
      for (int i = 0; i < S; ++i) {
        tc::barrier_wait(&full[stage], phase ^ 1, more);
        if (++stage == S) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == kProducts) {
    if (tc::one_lane()) {
      int stage = 0, buffer = 0;
      uint32_t phase = 0, sum_phase = 0;
      for (int t = worker; tries && t < total; t += workers) {
        for (int g = g0; g < g1; ++g) {
          tc::barrier_wait(&sum_empty[buffer], sum_phase ^ 1, tries);
          tc::barrier_wait(&full[stage], phase, tries);
          if (!tries) break;
          tc::fence_after();
          const uint8_t* at = tiles + stage * stage_bytes(BN);
          const uint64_t a = tc::operand(at, 1024), b = tc::operand(at + kTileA * kGroup, 1024);
#pragma unroll
          for (int k = 0; k < kGroup; k += 32)
            tc::product_e4m3(tmem + buffer * BN, tc::further(a, k), tc::further(b, k),
                             tc::shape(kTileA, BN, 0), k > 0);
          tc::products_done(&sum_full[buffer]);
          tc::products_done(&empty[stage]);
          if (++stage == S) stage = 0, phase ^= 1;
          if (++buffer == B) buffer = 0, sum_phase ^= 1;
        }
      }
      uint32_t more = tc::kTries;  // and all products
      tc::products_done(&drained);
      tc::barrier_wait(&drained, 0, more);
    }
  } else if (warp >= kScales) {
    // a warp for the lanes' scales and one for the columns': a row's scales lie together, so that
    // every load takes as many lines as lanes, and here nobody waits for them
    const bool lanes = warp == kScales;
    const int n = lanes ? kTileA : kScalesB;
    int slot = 0, ready = 0, behind = 0;
    uint32_t phase = 0;
    const auto pass_on = [&] {  // the oldest group whose scales are there
      __syncwarp();
      const float4* at = reinterpret_cast<const float4*>(lanes ? scales_a[ready] : scales_b[ready]);
      uint32_t odd = lane * 4 < n ? unusual_bits(at[lane]) : 0;
      if (kScalesB > 128 && !lanes) odd |= unusual_bits(at[32 + lane]);
      const bool any = __any_sync(0xffffffffu, odd >> 30);
      if (lane == 0) (lanes ? unusual[ready].x : unusual[ready].y) = any;
      tc::barrier_arrive_if_zero(&scales_full[ready], 0);
      if (++ready == kRing) ready = 0;
      --behind;
    };
    for (int t = worker; tries && t < total; t += workers) {
      int ta, tb;
      place(t, ta, tb);
      const float* from[kTileA / 32 > kScalesB / 32 ? kTileA / 32 : kScalesB / 32];
#pragma unroll
      for (int i = 0; i < (int)(sizeof(from) / sizeof(from[0])); ++i) {
        const int at = i * 32 + lane;
        const int64_t row = lanes  ? (int64_t)ta * kTileA + at
                            : SWAP ? (int64_t)tb * BN + at
                                   : (int64_t)tb * BN + at * kGroup;
        from[i] = lanes ? p.scale_a + (min(row, p.rows_a - 1) >> p.shift_a) * p.groups
                        : p.scale_b + (min(row, p.rows_b - 1) >> p.shift_b) * p.groups;
      }
      for (int g = g0; g < g1; ++g) {
        tc::barrier_wait_warp(&scales_empty[slot], phase ^ 1, tries);
        if (!tries) break;
        float* to = (lanes ? scales_a[slot] : scales_b[slot]) + lane;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(from) / sizeof(from[0])); ++i)
          if (i * 32 + lane < n) tc::copy4(to + i * 32, from[i] + g);
        if constexpr (SWAP) {
          tc::copies_group();
          if (++behind > kBehind) {
            tc::copies_wait<kBehind>();
            pass_on();
          }
        } else {
          tc::copies_arrive(&scales_full[slot]);
        }
        if (++slot == kRing) slot = 0, phase ^= 1;
      }
    }
    tc::copies_done();
    while (SWAP && tries && behind > 0) pass_on();
  } else {
    tc::registers_up<216>();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16) + half * H;
    int buffer = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0;
    // A wait that is given up leaves NaN in this and all further tiles, and no arrival any more, so that
    // nothing overwrites what others still read.  (A mark within the waits, as in the attention kernel,
    // took 16384 x 5120 x 5120 from 422 us to 467.)
#pragma unroll 1
    for (int t = worker; t < total; t += workers) {
      float sum[H];
#pragma unroll
      for (int i = 0; i < H; ++i) sum[i] = 0.f;
      int g = tries ? g0 : g1;
      // (unrolled, the loop copies the sums in every turn)
#pragma unroll 1
      for (; g < g1; ++g) {
        tc::barrier_wait_warp(&scales_full[slot], slot_phase, tries);
        const float* sb = scales_b[slot];
        const float of_lane = scales_a[slot][quarter * 32 + lane];
        const float by = SWAP ? of_lane : of_lane * sb[half * H / kGroup];
        tc::barrier_wait_warp(&sum_full[buffer], phase, tries);
        tc::fence_after();
        uint32_t r[2][PIECE];
        tc::tmem_load<PIECE>(r[0], mine + buffer * BN);
        bool plain;
        if constexpr (SWAP) {
          const uint2 u = unusual[slot];
          plain = !(u.x | u.y);
        } else {  // a normal number
          plain = __all_sync(0xffffffffu, (__float_as_uint(by) << 1) - 0x01000000u < 0xfd000000u);
        }
        if (!plain) break;
#pragma unroll
        for (int c = 0; c < H; c += PIECE) {
          tc::loads_done();
          if (c + PIECE < H) {  // on its way while this piece is added
            tc::tmem_load<PIECE>(r[(c / PIECE + 1) % 2], mine + buffer * BN + c + PIECE);
          } else {
            tc::fence_before();
            __syncwarp();
            tc::barrier_arrive_if_zero(&sum_empty[buffer], tries ? lane : 1);
          }
          const uint32_t(&now)[PIECE] = r[c / PIECE % 2];
#pragma unroll
          for (int i = 0; i < PIECE; i += 4) {
            float4 v = make_float4(by, by, by, by);
            if (SWAP) {
              v = *reinterpret_cast<const float4*>(sb + half * H + c + i);
              v.x *= by, v.y *= by, v.z *= by, v.w *= by;
            }
            sum[c + i] = fmaf(__uint_as_float(now[i]), v.x, sum[c + i]);
            sum[c + i + 1] = fmaf(__uint_as_float(now[i + 1]), v.y, sum[c + i + 1]);
            sum[c + i + 2] = fmaf(__uint_as_float(now[i + 2]), v.z, sum[c + i + 2]);
            sum[c + i + 3] = fmaf(__uint_as_float(now[i + 3]), v.w, sum[c + i + 3]);
          }
        }
        __syncwarp();
        tc::barrier_arrive_if_zero(&scales_empty[slot], tries ? lane : 1);
        if (++slot == kRing) slot = 0, slot_phase ^= 1;
        if (++buffer == B) buffer = 0, phase ^= 1;
      }
#pragma unroll 1
      for (; g < g1; ++g) {  // near the ends of float32's range
        tc::barrier_wait_warp(&scales_full[slot], slot_phase, tries);
        const float* sb = scales_b[slot];
        const float of_lane = scales_a[slot][quarter * 32 + lane];
        tc::barrier_wait_warp(&sum_full[buffer], phase, tries);
        tc::fence_after();
        uint32_t r[2][PIECE];
        tc::tmem_load<PIECE>(r[0], mine + buffer * BN);
#pragma unroll
        for (int c = 0; c < H; c += PIECE) {
          tc::loads_done();
          if (c + PIECE < H) {  // on its way while this piece is added
            tc::tmem_load<PIECE>(r[(c / PIECE + 1) % 2], mine + buffer * BN + c + PIECE);
          } else {
            tc::fence_before();
            __syncwarp();
            tc::barrier_arrive_if_zero(&sum_empty[buffer], tries ? lane : 1);
          }
          const uint32_t(&now)[PIECE] = r[c / PIECE % 2];
#pragma unroll
          for (int i = 0; i < PIECE; ++i)
            sum[c + i] += scaled(__uint_as_float(now[i]), of_lane,
                                 sb[SWAP ? half * H + c + i : half * H / kGroup]);
        }
        __syncwarp();
        tc::barrier_arrive_if_zero(&scales_empty[slot], tries ? lane : 1);
        if (++slot == kRing) slot = 0, slot_phase ^= 1;
        if (++buffer == B) buffer = 0, phase ^= 1;
      }
      if (!tries) {  // a result that nobody can take for one
        gave_up = 1;
#pragma unroll
        for (int i = 0; i < H; ++i) sum[i] = __int_as_float(0x7fffffff);
      }
      if (p.split > 1) {
        // every block's part of the tile, [column][lane], in its own shared memory (all of this
        // block's copies and products are done: their sums are here)
        float* to = reinterpret_cast<float*>(tiles) + quarter * 32 + lane;
#pragma unroll
        for (int i = 0; i < H; ++i) to[(half * H + i) * kTileA] = sum[i];
        break;  // joined below
      }
      int ta, tb;
      place(t, ta, tb);
      const int64_t row = (int64_t)ta * kTileA + quarter * 32 + lane;
      const int64_t col0 = (int64_t)tb * BN + half * H;
      const int most = (int)min((int64_t)H, p.rows_b - col0);
      if constexpr (SWAP) {
        if (row >= p.rows_a) continue;
        const float b = p.bias ? weight_at<T>(p.bias, row, p.bias_f32) : 0.f;
        T* out = static_cast<T*>(p.out) + col0 * p.out_stride + row;
#pragma unroll
        for (int i = 0; i < H; ++i) {
          if (i < most) *out = from_f32<T>(sum[i] + b);
          out += p.out_stride;
        }
      } else {
        // Through shared memory: 128 bytes of each of the warp's rows at a time, in 16-byte units at
        // place unit ^ (row & 7), as a tensor copy takes them (or 8 lanes a row, side by side).
        constexpr int W = 128 / sizeof(T), U = 16 / sizeof(T);
        uint8_t* at = staged + warp * 4096;
        const int64_t row0 = row - lane;
#pragma unroll
        for (int c = 0; c < H; c += W) {
          if (c >= most) break;
          if (p.vec && lane == 0) tc::stores_read();
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            float f[U];
#pragma unroll
            for (int k = 0; k < U; ++k) f[k] = sum[c + u * U + k];
            if (p.bias) {
#pragma unroll
              for (int k = 0; k < U; ++k)
                if (c + u * U + k < most)
                  f[k] += weight_at<T>(p.bias, col0 + c + u * U + k, p.bias_f32);
            }
            store_pack<T, U>(reinterpret_cast<T*>(at + lane * 128 + (u ^ (lane & 7)) * 16), f, U,
                             true);
          }
          if (p.vec) {  // what lies past the edges is left out
            tc::fence_shared();
            __syncwarp();
            if (lane == 0 && row0 < p.rows_a)
              tc::store_box(&map_out, at, (int)col0 + c, (int)row0);
            continue;
          }
          __syncwarp();
          const int u = lane & 7, n = most - c - u * U;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (row0 + r >= p.rows_a || n <= 0) continue;
            const Pack<T, U> v =
                *reinterpret_cast<const Pack<T, U>*>(at + r * 128 + (u ^ (r & 7)) * 16);
            T* out = static_cast<T*>(p.out) + (row0 + r) * p.out_stride + col0 + c + u * U;
#pragma unroll
            for (int k = 0; k < U; ++k)
              if (k < n) out[k] = v.v[k];
          }
        }
      }
    }
  }
  if (!SWAP && lane == 0) tc::stores_done();
  __syncwarp();  // the copies' and the products' warps went apart
  if (p.split > 1) {
    // the blocks of a cluster hold parts of one tile: each adds up its share of the columns, in the
    // blocks' order
    cg::cluster_group cluster = cg::this_cluster();
    __syncthreads();
    if (tc::marked(&gave_up)) {  // copies that were under way until now may lie over the parts
      for (int i = threadIdx.x; i < BN * kTileA; i += kThreads)
        reinterpret_cast<float*>(tiles)[i] = __int_as_float(0x7fffffff);
    }
    cluster.sync();
    int ta, tb;
    place(worker, ta, tb);
    const int r = threadIdx.x & (kTileA - 1);
    const int64_t row = (int64_t)ta * kTileA + r;
    if (threadIdx.x < kSums && row < p.rows_a) {
      const float* parts[kMostSplit];
#pragma unroll
      for (int i = 0; i < kMostSplit; ++i)
        parts[i] = cluster.map_shared_rank(reinterpret_cast<float*>(tiles), i < p.split ? i : 0);
      const float b = SWAP && p.bias ? weight_at<T>(p.bias, row, p.bias_f32) : 0.f;
      for (int c = rank * 2 + (threadIdx.x >> 7); c < BN; c += 2 * p.split) {
        const int64_t col = (int64_t)tb * BN + c;
        if (col >= p.rows_b) break;
        float v[kMostSplit], s = 0.f;
#pragma unroll
        for (int i = 0; i < kMostSplit; ++i) v[i] = i < p.split ? parts[i][c * kTileA + r] : 0.f;
#pragma unroll
        for (int i = 0; i < kMostSplit; ++i) s += v[i];
        static_cast<T*>(p.out)[col * p.out_stride + row] = from_f32<T>(s + b);
      }
    }
    cluster.sync();  // the parts are read by others
  }
  tc::fence_before();
  __syncthreads();
  if (warp == kProducts) {
    tc::fence_after();
    tc::tmem_free(tmem, kColumns);
  }
}

// Rows on boundaries of 16 bytes: what a tensor copy needs, for operands that do not lie so.
// blockIdx.y is the operand.
struct Rows {
  const uint8_t* from;
  int64_t stride, rows;
  uint4* to;
};
struct BothRows {
  Rows r[2];
};
__global__ void __launch_bounds__(256) align_rows_kernel(const BothRows both, int k, int units) {
  const Rows x = both.r[blockIdx.y];
  const int64_t n = x.rows * units;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t row = n >> 32 ? i / units : (unsigned)i / (unsigned)units;
    const int at = (int)(i - row * units) * 16;
    const uint8_t* p = x.from + row * x.stride + at;
    uint32_t w[4] = {};
    const uintptr_t off = reinterpret_cast<uintptr_t>(p) & 3;
    if (at >= 4 && at + 20 <= k) {
      // whole words around the 16 bytes: all of them lie within this row
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p - off);
      uint32_t v[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) v[j] = q[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], (unsigned)off * 8);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (at + j < k) w[j / 4] |= (uint32_t)p[j] << (j % 4 * 8);
    }
    x.to[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---------------------------------------------------------------- host

using tc::encoder;
using tc::EncodeTiled;
using tc::kMostStride;

// Boxes of 128 bytes x `high` rows; what lies past k or the rows reads as zero.
bool tile_map(CUtensorMap* map, const void* p, int64_t rows, int64_t k, int64_t stride, int high) {
  const EncodeTiled f = encoder();
  if (!f) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {kGroup, (cuuint32_t)high}, unit[2] = {1, 1};
  return f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, unit,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 128 bytes x 32 rows of the output.
template <typename T>
bool out_map(CUtensorMap* map, void* p, int64_t rows, int64_t n, int64_t stride) {
  const EncodeTiled f = encoder();
  if (!f || stride * (int64_t)sizeof(T) >= kMostStride) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * sizeof(T)};
  const cuuint32_t box[2] = {128 / sizeof(T), 32}, unit[2] = {1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return f(map, type, 2, p, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t aligned_stride(int64_t k) { return (k + 15) / 16 * 16; }
bool tiled(const void* p, int64_t rows, int64_t stride, int64_t k) {
  return aligned16(p) && (rows == 1 || (stride % 16 == 0 && stride >= k && stride < kMostStride));
}
size_t copy_bytes(const void* p, int64_t rows, int64_t stride, int64_t k) {
  return tiled(p, rows, stride, k) ? 0 : ((size_t)rows * aligned_stride(k) + 255) / 256 * 256;
}

struct Operand {
  const void* p;
  int64_t rows, stride;
};
// Both operands as tensor copies can take them, copied to the workspace where they are not.
cudaError_t prepare(Operand* const (&all)[2], int64_t k, uint8_t* ws, cudaStream_t st, int* launches) {
  BothRows to = {};
  int count = 0;
  int64_t most = 0;
  const int units = (int)(aligned_stride(k) / 16);
  for (Operand* o : all) {
    if (tiled(o->p, o->rows, o->stride, k)) {
      if (o->rows == 1) o->stride = aligned_stride(k);
      continue;
    }
    to.r[count++] = {static_cast<const uint8_t*>(o->p), o->stride, o->rows,
                     reinterpret_cast<uint4*>(ws)};
    most = std::max(most, o->rows * units);
    const size_t bytes = copy_bytes(o->p, o->rows, o->stride, k);
    o->p = ws;
    o->stride = aligned_stride(k);
    ws += bytes;
  }
  if (!count) return cudaSuccess;
  align_rows_kernel<<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, 148 * 8), count), 256, 0,
                      st>>>(to, (int)k, units);
  ++*launches;
  return cudaGetLastError();
}

template <int BN, bool SWAP, typename T>
cudaError_t launch(Operand a, Operand b, int64_t k, Product p, cudaStream_t st, int* launches) {
  p.tiles_a = (int)((p.rows_a + kTileA - 1) / kTileA);
  p.tiles_b = (int)((p.rows_b + BN - 1) / BN);
  CUtensorMap map_a, map_b, map_out = {};
  if (!tile_map(&map_a, a.p, a.rows, k, a.stride, kTileA) ||
      !tile_map(&map_b, b.p, b.rows, k, b.stride, BN))
    return cudaErrorInvalidValue;
  if (!SWAP && p.vec && !out_map<T>(&map_out, p.out, p.rows_a, p.rows_b, p.out_stride)) p.vec = false;
  const auto kernel = matmul_q8_kernel<BN, SWAP, T>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = tc::allow_shared(reinterpret_cast<const void*>(kernel),
                                         shared_bytes(BN, SWAP), allowed);
  if (e != cudaSuccess) return e;
  const int64_t total = (int64_t)p.tiles_a * p.tiles_b;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)(p.split > 1 ? total * p.split : std::min<int64_t>(total, 148)));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = shared_bytes(BN, SWAP);
  c.stream = st;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  c.attrs = &attr;
  c.numAttrs = p.split > 1;
  ++*launches;
  return cudaLaunchKernelEx(&c, kernel, map_a, map_b, map_out, (const Product)p);
}

template <typename T>
cudaError_t run(const salt_matmul_q8_args& a, const Operand& x, const Operand& w, cudaStream_t st,
                int* launches) {
  Product p = {};
  p.groups = (a.k + kGroup - 1) / kGroup;
  p.split = 1;
  p.out = a.out;
  p.out_stride = a.out_stride;
  p.bias = a.bias;
  p.bias_f32 = a.bias_type == SALT_F32;
  const int shift_w = a.weight_rows ? 0 : 7;
  // Time in us by rounds of resident blocks (one an SM); `each` is what a group of a tile takes,
  // measured at full rounds with a depth of 2048 to 8192.  (1024 x 4096 x 4096: 128 tiles of 128 x 256
  // take 28 us, 256 tiles of 128 x 128 37 us.)
  const auto time = [&](int64_t tiles, double each, int split) {
    return (double)((tiles * split + 147) / 148) * (each * ((p.groups + split - 1) / split) + 1) +
           (split > 1 ? 2 : 0);
  };
  const auto tiles = [&](int64_t lanes, int64_t columns, int bn) {
    return ((lanes + kTileA - 1) / kTileA) * ((columns + bn - 1) / bn);
  };
  // few tiles: blocks share the depth of each
  const auto split_of = [&](int bn) {
    const int64_t n = tiles(a.n, a.rows, bn);
    int s = 1;
    while (s < kMostSplit && n * s * 2 <= 148 && p.groups >= s * 4) s *= 2;
    return s;
  };
  const auto by_columns = [&](int bn, double each) {
    return time(tiles(a.n, a.rows, bn), each, split_of(bn));
  };
  const double least = std::min(by_columns(128, 0.5), time(tiles(a.n, a.rows, 256), 1.0, 1));
  if (!a.weight_rows && a.rows > 64) {
    const double wide = time(tiles(a.rows, a.n, 256), 0.63, 1),
                 narrow = time(tiles(a.rows, a.n, 128), 0.5, 1);
    if (std::min(wide, narrow) <= least) {
      p.rows_a = a.rows, p.rows_b = a.n;
      p.scale_a = a.x_scale, p.scale_b = a.weight_scale;
      p.shift_a = 0, p.shift_b = shift_w;
      p.vec = packed_rows(a.out, 16, sizeof(T), a.out_stride, 0);
      return wide <= narrow ? launch<256, false, T>(x, w, a.k, p, st, launches)
                            : launch<128, false, T>(x, w, a.k, p, st, launches);
    }
  }
  p.rows_a = a.n, p.rows_b = a.rows;
  p.scale_a = a.weight_scale, p.scale_b = a.x_scale;
  p.shift_a = shift_w, p.shift_b = 0;
  const int bn = a.rows <= 16   ? 16
                 : a.rows <= 32 ? 32
                 : a.rows <= 64 ? 64
                 : by_columns(128, 0.5) <= least ? 128
                                                 : 256;
  p.split = bn == 256 ? 1 : split_of(bn);
  switch (bn) {
    case 16: return launch<16, true, T>(w, x, a.k, p, st, launches);
    case 32: return launch<32, true, T>(w, x, a.k, p, st, launches);
    case 64: return launch<64, true, T>(w, x, a.k, p, st, launches);
    case 128: return launch<128, true, T>(w, x, a.k, p, st, launches);
    default: return launch<256, true, T>(w, x, a.k, p, st, launches);
  }
}

}  // namespace

size_t matmul_q8_bytes(const salt_matmul_q8_args& a) {
  if (!a.rows) return 0;
  return copy_bytes(a.x, a.rows, a.x_stride, a.k) + copy_bytes(a.weight, a.n, a.weight_stride, a.k);
}

cudaError_t matmul_q8_launch(const salt_matmul_q8_args& a, void* ws, cudaStream_t st,
                             int* launches) {
  if (!a.rows) return cudaSuccess;
  Operand x{a.x, a.rows, a.x_stride}, w{a.weight, a.n, a.weight_stride};
  cudaError_t e = prepare({&x, &w}, a.k, static_cast<uint8_t*>(ws), st, launches);
  if (e != cudaSuccess) return e;
  SALT_WITH_TYPE(a.type, T, e = run<T>(a, x, w, st, launches));
  return e;
}

}  // namespace salt
