// What the selective scan's forward and backward kernels share: how channels and states lie on
// threads, the split of a row into chunks, and the staging of a tile of tokens.
#pragma once
#include "sequence.cuh"

namespace salt {

constexpr int kScanChannels = 64;  // channels of a block (fewer backward where state > 16)

// A row's tokens are cut into `chunks` pieces of `chunk_len` tokens where channels and rows alone
// leave the GPU empty.  A first pass then runs the recurrence of each chunk from zero; the second
// starts each chunk from those results: h = exp(A * sum of steps) * h + (the chunk's own).
struct ScanSplit {
  int chunks, chunk_len;
  float* state;  // (batch, chunks, dim, state): [0] the initial state, [c] chunk c - 1's own result
  float* steps;  // (batch, chunks, dim): the sum of s over the chunk
};

// Which 64 (or fewer) channels a block has: they lie in one group, so that B and C are shared.
struct ScanBlock {
  int d0, n, group;
};
__device__ __forceinline__ ScanBlock scan_block(int id, int dim, int groups, int channels) {
  const int per = dim / groups, blocks = (per + channels - 1) / channels;
  ScanBlock s;
  s.group = id / blocks;
  const int at = (id - s.group * blocks) * channels;
  s.d0 = s.group * per + at;
  s.n = min(channels, per - at);
  return s;
}
inline int scan_blocks(int dim, int groups, int channels) {
  const int per = dim / groups;
  return groups * ((per + channels - 1) / channels);
}

// s of one token and channel: softplus(delta + bias), or their sum.
__device__ __forceinline__ float scan_step(float raw, int softplus) {
  return softplus ? softplus_f(raw) : raw;
}

// NS neighbouring states of `p`, those at or past `n` as zero.
template <int NS>
__device__ __forceinline__ void load_states(float (&v)[NS], const float* p, int n, bool vec) {
#pragma unroll
  for (int i = 0; i < NS; i += 4) {
    if (vec && i + 4 <= n) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i + k] = i + k < n ? p[i + k] : 0.f;
    }
  }
}
template <int NS>
__device__ __forceinline__ void store_states(float* p, const float (&v)[NS], int n, bool vec) {
#pragma unroll
  for (int i = 0; i < NS; i += 4) {
    if (vec && i + 4 <= n) {
      *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) p[i + k] = v[i + k];
    }
  }
}

// Sums v[0 .. NV) over the lanes that differ in the bits [FROM, TO) of the lane index, leaving each
// lane with NV / (number of lanes) of the sums (at least one): at every halving a lane sends the
// half that its partner keeps.  `first` is the index of the sums a lane ends up with.  With fewer
// values than lanes the last steps leave the same sum on several lanes.
template <int NV, int FROM, int TO>
__device__ __forceinline__ void lane_sums(float* v, int lane, int& first) {
  if constexpr (FROM < TO) {
    const bool up = lane & FROM;
    if constexpr (NV > 1) {
      constexpr int H = NV / 2;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float send = up ? v[i] : v[i + H], keep = up ? v[i + H] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, FROM);
      }
      if (up) first += H;
      lane_sums<H, FROM * 2, TO>(v, lane, first);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], FROM);
      lane_sums<1, FROM * 2, TO>(v, lane, first);
    }
  }
}

}  // namespace salt
