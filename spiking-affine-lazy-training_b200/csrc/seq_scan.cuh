// What the selective scan's forward and backward kernels share: how channels and states lie on
// threads, the split of a row into chunks, and the staging of a tile of tokens.
#pragma once
#include "sequence.cuh"

namespace salt {


// A row's tokens are cut into `chunks` pieces of `chunk_len` tokens where channels and rows alone
// leave the GPU empty.  A first pass then runs the recurrence of each chunk from zero; the second
// starts each chunk from those results: h = exp(A * sum of steps) * h + (the chunk's own).
struct ScanSplit {
  int chunks, chunk_len;
  float* state;  // (batch, chunks, dim, state): [0] the initial state, [c] chunk c - 1's own result
  float* steps;  // (batch, chunks, dim): the sum of s over the chunk
};

// Into how many chunks of equal length rows are cut: those that need the least time, counted in
// rounds of the `slots` blocks that the GPU runs at once.  A split row pays for its first pass,
// `first` of the time of the second.
inline ScanSplit scan_split(int64_t blocks, int64_t slots, int32_t len, float first) {
  ScanSplit s{1, len > 0 ? len : 1, nullptr, nullptr};
  float least = 0.f;
  for (int c = 1; c <= 64 && (c == 1 || c * 128 <= len); ++c) {
    const int64_t rounds = (blocks * c + slots - 1) / slots;
    const float time = (float)rounds / c * (c > 1 ? 1.f + first : 1.f);
    if (c > 1 && time > 0.97f * least) continue;  // not for a trifle
    least = time;
    s.chunks = c;
  }
  if (s.chunks == 1) return s;
  s.chunk_len = ((len + s.chunks - 1) / s.chunks + 31) / 32 * 32;  // whole tiles and checkpoints
  s.chunks = (len + s.chunk_len - 1) / s.chunk_len;
  return s;
}

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
__device__ __forceinline__ f32x2 scan_step2(f32x2 raw, int softplus) {
  return softplus ? softplus2(raw) : raw;
}

// A token's decays exp(s A) of two states, A2 = A log2(e).  The one-instruction exponential is low by
// 0.1 units of 2^-24 on average for arguments near 0, by 0.35 for those of 2^-8 to 2^-7, by 0.6 and
// then 0.9 for larger ones (measured over all binades).  A state is a product of as many decays as it
// lives tokens, so that such an error, small beside the rounding's, grows with their number and not
// with its root.  A shift of the arguments, which the multiply-add has for nothing, leaves at most
// 0.16 units under 2^-7 and 0.35 under 2^-4, and 1 of an argument of 0.  Relative errors of dA against
// 64 bits, without and with it: 1.7e-6 and 0.7e-6 for 4 rows of 2048 tokens (the doubling scan of the
// plain form: 1.0e-6); shifts of 0.2, 0.3 and 0.45 units leave 0.8e-6, 0.6e-6 and 0.9e-6 there, and
// 0.8e-6, 0.8e-6 and 1.5e-6 for 3 rows of 1500 tokens x 4 states.
constexpr float kDecayShift = 0.25f * 0x1p-24f * kLog2e;
__device__ __forceinline__ f32x2 decay2(f32x2 A2, f32x2 s) {
  return exp2_fast2(fma2(A2, s, pair(kDecayShift, kDecayShift)));
}

// Calls ... with S the shape for `state` states.
#define SALT_BY_STATE(state, S, S4, S8, S16, S32, S64, ...) \
  do {                                                      \
    if ((state) <= 4) {                                     \
      using S = S4;                                         \
      __VA_ARGS__;                                          \
    } else if ((state) <= 8) {                              \
      using S = S8;                                         \
      __VA_ARGS__;                                          \
    } else if ((state) <= 16) {                             \
      using S = S16;                                        \
      __VA_ARGS__;                                          \
    } else if ((state) <= 32) {                             \
      using S = S32;                                        \
      __VA_ARGS__;                                          \
    } else {                                                \
      using S = S64;                                        \
      __VA_ARGS__;                                          \
    }                                                       \
  } while (0)

// How a tile's rows reach shared memory: in asynchronous copies of 16 bytes where every row starts
// on such a boundary and no pack is cut, of 4 where it does on those, else by plain loads.
constexpr int kCopy16 = 16, kCopy4 = 4, kCopyPlain = 0;

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool valid) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  const int bytes = valid ? BYTES : 0;  // the rest of the BYTES is filled with zeros
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(from), "n"(BYTES),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// N neighbouring elements at `from`, of which `n` are there (none if n <= 0), into shared memory;
// zeros behind them.
template <int COPY, int N, typename T>
__device__ __forceinline__ void copy_pack(T* to, const T* from, int n) {
  if constexpr (COPY == kCopyPlain) {
    const Pack<T, N> p = load_pack<T, N>(from, n, false);
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = p.v[i];
  } else {
    constexpr int bytes = COPY < (int)(N * sizeof(T)) ? COPY : N * sizeof(T);
    constexpr int each = bytes / sizeof(T);
#pragma unroll
    for (int i = 0; i < N; i += each) copy_async<bytes>(to + i, from + (i < n ? i : 0), i < n);
  }
}

// A tile of TILE tokens from t0 on and CH channels, of which n are there, into shared memory; zeros
// where the row (at `stop`) or its channels end.  In copies of 16 bytes each thread moves the P
// channels of one token that it converts itself; narrower ones go element by element through the
// rows, so that a warp's lie together, and the block has to meet before it reads them.
template <int COPY, int P, int TILE, int CH, int THREADS, typename T>
__device__ __forceinline__ void copy_tile(T (*to)[CH], const T* from, int64_t stride, int t0,
                                          int stop, int n) {
  constexpr int E = COPY == kCopy16 ? P : COPY == kCopy4 ? 4 / sizeof(T) : 1;
  constexpr int per = CH / E;
#pragma unroll
  for (int i = threadIdx.x; i < TILE * per; i += THREADS) {
    const int q = i / per, c = i % per * E;
    copy_pack<COPY, E>(&to[q][c], from + (int64_t)(t0 + q) * stride + c, t0 + q < stop ? n - c : 0);
  }
}
// The way back for narrow rows, once the block has met: tokens [t0, end) of the tile.
template <int COPY, int TILE, int CH, int THREADS, typename T>
__device__ __forceinline__ void store_tile(T* to, T (*from)[CH], int64_t stride, int t0, int end,
                                           int n) {
  constexpr int E = COPY == kCopy4 ? 4 / sizeof(T) : 1, per = CH / E;
#pragma unroll
  for (int i = threadIdx.x; i < TILE * per; i += THREADS) {
    const int q = i / per, c = i % per * E;
    if (t0 + q < end && c < n)
      *reinterpret_cast<Pack<T, E>*>(to + (int64_t)(t0 + q) * stride + c) =
          *reinterpret_cast<const Pack<T, E>*>(&from[q][c]);
  }
}

// A pack of shared memory that copy_pack filled.
template <int N, typename T>
__device__ __forceinline__ Pack<T, N> pack_at(const T* p) {
  return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T>
__device__ __forceinline__ void widen4(float* to, const T* from) {
  const Pack<T, 4> p = pack_at<4>(from);
  const float2 lo = halves(pair_of(p, 0)), hi = halves(pair_of(p, 2));
  *reinterpret_cast<float4*>(to) = make_float4(lo.x, lo.y, hi.x, hi.y);
}

// N values to global memory where rows are wide (n is a multiple of N or not positive), else to the
// same place of the tile that store_tile writes.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void scan_store(T* global, T* tile, const float* f, int n) {
  if (WIDE && n <= 0) return;
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(f[i]);
  *reinterpret_cast<Pack<T, N>*>(WIDE ? global : tile) = r;
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
