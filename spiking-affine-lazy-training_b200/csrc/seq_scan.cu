// Selective state space scan, whole rows and single tokens.
//
// h = exp(s A) h + s x B, y = C h: per token and channel one exponential and four multiply-adds for
// each state, against one read of x, delta and z and one write of out for all of them.  What bounds
// the scan is the exponentials (16 a cycle and SM) and the shared memory that hands B, C and s to
// every lane (128 bytes a cycle), not memory: 8 rows of 2048 tokens x 4096 channels x 16 states in
// bf16 take 488 us, where the exponentials (the states' and four a token and channel) need 290 us
// and the bytes 83 us.  The same rows ragged, from none to 2048 tokens: 304 to 319 us by the order of
// their lengths.
#include <algorithm>

#include "seq_scan.cuh"

namespace salt {

namespace {

// LPC lanes hold a channel's states, NS each, and CPT channels each: what a lane reads of B and C
// serves both.  A thread loads and stores 8 neighbouring channels of one token.
template <int NS_, int LPC_, int CPT_>
struct Shape {
  static constexpr int NS = NS_, LPC = LPC_, CPT = CPT_;
  static constexpr int kChannels = LPC == 1 ? 64 : 32;  // of a block
  static constexpr int kThreads = kChannels * LPC / CPT;
  static constexpr int kIo = kChannels / kVec;  // threads of one token
  static constexpr int kTile = kThreads / kIo;  // tokens
  static constexpr int kStates = NS * LPC;
  static constexpr int kStepPitch = kChannels + 4;  // 4 tokens' stores on 32 banks
  static constexpr int kYPitch = kChannels + 8;
};

// Where a channel of a block lies in shared memory: channel 8 v + k at place kIo k + v, so that the
// threads of a token store next to each other.  This is the channel at a place.
template <class S>
__device__ __forceinline__ int scan_channel(int place) {
  return place % S::kIo * kVec + place / S::kIo;
}

constexpr int kStages = 2;  // tiles in shared memory as they were loaded: this one and the next

template <typename T, class S, bool FULL>
struct ScanShared {
  struct Raw {
    alignas(16) T x[S::kTile][S::kChannels], delta[S::kTile][S::kChannels];
    alignas(16) T z[FULL ? S::kTile : 1][S::kChannels];
    alignas(16) T bc[FULL ? 2 : 1][S::kTile][S::kStates];
  } raw[kStages];  // loaded into registers a tile ahead they took 20 % longer
  alignas(16) float2 step[S::kTile][S::kStepPitch];  // s and s * x
  alignas(16) float B[S::kTile][S::kStates];
  alignas(16) float C[FULL ? S::kTile : 1][S::kStates];
  alignas(8) float y[FULL ? S::kTile : 1][S::kYPitch];
};

// The state in front of chunk c, from the first pass's results.
template <int NS>
__device__ __forceinline__ void chunk_start(float (&h)[NS], const float (&A2)[NS],
                                            const ScanSplit& sp, int64_t b, int c, int64_t dim,
                                            int64_t d, int state, int n0, bool vec) {
  const int64_t step = dim * state;
  const float* own = sp.state + (b * sp.chunks * dim + d) * state + n0;
  load_states<NS>(h, own + (c ? step : 0), state - n0, vec);
  for (int k = 2; k <= c; ++k) {
    float l[NS];
    load_states<NS>(l, own + k * step, state - n0, vec);
    const float s = sp.steps[(b * sp.chunks + k - 1) * dim + d];
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = fmaf(exp2_fast(A2[i] * s), h[i], l[i]);
  }
}

// Warps of an SM that the registers are held down for.  What measured best at 16 states (8 rows of
// 2048 x 4096, and the same ragged): one channel a lane at 20 warps 516 and 322 us, at 24 warps and
// loops of 4 tokens 550 and 329 us; two channels at 16 warps 500 and 373 us, whose fewer reads of
// shared memory do not make up for half the warps.
template <typename T, class S>
constexpr int resident() {
  return (S::NS == 4 ? 20 : 16) * 32 / S::kThreads;
}

// FULL: the scan.  Otherwise the first pass over a split row: chunk c's state from zero (chunk 0's
// from the initial state) into place c + 1, and the sum of its steps; the last chunk has no
// successor and is not run.
template <typename T, class S, bool FULL, int COPY>
__global__ void __launch_bounds__(S::kThreads, resident<T, S>())
selective_scan_kernel(salt_selective_scan_args a, ScanSplit sp, int blocks, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, CPT = S::CPT, H = NS / 2;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  ScanShared<T, S, FULL>& sm = *reinterpret_cast<ScanShared<T, S, FULL>*>(raw_shared);
  const int tid = threadIdx.x, chunks = FULL ? sp.chunks : sp.chunks - 1;
  const int64_t b = blockIdx.x / (blocks * chunks);
  const int rest = (int)(blockIdx.x - b * blocks * chunks), c = rest / blocks;
  const ScanBlock cb = scan_block(rest - c * blocks, a.dim, a.groups, S::kChannels);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, end = min(begin + sp.chunk_len, a.len);
  const int stop = min(real, end);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;  // the chunk with the last token

  // this thread's channels and states in the recurrence
  const int at = tid / LPC * CPT, n0 = tid % LPC * NS, ns = a.state - n0;
  bool mine[CPT];
  int64_t d[CPT];
  f32x2 A2[CPT][H], h[CPT][H];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int ch = scan_channel<S>(at + j);
    mine[j] = ch < cb.n;
    d[j] = cb.d0 + (mine[j] ? ch : 0);
    float f[NS], s[NS];
    load_states<NS>(f, a.A + d[j] * a.state + n0, mine[j] ? ns : 0, svec);
#pragma unroll
    for (int i = 0; i < NS; ++i) f[i] *= kLog2e;
    if (FULL && sp.chunks > 1)
      chunk_start<NS>(s, f, sp, b, min(c, last), a.dim, d[j], a.state, n0, svec);
    else
      load_states<NS>(s, a.initial_state + (b * a.dim + d[j]) * a.state + n0,
                      mine[j] && a.initial_state && c == 0 ? ns : 0, svec);
    if (!FULL && c == 0 && mine[j])
      store_states<NS>(sp.state + (b * sp.chunks * a.dim + d[j]) * a.state + n0, s, ns, svec);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      A2[j][i] = pair(f[2 * i], f[2 * i + 1]);
      h[j][i] = pair(s[2 * i], s[2 * i + 1]);
    }
  }
  auto store_h = [&](int j, float* to) {
    float f[NS];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float2 v = halves(h[j][i]);
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
    store_states<NS>(to + d[j] * a.state + n0, f, ns, svec);
  };

  // and its 8 channels of one token in loads and stores
  const int io_t = tid / S::kIo, io_v = tid % S::kIo;
  const int io_d = cb.d0 + io_v * kVec, io_n = cb.n - io_v * kVec;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + cb.d0;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + cb.d0;
  const T* z = FULL && a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + cb.d0 : nullptr;
  T* out = static_cast<T*>(a.out) + b * a.out_batch_stride + cb.d0;
  constexpr bool WIDE = COPY == kCopy16;
  const T* B = static_cast<const T*>(a.B) + b * a.B_batch_stride + (int64_t)cb.group * a.state;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  f32x2 bias[kVec / 2], skip[kVec / 2];
#pragma unroll
  for (int k = 0; k < kVec; k += 2) {
    const bool one = k < io_n, two = k + 1 < io_n;
    bias[k / 2] = a.delta_bias ? pair(one ? a.delta_bias[io_d + k] : 0.f,
                                      two ? a.delta_bias[io_d + k + 1] : 0.f)
                               : 0;
    skip[k / 2] =
        a.D ? pair(one ? a.D[io_d + k] : 0.f, two ? a.D[io_d + k + 1] : 0.f) : 0;
  }
  // In copies of 16 bytes each thread copies what it converts itself: its 8 channels of one token,
  // and packs of 4 states of B and C.  So a copy has arrived for its reader once that thread has
  // waited for it.
  constexpr int kPacks = S::kTile * S::kStates / 4;
  auto load = [&](int t0) {
    auto& raw = sm.raw[t0 / S::kTile % kStages];
    auto tile = [&](T(*to)[S::kChannels], const T* from, int64_t stride) {
      copy_tile<COPY, kVec, S::kTile, S::kChannels, S::kThreads>(to, from, stride, t0, stop, cb.n);
    };
    tile(raw.x, x, a.x_stride);
    tile(raw.delta, delta, a.delta_stride);
    if (z) tile(raw.z, z, a.z_stride);
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      const int left = t0 + q < stop ? a.state - n1 : 0;
      copy_pack<COPY, 4>(&raw.bc[0][q][n1], B + (t0 + q) * a.B_stride + n1, left);
      if (FULL)
        copy_pack<COPY, 4>(&raw.bc[FULL ? 1 : 0][q][n1], C + (t0 + q) * a.C_stride + n1, left);
    }
    copies_commit();
  };

  float sum[CPT] = {};
  if (begin < stop) load(begin);
  for (int t0 = begin; t0 < (FULL ? end : stop); t0 += S::kTile) {
    const int t = t0 + io_t;
    auto& raw = sm.raw[t0 / S::kTile % kStages];
    if (t0 < stop) {
      if (t0 + S::kTile < stop) {
        load(t0 + S::kTile);
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      if (!WIDE) __syncthreads();
      const auto px = pack_at<kVec>(&raw.x[io_t][io_v * kVec]);
      const auto pd = pack_at<kVec>(&raw.delta[io_t][io_v * kVec]);
#pragma unroll
      for (int k = 0; k < kVec; k += 2) {
        const f32x2 in = add2(pair_of(pd, k), bias[k / 2]);
        // past the last token s = 0: the state stays as it is
        const f32x2 s2 = t < stop ? scan_step2(in, a.softplus) : 0;
        const float2 s = halves(s2), sx = halves(mul2(s2, pair_of(px, k)));
        sm.step[io_t][k * S::kIo + io_v] = make_float2(s.x, sx.x);
        sm.step[io_t][(k + 1) * S::kIo + io_v] = make_float2(s.y, sx.y);
      }
      for (int i = tid; i < kPacks; i += S::kThreads) {
        const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
        widen4(&sm.B[q][n1], &raw.bc[0][q][n1]);
        if (FULL) widen4(&sm.C[FULL ? q : 0][n1], &raw.bc[FULL ? 1 : 0][q][n1]);
      }
    }
    __syncthreads();
    if (t0 < stop) {
      constexpr int kUnroll = 4;
#pragma unroll kUnroll
      for (int g = 0; g < S::kTile; g += 4) {
        if (FULL && a.checkpoints && (t0 + g) % SALT_SCAN_CHECKPOINT == 0 && t0 + g < stop) {
          const int64_t per = (a.len + SALT_SCAN_CHECKPOINT - 1) / SALT_SCAN_CHECKPOINT;
          float* to = a.checkpoints + (b * per + (t0 + g) / SALT_SCAN_CHECKPOINT) * a.dim * a.state;
#pragma unroll
          for (int j = 0; j < CPT; ++j)
            if (mine[j]) store_h(j, to);
        }
        float yq[4 * CPT];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x2 s[CPT], sx[CPT], y2[CPT];
          float2 st[CPT];
          if constexpr (CPT == 2) {
            const float4 v = *reinterpret_cast<const float4*>(&sm.step[g + q][at]);
            st[0] = make_float2(v.x, v.y), st[1] = make_float2(v.z, v.w);
          } else {
            st[0] = sm.step[g + q][at];
          }
#pragma unroll
          for (int j = 0; j < CPT; ++j) {
            s[j] = pair(st[j].x, st[j].x), sx[j] = pair(st[j].y, st[j].y);
            if (!FULL) sum[j] += st[j].x;
          }
#pragma unroll
          for (int i = 0; i < NS; i += 4) {
            const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&sm.B[g + q][n0 + i]);
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
              f32x2 &h0 = h[j][i / 2], &h1 = h[j][i / 2 + 1];
              h0 = fma2(decay2(A2[j][i / 2], s[j]), h0, mul2(sx[j], bn.x));
              h1 = fma2(decay2(A2[j][i / 2 + 1], s[j]), h1, mul2(sx[j], bn.y));
            }
            if (FULL) {
              const ulonglong2 cn = *reinterpret_cast<const ulonglong2*>(&sm.C[g + q][n0 + i]);
#pragma unroll
              for (int j = 0; j < CPT; ++j) {
                y2[j] = i ? fma2(h[j][i / 2], cn.x, y2[j]) : mul2(h[j][0], cn.x);
                y2[j] = fma2(h[j][i / 2 + 1], cn.y, y2[j]);
              }
            }
          }
          if (FULL) {
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
              const float2 v = halves(y2[j]);
              yq[q * CPT + j] = v.x + v.y;
            }
          }
        }
        if (FULL) {
          int first = 0;
          lane_sums<4 * CPT, 1, LPC>(yq, tid, first);
          constexpr int kept = 4 * CPT / LPC;
#pragma unroll
          for (int i = 0; i < kept; ++i)
            sm.y[g + (first + i) / CPT][at + (first + i) % CPT] = yq[i];
        }
      }
    }
    __syncthreads();
    if (FULL && t < end) {
      const auto px = pack_at<kVec>(&raw.x[io_t][io_v * kVec]);
      const auto pz = pack_at<kVec>(&raw.z[FULL ? io_t : 0][io_v * kVec]);
      float y[kVec];
#pragma unroll
      for (int k = 0; k < kVec; k += 2) {
        f32x2 v = 0;
        if (t < stop) {
          v = fma2(skip[k / 2], pair_of(px, k),
                   pair(sm.y[FULL ? io_t : 0][k * S::kIo + io_v],
                        sm.y[FULL ? io_t : 0][(k + 1) * S::kIo + io_v]));
          if (z) {
            const f32x2 g = pair_of(pz, k);
            v = mul2(v, mul2(g, sigmoid2(g)));
          }
        }
        const float2 f = halves(v);
        y[k] = f.x, y[k + 1] = f.y;
      }
      scan_store<T, kVec, WIDE>(out + t * a.out_stride + io_v * kVec, &raw.x[io_t][io_v * kVec], y,
                                io_n);
    }
    if (FULL && !WIDE) {
      __syncthreads();
      store_tile<COPY, S::kTile, S::kChannels, S::kThreads>(out, raw.x, a.out_stride, t0, end,
                                                            cb.n);
      __syncthreads();
    }
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    if (!mine[j]) continue;
    if (!FULL) {
      store_h(j, sp.state + (b * sp.chunks + c + 1) * a.dim * a.state);
      if (n0 == 0) sp.steps[(b * sp.chunks + c) * a.dim + d[j]] = sum[j];
    } else if (c == last && a.final_state) {
      store_h(j, a.final_state + b * a.dim * a.state);
    }
  }
}

// ---------------------------------------------------------------- single tokens

constexpr int kStepChannels = 64;  // of a block

template <int NS_, int LPC_>
struct StepShape {
  static constexpr int NS = NS_, LPC = LPC_;
  static constexpr int kThreads = kStepChannels * LPC;
};

// What one token's row needs beside its states; loaded a row ahead.
template <typename T, int NS>
struct StepRow {
  T x, delta, z;
  Pack<T, 4> B[NS / 4], C[NS / 4];
};

// Rows whose states are on their way to shared memory, in 32 KB of it at most.
template <class S>
constexpr int step_depth() {
  const int fit = 32 * 1024 / (S::kThreads * S::NS * 4);
  return fit < 4 ? fit : 4;
}

// A block holds A of its 64 channels and walks over `rows` tokens' rows.  The states' bytes, read
// and written once, are the bound: 8 a state and token, against 2 of x, z, delta and out.  VEC:
// states come by asynchronous copies, each thread its own, some rows ahead; registers would hold
// one row ahead at most.  256 rows x 8192 channels x 16 states: 67 to 70 us, 4.1 TB/s or 63 % of
// the measured copy rate (82 us with 4 lanes a channel, each of which works out s and the gate; 76
// us with the states a row ahead in registers).
template <typename T, class S, bool VEC>
__global__ void __launch_bounds__(S::kThreads)
selective_scan_step_kernel(salt_selective_scan_step_args a, int blocks, int rows) {
  constexpr int NS = S::NS, LPC = S::LPC, kStepDepth = step_depth<S>();
  __shared__ float4 ring[VEC ? kStepDepth : 1][NS / 4][S::kThreads];
  const int tid = threadIdx.x, part = blockIdx.x / blocks;
  const ScanBlock cb = scan_block(blockIdx.x - part * blocks, a.dim, a.groups, kStepChannels);
  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  const int64_t begin = (int64_t)part * rows, end = min((int64_t)a.batch, begin + rows);
  // the rows' slots, one a lane: a state's load does not wait for its slot's
  const int lane = tid & 31;
  int mine_slot = (int)begin + lane;
  if (a.slots && begin + lane < end) mine_slot = a.slots[begin + lane];
  auto pool_of = [&](int64_t b) -> float* {  // NULL: an empty row
    const int64_t slot = __shfl_sync(0xffffffffu, mine_slot, (int)(b - begin) & 31);
    return slot >= 0 && slot < a.n_slots ? a.pool + (slot * a.dim + d) * a.state + n0 : nullptr;
  };
  auto fetch = [&](int64_t b) {
    if (b < end) {
      const float* pool = pool_of(b);
      if (pool)
#pragma unroll
        for (int i = 0; i < NS; i += 4)
          copy_async<16>(&ring[(b - begin) % kStepDepth][i / 4][tid], pool + (i < ns ? i : 0),
                         i < ns);
    }
    copies_commit();
  };
  auto load = [&](StepRow<T, NS>& r, int64_t b) {
    r.x = static_cast<const T*>(a.x)[b * a.x_stride + d];
    r.delta = static_cast<const T*>(a.delta)[b * a.delta_stride + d];
    if (a.z) r.z = static_cast<const T*>(a.z)[b * a.z_stride + d];
    const int64_t at = (int64_t)cb.group * a.state + (ns > 0 ? n0 : 0);
#pragma unroll
    for (int i = 0; i < NS; i += 4) {
      const T* B = static_cast<const T*>(a.B) + b * a.B_stride + at;
      const T* C = static_cast<const T*>(a.C) + b * a.C_stride + at;
      r.B[i / 4] = VEC ? load_whole<T, 4>(B, i, ns) : load_pack<T, 4>(B + i, ns - i, false);
      r.C[i / 4] = VEC ? load_whole<T, 4>(C, i, ns) : load_pack<T, 4>(C + i, ns - i, false);
    }
  };
  if (VEC)
#pragma unroll
    for (int i = 0; i < kStepDepth - 1; ++i) fetch(begin + i);
  StepRow<T, NS> now, next;
  load(now, begin);
  f32x2 A2[NS / 2];
  {
    float f[NS];
    load_states<NS>(f, a.A + d * a.state + n0, ns, VEC);
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) A2[i] = pair(f[2 * i] * kLog2e, f[2 * i + 1] * kLog2e);
  }
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
  for (int64_t b = begin; b < end; ++b) {
    if (b + 1 < end) load(next, b + 1);
    T* out = static_cast<T*>(a.out) + b * a.out_stride + d;
    float* pool = pool_of(b);
    float h[NS];
    if (VEC) {
      fetch(b + kStepDepth - 1);
      copies_wait<kStepDepth - 1>();
#pragma unroll
      for (int i = 0; i < NS; i += 4) {
        const float4 v = ring[(b - begin) % kStepDepth][i / 4][tid];
        h[i] = v.x, h[i + 1] = v.y, h[i + 2] = v.z, h[i + 3] = v.w;
      }
    } else if (pool) {
      load_states<NS>(h, pool, ns, false);
    }
    if (pool) {
      const float x = to_f32(now.x), s = scan_step(to_f32(now.delta) + bias, a.softplus);
      const f32x2 s2 = both(s), sx2 = both(s * x);
      f32x2 y2 = 0;
#pragma unroll
      for (int i = 0; i < NS; i += 2) {
        const bool in = !VEC || i < ns;  // load_whole leaves this to its user
        const f32x2 bn = in ? pair_of(now.B[i / 4], i % 4) : 0;
        const f32x2 cn = in ? pair_of(now.C[i / 4], i % 4) : 0;
        const f32x2 v =
            fma2(decay2(A2[i / 2], s2), pair(h[i], h[i + 1]), mul2(sx2, bn));
        y2 = fma2(v, cn, y2);
        const float2 f = halves(v);
        h[i] = f.x, h[i + 1] = f.y;
      }
      const float2 yy = halves(y2);
      float y = yy.x + yy.y;
      if (mine) store_states<NS>(pool, h, ns, VEC);
#pragma unroll
      for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (mine && n0 == 0) {
        y = fmaf(skip, x, y);
        if (a.z) {
          const float z = to_f32(now.z);
          y *= z * sigmoid(z);
        }
        *out = from_f32<T>(y);
      }
    } else if (mine && n0 == 0) {
      *out = from_f32<T>(0.f);  // the whole block skips an empty row
    }
    now = next;
  }
}

// ---------------------------------------------------------------- host side

using Scan4 = Shape<4, 1, 2>;
using Scan8 = Shape<4, 2, 2>;
using Scan16 = Shape<4, 4, 1>;
using Scan32 = Shape<8, 4, 2>;
using Scan64 = Shape<8, 8, 2>;
#define SALT_SCAN_SHAPE(state, S, ...) \
  SALT_BY_STATE(state, S, Scan4, Scan8, Scan16, Scan32, Scan64, __VA_ARGS__)
int scan_channels(int32_t state) { return state <= 4 ? Scan4::kChannels : Scan16::kChannels; }

using Step4 = StepShape<4, 1>;
using Step8 = StepShape<8, 1>;
using Step16 = StepShape<8, 2>;
using Step32 = StepShape<16, 2>;
using Step64 = StepShape<16, 4>;
#define SALT_STEP_SHAPE(state, S, ...) \
  SALT_BY_STATE(state, S, Step4, Step8, Step16, Step32, Step64, __VA_ARGS__)

// One row of 16384 tokens x 2048 channels x 16 states: 406 us in 23 chunks, where 5 chunks take
// 530 us, and the first pass 0.55 of the second's time.  Both constants are those of 9 to 16 states in
// 16 bits; the rule takes them for all shapes, although the GPU holds about 20 of the blocks for up
// to 8 states an SM, 8 of those for 32 and 3 for 64 (4 rows of 2048 tokens x 2048 channels in bf16:
// 138, 146, 332 and 651 us at 4, 8, 32 and 64 states).
constexpr int kSlots = 148 * 5;      // blocks of 128 threads at 96 registers
constexpr float kFirstPass = 0.55f;  // its time, of the second pass's

template <typename T, class S, bool FULL>
cudaError_t scan_launch(const salt_selective_scan_args& a, const ScanSplit& sp, int blocks,
                        int chunks, int copy, bool svec, cudaStream_t st) {
  constexpr size_t shared = sizeof(ScanShared<T, S, FULL>);
  const auto kernel = copy == kCopy16  ? selective_scan_kernel<T, S, FULL, kCopy16>
                      : copy == kCopy4 ? selective_scan_kernel<T, S, FULL, kCopy4>
                                       : selective_scan_kernel<T, S, FULL, kCopyPlain>;
  if (shared > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(unsigned)((int64_t)a.batch * blocks * chunks), S::kThreads, shared, st>>>(a, sp, blocks,
                                                                                    svec);
  return cudaGetLastError();
}

ScanSplit split_of(const salt_selective_scan_args& a) {
  const int64_t blocks = (int64_t)a.batch * scan_blocks(a.dim, a.groups, scan_channels(a.state));
  return scan_split(blocks, kSlots, a.len, kFirstPass);
}

}  // namespace

size_t selective_scan_bytes(const salt_selective_scan_args& a) {
  const ScanSplit s = split_of(a);
  if (s.chunks == 1) return 0;
  return (size_t)a.batch * s.chunks * a.dim * (a.state + 1) * sizeof(float);
}

cudaError_t selective_scan_launch(const salt_selective_scan_args& a, void* ws, cudaStream_t st,
                                  int* launches) {
  if (a.batch == 0) return cudaSuccess;
  ScanSplit sp = split_of(a);
  if (sp.chunks > 1) {
    sp.state = static_cast<float*>(ws);
    sp.steps = sp.state + (size_t)a.batch * sp.chunks * a.dim * a.state;
  }
  const int blocks = scan_blocks(a.dim, a.groups, scan_channels(a.state));
  const size_t ts = type_size(a.type);
  // the widest copies that no row's start and end stand against
  auto fits = [&](int64_t bytes) {
    const int64_t whole = bytes / ts, few = std::min<int64_t>(bytes, 4 * ts);
    return (a.dim / a.groups) % (bytes == 16 ? (int)kVec : (int)whole) == 0 &&
           a.state % (few / ts) == 0 && packed_rows(a.x, bytes, ts, a.x_batch_stride, a.x_stride) &&
           packed_rows(a.delta, bytes, ts, a.delta_batch_stride, a.delta_stride) &&
           (!a.z || packed_rows(a.z, bytes, ts, a.z_batch_stride, a.z_stride)) &&
           packed_rows(a.out, bytes, ts, a.out_batch_stride, a.out_stride) &&
           packed_rows(a.B, few, ts, a.B_batch_stride, a.B_stride) &&
           packed_rows(a.C, few, ts, a.C_batch_stride, a.C_stride);
  };
  const int copy = fits(16) ? kCopy16 : fits(4) ? kCopy4 : kCopyPlain;
  const bool svec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.initial_state) &&
                    aligned16(a.final_state) && aligned16(a.checkpoints);
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, SALT_SCAN_SHAPE(a.state, S, {
    if (sp.chunks > 1) {
      e = scan_launch<T, S, false>(a, sp, blocks, sp.chunks - 1, copy, svec, st);
      ++*launches;
    }
    if (e == cudaSuccess) {
      e = scan_launch<T, S, true>(a, sp, blocks, sp.chunks, copy, svec, st);
      ++*launches;
    }
  }));
  return e;
}

cudaError_t selective_scan_step_launch(const salt_selective_scan_step_args& a, cudaStream_t st,
                                       int* launches) {
  if (a.batch == 0) return cudaSuccess;
  const int blocks = scan_blocks(a.dim, a.groups, kStepChannels);
  // A is loaded once for the rows that a block walks over (at most 32: a lane holds a row's slot)
  int rows = 1;
  while (rows < 8 && (int64_t)blocks * ((a.batch + 2 * rows - 1) / (2 * rows)) >= 148 * 8)
    rows *= 2;
  const int parts = (a.batch + rows - 1) / rows;
  const size_t ts = type_size(a.type);
  const bool vec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.pool) &&
                   pack_rows(a.B, 4, ts, a.B_stride) && pack_rows(a.C, 4, ts, a.C_stride);
  const unsigned grid = (unsigned)((int64_t)blocks * parts);
  SALT_WITH_TYPE(a.type, T, SALT_STEP_SHAPE(a.state, S, {
    if (vec)
      selective_scan_step_kernel<T, S, true>
          <<<grid, S::kThreads, 0, st>>>(a, blocks, rows);
    else
      selective_scan_step_kernel<T, S, false>
          <<<grid, S::kThreads, 0, st>>>(a, blocks, rows);
  }));
  ++*launches;
  return cudaGetLastError();
}

}  // namespace salt
