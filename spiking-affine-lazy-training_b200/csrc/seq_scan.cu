// Selective state space scan, whole rows and single tokens.
//
// Per token and channel the recurrence costs one exponential and four multiply-adds for each
// state, against one read of x, delta and z and one write of out for all of them: what bounds the
// kernel is the exponentials (16 a cycle and SM), not memory.
#include <algorithm>

#include "seq_scan.cuh"

namespace salt {

namespace {

// LPC lanes hold a channel's states, NS each.
template <int NS_, int LPC_>
struct Shape {
  static constexpr int NS = NS_, LPC = LPC_;
  static constexpr int kThreads = kScanChannels * LPC;
  static constexpr int kTile = kThreads / (kScanChannels / kVec);  // tokens: one pack a thread
  static constexpr int kStates = NS * LPC;
  static constexpr int kYPitch = kScanChannels + 8;  // 4 tokens x 8 channels on 32 banks
};

template <class S>
struct ScanShared {
  float2 step[S::kTile][kScanChannels];  // s and s * x
  float y[S::kTile][S::kYPitch];
  float B[S::kTile][S::kStates], C[S::kTile][S::kStates];
};

// B or C of a tile into shared memory as float32, zero past `real` and past the last state.
template <typename T, class S>
__device__ __forceinline__ void stage_states(float (*to)[S::kStates], const T* from,
                                             int64_t stride, int state, int t0, int real) {
  for (int i = threadIdx.x; i < S::kTile * S::kStates; i += S::kThreads) {
    const int t = i / S::kStates, n = i % S::kStates;
    to[t][n] = (t0 + t < real && n < state) ? to_f32(from[(t0 + t) * stride + n]) : 0.f;
  }
}

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

template <typename T, class S>
__global__ void __launch_bounds__(S::kThreads)
selective_scan_kernel(salt_selective_scan_args a, ScanSplit sp, int blocks, bool vec, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC;
  __shared__ ScanShared<S> sm;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / (blocks * sp.chunks);
  const int rest = (int)(blockIdx.x - b * blocks * sp.chunks), c = rest / blocks;
  const ScanBlock cb = scan_block(rest - c * blocks, a.dim, a.groups, kScanChannels);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, end = min(begin + sp.chunk_len, a.len);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;  // the chunk with the last token

  // this thread's channel and states in the recurrence
  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  float A2[NS], h[NS];
  load_states<NS>(A2, a.A + d * a.state + n0, mine ? ns : 0, svec);
#pragma unroll
  for (int i = 0; i < NS; ++i) A2[i] *= kLog2e;
  if (sp.chunks > 1) {
    chunk_start<NS>(h, A2, sp, b, min(c, last), a.dim, d, a.state, n0, svec);
  } else {
    load_states<NS>(h, a.initial_state + (b * a.dim + d) * a.state + n0,
                    mine && a.initial_state ? ns : 0, svec);
  }

  // and its 8 channels of one token in loads and stores
  const int io_t = tid / (kScanChannels / kVec), io_c = tid % (kScanChannels / kVec) * kVec;
  const int io_d = cb.d0 + io_c, io_n = cb.n - io_c;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + io_d;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + io_d;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + io_d : nullptr;
  T* out = static_cast<T*>(a.out) + b * a.out_batch_stride + io_d;
  const T* B = static_cast<const T*>(a.B) + b * a.B_batch_stride + (int64_t)cb.group * a.state;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  float bias[kVec], skip[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    bias[k] = a.delta_bias && k < io_n ? a.delta_bias[io_d + k] : 0.f;
    skip[k] = a.D && k < io_n ? a.D[io_d + k] : 0.f;
  }

  for (int t0 = begin; t0 < end; t0 += S::kTile) {
    const int t = t0 + io_t;
    float xs[kVec], y[kVec];
    Pack<T, kVec> pz;
    if (t0 < real) {
      const int n = t < real ? io_n : 0;
      const Pack<T, kVec> px = load_pack<T, kVec>(x + t * a.x_stride, n, vec);
      const Pack<T, kVec> pd = load_pack<T, kVec>(delta + t * a.delta_stride, n, vec);
      if (z) pz = load_pack<T, kVec>(z + t * a.z_stride, n, vec);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        xs[k] = to_f32(px.v[k]);
        // past the last token s = 0: the state stays as it is
        const float s = t < real ? scan_step(to_f32(pd.v[k]) + bias[k], a.softplus) : 0.f;
        sm.step[io_t][io_c + k] = make_float2(s, s * xs[k]);
      }
      stage_states<T, S>(sm.B, B, a.B_stride, a.state, t0, min(real, end));
      stage_states<T, S>(sm.C, C, a.C_stride, a.state, t0, min(real, end));
      __syncthreads();
#pragma unroll 1
      for (int g = 0; g < S::kTile; g += 4) {
        if (a.checkpoints && mine && (t0 + g) % SALT_SCAN_CHECKPOINT == 0 && t0 + g < real) {
          const int64_t per = (a.len + SALT_SCAN_CHECKPOINT - 1) / SALT_SCAN_CHECKPOINT;
          store_states<NS>(a.checkpoints +
                               ((b * per + (t0 + g) / SALT_SCAN_CHECKPOINT) * a.dim + d) * a.state +
                               n0,
                           h, ns, svec);
        }
        float yq[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 st = sm.step[g + q][ch];
          yq[q] = 0.f;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            h[i] = fmaf(exp2_fast(A2[i] * st.x), h[i], st.y * sm.B[g + q][n0 + i]);
            yq[q] = fmaf(h[i], sm.C[g + q][n0 + i], yq[q]);
          }
        }
        int first = 0;
        lane_sums<4, 1, LPC>(yq, tid, first);
#pragma unroll
        for (int q = 0; q < 4 / LPC; ++q) sm.y[g + first + q][ch] = yq[q];
      }
      __syncthreads();
    }
    if (t < end) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        y[k] = 0.f;
        if (t < real) {
          y[k] = fmaf(skip[k], xs[k], sm.y[io_t][io_c + k]);
          if (z) {
            const float v = to_f32(pz.v[k]);
            y[k] *= v * sigmoid(v);
          }
        }
      }
      store_pack<T, kVec>(out + t * a.out_stride, y, io_n, vec);
    }
  }
  if (c == last && mine && a.final_state)
    store_states<NS>(a.final_state + (b * a.dim + d) * a.state + n0, h, ns, svec);
}

// The first pass over a split row: chunk c's state from zero (chunk 0's from the initial state)
// into place c + 1, and the sum of its steps.  The last chunk has no successor and is not run.
template <typename T, class S>
__global__ void __launch_bounds__(S::kThreads)
scan_state_kernel(salt_selective_scan_args a, ScanSplit sp, int blocks, bool vec, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC;
  __shared__ float2 step[S::kTile][kScanChannels];
  __shared__ float sB[S::kTile][S::kStates];
  const int tid = threadIdx.x, run = sp.chunks - 1;
  const int64_t b = blockIdx.x / (blocks * run);
  const int rest = (int)(blockIdx.x - b * blocks * run), c = rest / blocks;
  const ScanBlock cb = scan_block(rest - c * blocks, a.dim, a.groups, kScanChannels);
  const int begin = c * sp.chunk_len;
  const int real = min(row_tokens(a.n_real, (int)b, a.len), begin + sp.chunk_len);
  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  float A2[NS], h[NS], sum = 0.f;
  load_states<NS>(A2, a.A + d * a.state + n0, mine ? ns : 0, svec);
#pragma unroll
  for (int i = 0; i < NS; ++i) A2[i] *= kLog2e;
  const int64_t at = ((b * sp.chunks + c) * a.dim + d) * a.state + n0;
  load_states<NS>(h, a.initial_state + (b * a.dim + d) * a.state + n0,
                  c == 0 && mine && a.initial_state ? ns : 0, svec);
  if (c == 0 && mine) store_states<NS>(sp.state + at, h, ns, svec);
  const int io_t = tid / (kScanChannels / kVec), io_c = tid % (kScanChannels / kVec) * kVec;
  const int io_d = cb.d0 + io_c, io_n = cb.n - io_c;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + io_d;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + io_d;
  const T* B = static_cast<const T*>(a.B) + b * a.B_batch_stride + (int64_t)cb.group * a.state;
  float bias[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    bias[k] = a.delta_bias && k < io_n ? a.delta_bias[io_d + k] : 0.f;
  for (int t0 = begin; t0 < real; t0 += S::kTile) {
    const int t = t0 + io_t, n = t < real ? io_n : 0;
    const Pack<T, kVec> px = load_pack<T, kVec>(x + t * a.x_stride, n, vec);
    const Pack<T, kVec> pd = load_pack<T, kVec>(delta + t * a.delta_stride, n, vec);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const float s = t < real ? scan_step(to_f32(pd.v[k]) + bias[k], a.softplus) : 0.f;
      step[io_t][io_c + k] = make_float2(s, s * to_f32(px.v[k]));
    }
    stage_states<T, S>(sB, B, a.B_stride, a.state, t0, real);
    __syncthreads();
#pragma unroll 4
    for (int q = 0; q < S::kTile; ++q) {
      const float2 st = step[q][ch];
      sum += st.x;
#pragma unroll
      for (int i = 0; i < NS; ++i) h[i] = fmaf(exp2_fast(A2[i] * st.x), h[i], st.y * sB[q][n0 + i]);
    }
  }
  if (!mine) return;
  store_states<NS>(sp.state + at + (int64_t)a.dim * a.state, h, ns, svec);
  if (n0 == 0) sp.steps[(b * sp.chunks + c) * a.dim + d] = sum;
}

// ---------------------------------------------------------------- single tokens

template <typename T, class S>
__global__ void __launch_bounds__(S::kThreads)
selective_scan_step_kernel(salt_selective_scan_step_args a, int blocks, int rows, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC;
  const int tid = threadIdx.x, part = blockIdx.x / blocks;
  const ScanBlock cb = scan_block(blockIdx.x - part * blocks, a.dim, a.groups, kScanChannels);
  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  float A2[NS];
  load_states<NS>(A2, a.A + d * a.state + n0, ns, svec);
#pragma unroll
  for (int i = 0; i < NS; ++i) A2[i] *= kLog2e;
  const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
  for (int64_t b = (int64_t)part * rows; b < min((int64_t)a.batch, (int64_t)(part + 1) * rows);
       ++b) {
    const int64_t slot = a.slots ? a.slots[b] : b;
    T* out = static_cast<T*>(a.out) + b * a.out_stride + d;
    if (slot < 0 || slot >= a.n_slots) {
      if (mine && n0 == 0) *out = from_f32<T>(0.f);
      continue;  // the whole block
    }
    float* pool = a.pool + (slot * a.dim + d) * a.state + n0;
    float h[NS];
    load_states<NS>(h, pool, ns, svec);
    const float x = to_f32(static_cast<const T*>(a.x)[b * a.x_stride + d]);
    const float s =
        scan_step(to_f32(static_cast<const T*>(a.delta)[b * a.delta_stride + d]) + bias, a.softplus);
    const T* B = static_cast<const T*>(a.B) + b * a.B_stride + (int64_t)cb.group * a.state + n0;
    const T* C = static_cast<const T*>(a.C) + b * a.C_stride + (int64_t)cb.group * a.state + n0;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const float bn = i < ns ? to_f32(B[i]) : 0.f, cn = i < ns ? to_f32(C[i]) : 0.f;
      h[i] = fmaf(exp2_fast(A2[i] * s), h[i], s * x * bn);
      y = fmaf(h[i], cn, y);
    }
    if (mine) store_states<NS>(pool, h, ns, svec);
#pragma unroll
    for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (mine && n0 == 0) {
      y = fmaf(skip, x, y);
      if (a.z) {
        const float z = to_f32(static_cast<const T*>(a.z)[b * a.z_stride + d]);
        y *= z * sigmoid(z);
      }
      *out = from_f32<T>(y);
    }
  }
}

// ---------------------------------------------------------------- host side

#define SALT_SCAN_SHAPE(state, S, ...)  \
  do {                                  \
    if ((state) <= 4) {                 \
      using S = Shape<4, 1>;            \
      __VA_ARGS__;                      \
    } else if ((state) <= 8) {          \
      using S = Shape<4, 2>;            \
      __VA_ARGS__;                      \
    } else if ((state) <= 16) {         \
      using S = Shape<4, 4>;            \
      __VA_ARGS__;                      \
    } else if ((state) <= 32) {         \
      using S = Shape<8, 4>;            \
      __VA_ARGS__;                      \
    } else {                            \
      using S = Shape<16, 4>;           \
      __VA_ARGS__;                      \
    }                                   \
  } while (0)

constexpr int kFillBlocks = 148 * 2;

ScanSplit scan_split(const salt_selective_scan_args& a) {
  ScanSplit s{1, std::max(a.len, 1), nullptr, nullptr};
  const int64_t blocks = (int64_t)a.batch * scan_blocks(a.dim, a.groups, kScanChannels);
  if (blocks >= kFillBlocks || blocks == 0) return s;
  const int want = (int)((2 * kFillBlocks + blocks - 1) / blocks);
  const int each = std::max(128, (a.len + want - 1) / want);
  s.chunk_len = (each + 31) / 32 * 32;  // whole tiles and checkpoints of every shape
  s.chunks = std::max(1, (a.len + s.chunk_len - 1) / s.chunk_len);
  if (s.chunks == 1) s.chunk_len = std::max(a.len, 1);
  return s;
}

}  // namespace

size_t selective_scan_bytes(const salt_selective_scan_args& a) {
  const ScanSplit s = scan_split(a);
  if (s.chunks == 1) return 0;
  return (size_t)a.batch * s.chunks * a.dim * (a.state + 1) * sizeof(float);
}

cudaError_t selective_scan_launch(const salt_selective_scan_args& a, void* ws, cudaStream_t st,
                                  int* launches) {
  if (a.batch == 0) return cudaSuccess;
  ScanSplit sp = scan_split(a);
  if (sp.chunks > 1) {
    sp.state = static_cast<float*>(ws);
    sp.steps = sp.state + (size_t)a.batch * sp.chunks * a.dim * a.state;
  }
  const int blocks = scan_blocks(a.dim, a.groups, kScanChannels);
  const size_t ts = type_size(a.type);
  const bool vec = (a.groups == 1 || (a.dim / a.groups * ts) % 16 == 0) &&
                   vec_rows(a.x, ts, a.x_batch_stride, a.x_stride) &&
                   vec_rows(a.delta, ts, a.delta_batch_stride, a.delta_stride) &&
                   vec_rows(a.z, ts, a.z_batch_stride, a.z_stride) &&
                   vec_rows(a.out, ts, a.out_batch_stride, a.out_stride);
  const bool svec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.initial_state) &&
                    aligned16(a.final_state) && aligned16(a.checkpoints);
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, SALT_SCAN_SHAPE(a.state, S, {
    if (sp.chunks > 1) {
      scan_state_kernel<T, S><<<(unsigned)((int64_t)a.batch * blocks * (sp.chunks - 1)),
                                S::kThreads, 0, st>>>(a, sp, blocks, vec, svec);
      ++*launches;
      e = cudaGetLastError();
    }
    if (e == cudaSuccess) {
      selective_scan_kernel<T, S><<<(unsigned)((int64_t)a.batch * blocks * sp.chunks),
                                    S::kThreads, 0, st>>>(a, sp, blocks, vec, svec);
      ++*launches;
      e = cudaGetLastError();
    }
  }));
  return e;
}

cudaError_t selective_scan_step_launch(const salt_selective_scan_step_args& a, cudaStream_t st,
                                       int* launches) {
  if (a.batch == 0) return cudaSuccess;
  const int blocks = scan_blocks(a.dim, a.groups, kScanChannels);
  // A's rows are loaded once for the token rows that a block walks over
  int rows = 1;
  while (rows < 8 && (int64_t)blocks * ((a.batch + 2 * rows - 1) / (2 * rows)) >= 148 * 8) rows *= 2;
  const int parts = (a.batch + rows - 1) / rows;
  const bool svec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.pool);
  SALT_WITH_TYPE(a.type, T, SALT_SCAN_SHAPE(a.state, S, {
    selective_scan_step_kernel<T, S>
        <<<(unsigned)((int64_t)blocks * parts), S::kThreads, 0, st>>>(a, blocks, rows, svec);
  }));
  ++*launches;
  return cudaGetLastError();
}

}  // namespace salt
