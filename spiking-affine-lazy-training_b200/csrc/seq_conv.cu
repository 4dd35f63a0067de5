// Short causal convolution over the tokens of each channel, its single-token form and its gradient.
//
// All three are bound by memory: an element is read and written once for 2 * width + 5 operations
// (about 4 times that backward).  A thread takes a few neighbouring channels through a run of
// tokens, with the last width - 1 inputs in registers, so that an input is loaded once for all its
// taps; only the width - 1 tokens in front of a run are read twice.
#include <algorithm>

#include "sequence.cuh"

namespace salt {

namespace {

// weight[d][k] of channels d0 .. d0 + N; tap W - 1 is the newest input's.
template <typename T, int N, int W>
__device__ __forceinline__ void load_taps(float (&w)[N][W], const void* weight, int d0, int n,
                                          bool w_f32) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < W; ++k)
      w[i][k] = i < n ? weight_at<T>(weight, (int64_t)(d0 + i) * W + k, w_f32) : 0.f;
}

// Token s of a channel, for s < 0 from the initial state (token s is its entry W - 1 + s), zero
// where there is none.
template <typename T, int W>
__device__ __forceinline__ float token_at(const T* x, int64_t stride, const T* init, int d, int s) {
  if (s >= 0) return to_f32(x[s * stride + d]);
  return init ? to_f32(init[(int64_t)d * (W - 1) + W - 1 + s]) : 0.f;
}

// ---------------------------------------------------------------- whole rows

// Thread = 8 channels x `run` tokens; threads count channel packs fastest, then runs, then rows.
template <typename T, int W>
__global__ void __launch_bounds__(128)
causal_conv_kernel(salt_causal_conv_args a, int packs, int runs, int run, bool vec, bool w_f32) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per_row = (int64_t)packs * runs;
  if (id >= per_row * a.batch) return;
  const int b = (int)(id / per_row);
  const int rest = (int)(id - b * per_row);
  const int c = rest / packs, d0 = (rest - c * packs) * kVec;
  const int n = a.dim - d0;
  const int real = row_tokens(a.n_real, b, a.len);
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride;
  const int64_t state0 = (int64_t)b * a.dim * (W - 1);
  const T* init = a.initial_state ? static_cast<const T*>(a.initial_state) + state0 : nullptr;
  T* out = static_cast<T*>(a.out) + b * a.out_batch_stride;
  const int t0 = c * run, t1 = min(t0 + run, a.len);
  float w[kVec][W], bias[kVec], win[W][kVec];  // win[W - 1] is the newest input
  load_taps<T, kVec, W>(w, a.weight, d0, n, w_f32);
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    bias[k] = a.bias && k < n ? weight_at<T>(a.bias, d0 + k, w_f32) : 0.f;
#pragma unroll
  for (int j = 1; j < W; ++j) {
    const int s = t0 + j - W;
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      win[j][k] = k < n && s < real ? token_at<T, W>(x, a.x_stride, init, d0 + k, s) : 0.f;
  }
  // Reads its own channels of initial_state, here and above, before it writes: they may be one.
  if (c == 0 && a.final_state) {
    T* fin = static_cast<T*>(a.final_state) + state0;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      if (k >= n) break;
      float f[W];
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        f[j] = token_at<T, W>(x, a.x_stride, init, d0 + k, real - (W - 1) + j);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) fin[(int64_t)(d0 + k) * (W - 1) + j] = from_f32<T>(f[j]);
    }
  }
#pragma unroll 4
  for (int t = t0; t < t1; ++t) {
    const Pack<T, kVec> p = load_pack<T, kVec>(x + t * a.x_stride + d0, t < real ? n : 0, vec);
    float y[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j][k] = win[j + 1][k];
      win[W - 1][k] = to_f32(p.v[k]);
      float s = bias[k];
#pragma unroll
      for (int j = 0; j < W; ++j) s = fmaf(w[k][j], win[j][k], s);
      if (a.silu) s *= sigmoid(s);
      y[k] = t < real ? s : 0.f;
    }
    store_pack<T, kVec>(out + t * a.out_stride + d0, y, n, vec);
  }
}

// ---------------------------------------------------------------- single tokens

template <typename T, int W>
__global__ void __launch_bounds__(128)
causal_conv_step_kernel(salt_causal_conv_step_args a, int64_t total, bool w_f32) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= total) return;
  const int b = (int)(id / a.dim), d = (int)(id - (int64_t)b * a.dim);
  const int64_t slot = a.slots ? a.slots[b] : b;
  T* out = static_cast<T*>(a.out) + b * a.out_stride + d;
  if (slot < 0 || slot >= a.n_slots) {
    *out = from_f32<T>(0.f);
    return;
  }
  T* state = static_cast<T*>(a.state) + (slot * a.dim + d) * (W - 1);
  T in[W];
  in[W - 1] = static_cast<const T*>(a.x)[b * a.x_stride + d];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) in[j] = state[j];
  float s = a.bias ? weight_at<T>(a.bias, d, w_f32) : 0.f;
#pragma unroll
  for (int j = 0; j < W; ++j)
    s = fmaf(weight_at<T>(a.weight, (int64_t)d * W + j, w_f32), to_f32(in[j]), s);
  if (a.silu) s *= sigmoid(s);
  *out = from_f32<T>(s);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) state[j] = in[j + 1];
}

// ---------------------------------------------------------------- gradient

constexpr int kBackVec = 4;   // channels of a thread: 8 would need 150 registers
constexpr int kBackRuns = 8;  // runs of tokens in a block, one per warp
constexpr int kBackLanes = 32;

// A warp takes 128 channels through `run` tokens, a block 8 such runs one after the other in the
// row.  g[t] = dy[t] * act'(p[t]) for the run and the width - 1 tokens behind it gives
// dx[s] = sum_k w[k] g[s + width - 1 - k]; the weight's gradient takes the run's own tokens only.
template <typename T, int W>
__global__ void __launch_bounds__(kBackLanes * kBackRuns)
causal_conv_backward_kernel(salt_causal_conv_backward_args a, int packs, int chunks, int run,
                            bool vec, bool w_f32, float* parts) {
  __shared__ float red[kBackRuns][kBackLanes * kBackVec];
  constexpr int V = kBackVec;
  const int pack = blockIdx.x % packs, part_id = blockIdx.x / packs;  // part_id = b * chunks + chunk
  const int b = part_id / chunks, chunk = part_id - b * chunks;
  const int lane = threadIdx.x, d0 = (pack * kBackLanes + lane) * V, n = a.dim - d0;
  const int t0 = (chunk * kBackRuns + threadIdx.y) * run, t1 = min(t0 + run, a.len);
  const int real = row_tokens(a.n_real, b, a.len);
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride;
  T* dx = static_cast<T*>(a.dx) + b * a.dx_batch_stride;
  const int64_t state0 = (int64_t)b * a.dim * (W - 1);
  const T* init = a.initial_state ? static_cast<const T*>(a.initial_state) + state0 : nullptr;
  float w[V][W], bias[V], win[W][V], g[W][V], dw[V][W], db[V];  // [W - 1] is the newest token
  load_taps<T, V, W>(w, a.weight, d0, n, w_f32);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    bias[k] = a.bias && k < n ? weight_at<T>(a.bias, d0 + k, w_f32) : 0.f;
    db[k] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[k][j] = win[j][k] = g[j][k] = 0.f;
  }
  if (n > 0 && (t0 < t1 || t0 == 0)) {  // a row without tokens has an initial state's gradient
#pragma unroll
    for (int j = 1; j < W; ++j) {
      const int s = t0 + j - W;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k < n && s < real) win[j][k] = token_at<T, W>(x, a.x_stride, init, d0 + k, s);
    }
#pragma unroll 4
    for (int t = t0; t < t1 + W - 1; ++t) {
      const int m = t < real ? n : 0;
      const Pack<T, V> px = load_pack<T, V>(x + t * a.x_stride + d0, m, vec);
      const Pack<T, V> pd = load_pack<T, V>(dy + t * a.dy_stride + d0, m, vec);
      const int s = t - (W - 1);
      float out[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          win[j][k] = win[j + 1][k];
          g[j][k] = g[j + 1][k];
        }
        win[W - 1][k] = to_f32(px.v[k]);
        float gt = to_f32(pd.v[k]);
        if (a.silu) {
          float p = bias[k];
#pragma unroll
          for (int j = 0; j < W; ++j) p = fmaf(w[k][j], win[j][k], p);
          gt *= silu_slope(p, sigmoid(p));
        }
        g[W - 1][k] = t < real ? gt : 0.f;
        if (t < t1) {
          db[k] += g[W - 1][k];
#pragma unroll
          for (int j = 0; j < W; ++j) dw[k][j] = fmaf(g[W - 1][k], win[j][k], dw[k][j]);
        }
        // token s met tap j at token s + W - 1 - j = t - j
        out[k] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) out[k] = fmaf(w[k][j], g[W - 1 - j][k], out[k]);
        if (s >= real) out[k] = 0.f;
      }
      if (s >= t0) {
        store_pack<T, V>(dx + s * a.dx_stride + d0, out, n, vec);
      } else if (t0 == 0 && a.dinitial) {
        T* di = static_cast<T*>(a.dinitial) + state0;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k < n) di[(int64_t)(d0 + k) * (W - 1) + t] = from_f32<T>(out[k]);
      }
    }
  }
  // the block's sum over its runs, in order, one tap (and the bias) after the other
  float* part = parts + (int64_t)part_id * a.dim * (W + 1);
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) red[threadIdx.y][lane * V + k] = j < W ? dw[k][j % W] : db[k];
    __syncthreads();
    const int i = threadIdx.y * kBackLanes + lane;
    const int d = pack * kBackLanes * V + i;
    if (i < kBackLanes * V && d < a.dim) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kBackRuns; ++r) s += red[r][i];
      part[(int64_t)j * a.dim + d] = s;
    }
  }
}

// Adds the partial sums (parts, width + 1, dim) into dweight (dim, width) and dbias (dim).
__global__ void conv_weight_gradient(const float* __restrict__ parts, int64_t n_parts, int dim,
                                     int width, float* dweight, float* dbias) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, n = (int64_t)dim * (width + 1);
  if (i >= n) return;
  const int j = (int)(i / dim), d = (int)(i - (int64_t)j * dim);
  float s = 0.f;
  for (int64_t p = 0; p < n_parts; ++p) s += parts[p * n + i];
  if (j < width)
    dweight[(int64_t)d * width + j] = s;
  else if (dbias)
    dbias[d] = s;
}

#define SALT_WITH_WIDTH(width, ...)                  \
  do {                                               \
    switch (width) {                                 \
      case 1: { constexpr int W = 1; __VA_ARGS__; break; } \
      case 2: { constexpr int W = 2; __VA_ARGS__; break; } \
      case 3: { constexpr int W = 3; __VA_ARGS__; break; } \
      case 4: { constexpr int W = 4; __VA_ARGS__; break; } \
      case 5: { constexpr int W = 5; __VA_ARGS__; break; } \
      case 6: { constexpr int W = 6; __VA_ARGS__; break; } \
      case 7: { constexpr int W = 7; __VA_ARGS__; break; } \
      default: { constexpr int W = 8; __VA_ARGS__; break; } \
    }                                                \
  } while (0)

// Tokens of a thread's run: long enough that the tokens read twice are few, short enough that the
// threads fill the GPU.
int conv_run(int64_t packs, int32_t batch, int32_t len) {
  int run = 32;
  while (run > 4 && packs * batch * ((len + run - 1) / run) < 148 * 1024) run >>= 1;
  return run;
}

struct ConvBackPlan {
  int run, chunks, packs;
};
ConvBackPlan conv_back_plan(const salt_causal_conv_backward_args& a) {
  ConvBackPlan p;
  p.packs = (a.dim + kBackLanes * kBackVec - 1) / (kBackLanes * kBackVec);
  p.run = 64;
  while (p.run > 8 && (int64_t)p.packs * a.batch *
                              ((a.len + p.run * kBackRuns - 1) / (p.run * kBackRuns)) <
                          148 * 2)
    p.run >>= 1;
  p.chunks = std::max(1, (a.len + p.run * kBackRuns - 1) / (p.run * kBackRuns));
  return p;
}

}  // namespace

cudaError_t causal_conv_launch(const salt_causal_conv_args& a, cudaStream_t st, int* launches) {
  if (a.batch == 0) return cudaSuccess;
  const int packs = (a.dim + kVec - 1) / kVec;
  const int run = conv_run(packs, a.batch, a.len);
  const int runs = std::max(1, (a.len + run - 1) / run);  // a row without tokens has a final state
  const size_t ts = type_size(a.type);
  const bool vec = vec_rows(a.x, ts, a.x_batch_stride, a.x_stride) &&
                   vec_rows(a.out, ts, a.out_batch_stride, a.out_stride);
  const int64_t threads = (int64_t)packs * runs * a.batch;
  const unsigned blocks = (unsigned)((threads + 127) / 128);
  const bool w_f32 = a.weight_type == SALT_F32;
  SALT_WITH_TYPE(a.type, T, SALT_WITH_WIDTH(a.width, {
    causal_conv_kernel<T, W><<<blocks, 128, 0, st>>>(a, packs, runs, run, vec, w_f32);
  }));
  ++*launches;
  return cudaGetLastError();
}

cudaError_t causal_conv_step_launch(const salt_causal_conv_step_args& a, cudaStream_t st,
                                    int* launches) {
  if (a.batch == 0) return cudaSuccess;
  const int64_t total = (int64_t)a.batch * a.dim;
  const unsigned blocks = (unsigned)((total + 127) / 128);
  const bool w_f32 = a.weight_type == SALT_F32;
  SALT_WITH_TYPE(a.type, T, SALT_WITH_WIDTH(a.width, {
    causal_conv_step_kernel<T, W><<<blocks, 128, 0, st>>>(a, total, w_f32);
  }));
  ++*launches;
  return cudaGetLastError();
}

size_t causal_conv_backward_bytes(const salt_causal_conv_backward_args& a) {
  const ConvBackPlan p = conv_back_plan(a);
  return (size_t)p.chunks * a.batch * a.dim * (a.width + 1) * sizeof(float);
}

cudaError_t causal_conv_backward_launch(const salt_causal_conv_backward_args& a, void* ws,
                                        cudaStream_t st, int* launches) {
  const ConvBackPlan p = conv_back_plan(a);
  const size_t ts = type_size(a.type);
  const bool vec = vec_rows(a.x, ts, a.x_batch_stride, a.x_stride) &&
                   vec_rows(a.dy, ts, a.dy_batch_stride, a.dy_stride) &&
                   vec_rows(a.dx, ts, a.dx_batch_stride, a.dx_stride);
  const bool w_f32 = a.weight_type == SALT_F32;
  float* parts = static_cast<float*>(ws);
  if (a.batch > 0) {
    const unsigned blocks = (unsigned)((int64_t)p.packs * p.chunks * a.batch);
    const dim3 block(kBackLanes, kBackRuns);
    SALT_WITH_TYPE(a.type, T, SALT_WITH_WIDTH(a.width, {
      causal_conv_backward_kernel<T, W><<<blocks, block, 0, st>>>(a, p.packs, p.chunks, p.run, vec,
                                                               w_f32, parts);
    }));
    ++*launches;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  const int64_t n = (int64_t)a.dim * (a.width + 1);
  conv_weight_gradient<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(
      parts, (int64_t)p.chunks * a.batch, a.dim, a.width, a.dweight, a.dbias);
  ++*launches;
  return cudaGetLastError();
}

}  // namespace salt
