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

// Values of V channels as pairs; one channel has a zero beside it.
template <int V>
__device__ __forceinline__ void to_pairs(f32x2 (&p)[(V + 1) / 2], const float* f) {
#pragma unroll
  for (int k = 0; k < (V + 1) / 2; ++k) p[k] = pair(f[2 * k], V == 1 ? 0.f : f[2 * k + (V > 1)]);
}

// weight[d][j] of channels d0 .. d0 + V, of which n (V or none) are there, as w[j]; tap W - 1 is
// the newest input's.  The V W values lie together: W packs.
template <typename T, int V, int W>
__device__ __forceinline__ void load_taps(f32x2 (&w)[W][(V + 1) / 2], f32x2 (&bias)[(V + 1) / 2],
                                          const void* weight, const void* from, int d0, int n,
                                          bool w_f32, bool vec) {
  float f[W][V];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float g[V];
    load_weights<T, V>(g, weight, (int64_t)d0 * W + i * V, n * W - i * V, w_f32, vec);
#pragma unroll
    for (int k = 0; k < V; ++k) f[(i * V + k) % W][(i * V + k) / W] = g[k];
  }
#pragma unroll
  for (int j = 0; j < W; ++j) to_pairs<V>(w[j], f[j]);
  float g[V];
#pragma unroll
  for (int k = 0; k < V; ++k) g[k] = from && k < n ? weight_at<T>(from, d0 + k, w_f32) : 0.f;
  to_pairs<V>(bias, g);
}

// Token s of N neighbouring channels of a row, the first at x + s * stride and init: for s < 0 from
// the initial state (token s is its entry W - 1 + s), zero where there is none and past `real`.
template <typename T, int N, int W>
__device__ __forceinline__ void load_token(float (&f)[N], const T* x, int64_t stride, const T* init,
                                           int s, int real, int n, bool vec) {
  if (s >= 0 || !init) {
    const Pack<T, N> p = load_pack<T, N>(x + s * stride, s >= 0 && s < real ? n : 0, vec);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = to_f32(p.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = k < n ? to_f32(init[k * (W - 1) + W - 1 + s]) : 0.f;
  }
}

// ---------------------------------------------------------------- whole rows

// For 4 ragged rows of 4096 tokens x 4096 channels in bf16: 45 us, 4.5 TB/s or 69 % of the measured
// copy rate.  8 channels a thread take twice the registers (50.7 us); loads of 8 tokens together
// 50.2 us, of 2 60.7 us (at 8 channels).
constexpr int kAhead = 4;   // tokens whose loads go out together
constexpr int kRowVec = 4;  // channels of a thread

// Thread = V channels x `run` tokens; threads count channel packs fastest, then runs, then rows.
template <typename T, int V, int W>
__global__ void __launch_bounds__(128)
causal_conv_kernel(salt_causal_conv_args a, int packs, int runs, int run, bool w_f32, bool w_vec) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per_row = (int64_t)packs * runs;
  if (id >= per_row * a.batch) return;
  const int b = (int)(id / per_row);
  const uint32_t rest = (uint32_t)(id - b * per_row);  // a row has under 2^32 threads
  const int c = rest / (uint32_t)packs, d0 = (int)(rest - c * (uint32_t)packs) * V;
  const int n = a.dim - d0;  // at least V: V divides dim
  const int real = row_tokens(a.n_real, b, a.len);
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + d0;
  const int64_t state0 = ((int64_t)b * a.dim + d0) * (W - 1);
  const T* init = a.initial_state ? static_cast<const T*>(a.initial_state) + state0 : nullptr;
  T* out = static_cast<T*>(a.out) + b * a.out_batch_stride + d0;
  const int t0 = c * run, t1 = min(t0 + run, a.len), stop = min(t1, real);
  constexpr int H = (V + 1) / 2;
  f32x2 win[W][H];  // win[W - 1] is the newest input
  if (t0 < stop) {
#pragma unroll
    for (int j = 1; j < W; ++j) {
      float f[V];
      load_token<T, V, W>(f, x, a.x_stride, init, t0 + j - W, real, n, true);
      to_pairs<V>(win[j], f);
    }
  }
  // initial_state and final_state may be one array: of a row's threads this one alone reads its
  // channels of the first, here and above, before it writes the second.
  if (c == 0 && a.final_state && W > 1) {
    T* fin = static_cast<T*>(a.final_state) + state0;
    float f[W][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      load_token<T, V, W>(f[j], x, a.x_stride, init, real - (W - 1) + j, real, n, true);
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int j = 0; j < W - 1; ++j) fin[k * (W - 1) + j] = from_f32<T>(f[j][k]);
  }
  int t = t0;
  if (t0 < stop) {
    f32x2 w[W][H], bias[H];
    load_taps<T, V, W>(w, bias, a.weight, a.bias, d0, n, w_f32, w_vec);
    // The loads of kAhead tokens go out together; behind the first store the compiler would have to
    // keep them in order.
    for (; t < stop; t += kAhead) {
      Pack<T, V> p[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        p[q] = load_whole<T, V>(x, min(t + q, stop - 1) * a.x_stride, INT64_MAX);
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        float y[V + 1];
#pragma unroll
        for (int k = 0; k < H; ++k) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j) win[j][k] = win[j + 1][k];
          win[W - 1][k] = pair_in(p[q], k);
          f32x2 s = bias[k];
#pragma unroll
          for (int j = 0; j < W; ++j) s = fma2(w[j][k], win[j][k], s);
          if (a.silu) s = mul2(s, sigmoid2(s));
          const float2 f = halves(s);
          y[2 * k] = f.x, y[2 * k + 1] = f.y;
        }
        if (t + q < stop) store_pack<T, V>(out + (t + q) * a.out_stride, y, V, true);
      }
    }
    t = stop;
  }
  const float zero[V] = {};
#pragma unroll 4
  for (; t < t1; ++t) store_pack<T, V>(out + t * a.out_stride, zero, V, true);
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

// Forward and backward of 8 rows of 2048 tokens x 2048 channels in bf16 take 123 us, 2.7 TB/s or
// 42 % of the copy rate: 37 us forward, 80 us backward, 6 us the sum of the parts.  The backward
// kernel holds 16 warps on an SM (128 registers for weights, inputs, gradients and their sums) and
// issues in every second cycle.  Channels of a thread: 2 154 us, 8 276 us (before the arithmetic in
// pairs); loads of 2 tokens together 154 us, of 8 130 us.
constexpr int kBackVec = 4;    // channels of a thread
constexpr int kBackAhead = 4;  // tokens whose loads go out together
constexpr int kBackRuns = 8;  // runs of tokens in a block, one per warp
constexpr int kBackLanes = 32;

// A warp takes 32 V channels through `run` tokens, a block 8 such runs one after the other in the
// row.  g[t] = dy[t] * act'(p[t]) for the run and the width - 1 tokens behind it gives
// dx[s] = sum_k w[k] g[s + width - 1 - k]; the weight's gradient takes the run's own tokens only.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kBackLanes * kBackRuns, W <= 4 ? 2 : 1)
causal_conv_backward_kernel(salt_causal_conv_backward_args a, int packs, int chunks, int run,
                            bool w_f32, bool w_vec, float* parts) {
  __shared__ float red[kBackRuns][kBackLanes * V];
  // part_id = b * chunks + chunk
  const int pack = blockIdx.x % packs, part_id = blockIdx.x / packs;
  const int b = part_id / chunks, chunk = part_id - b * chunks;
  const int lane = threadIdx.x, d0 = (pack * kBackLanes + lane) * V;
  const int n = d0 < a.dim ? V : 0;  // V divides dim
  const int t0 = (chunk * kBackRuns + threadIdx.y) * run, t1 = min(t0 + run, a.len);
  const int real = row_tokens(a.n_real, b, a.len);
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + d0;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + d0;
  T* dx = static_cast<T*>(a.dx) + b * a.dx_batch_stride + d0;
  const int64_t state0 = ((int64_t)b * a.dim + d0) * (W - 1);
  const T* init = a.initial_state ? static_cast<const T*>(a.initial_state) + state0 : nullptr;
  constexpr int H = (V + 1) / 2;
  // [W - 1] is the newest token
  f32x2 w[W][H], bias[H], win[W][H], g[W][H] = {}, dw[W][H] = {}, db[H] = {};
  if (n > 0 && (t0 < t1 || t0 == 0)) {  // a row without tokens has an initial state's gradient
    load_taps<T, V, W>(w, bias, a.weight, a.bias, d0, n, w_f32, w_vec);
#pragma unroll
    for (int j = 1; j < W; ++j) {
      float f[V];
      load_token<T, V, W>(f, x, a.x_stride, init, t0 + j - W, real, n, true);
      to_pairs<V>(win[j], f);
    }
    // without tokens there is nothing to load, and dinitial is 0
    for (int k = 0; a.len == 0 && a.dinitial && k < V * (W - 1); ++k)
      static_cast<T*>(a.dinitial)[state0 + k] = from_f32<T>(0.f);
    for (int tt = t0; a.len > 0 && tt < t1 + W - 1; tt += kBackAhead) {
      Pack<T, V> ax[kBackAhead], ad[kBackAhead];
#pragma unroll
      for (int q = 0; q < kBackAhead; ++q) {
        const int t = min(tt + q, max(real, 1) - 1);  // past the row's end its last token
        ax[q] = load_whole<T, V>(x, t * a.x_stride, INT64_MAX);
        ad[q] = load_whole<T, V>(dy, t * a.dy_stride, INT64_MAX);
      }
#pragma unroll
      for (int q = 0; q < kBackAhead; ++q) {
        const int t = tt + q, s = t - (W - 1);
        float out[V + 1];
#pragma unroll
        for (int k = 0; k < H; ++k) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j) {
            win[j][k] = win[j + 1][k];
            g[j][k] = g[j + 1][k];
          }
          win[W - 1][k] = t < real ? pair_in(ax[q], k) : 0;
          f32x2 gt = t < real ? pair_in(ad[q], k) : 0;
          if (a.silu) {
            f32x2 p = bias[k];
#pragma unroll
            for (int j = 0; j < W; ++j) p = fma2(w[j][k], win[j][k], p);
            gt = mul2(gt, silu_slope2(p, sigmoid2(p)));
          }
          g[W - 1][k] = gt;
          const f32x2 own = t < t1 ? gt : 0;
          db[k] = add2(db[k], own);
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][k] = fma2(own, win[j][k], dw[j][k]);
          // token s met tap j at token s + W - 1 - j = t - j
          f32x2 v = mul2(w[0][k], g[W - 1][k]);
#pragma unroll
          for (int j = 1; j < W; ++j) v = fma2(w[j][k], g[W - 1 - j][k], v);
          const float2 f = halves(s < real ? v : 0);
          out[2 * k] = f.x, out[2 * k + 1] = f.y;
        }
        // tokens behind the run (and, in the last round, behind its gradients) are another's
        if (s >= t0) {
          if (s < t1) store_pack<T, V>(dx + s * a.dx_stride, out, V, true);
        } else if (t0 == 0 && a.dinitial) {
          T* di = static_cast<T*>(a.dinitial) + state0;
#pragma unroll
          for (int k = 0; k < V; ++k) di[k * (W - 1) + t] = from_f32<T>(out[k]);
        }
      }
    }
  }
  // the block's sum over its runs, in order, one tap (and the bias) after the other
  float* part = parts + (int64_t)part_id * a.dim * (W + 1);
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float2 f = halves(j < W ? dw[j % W][k / 2] : db[k / 2]);
      red[threadIdx.y][lane * V + k] = k % 2 ? f.y : f.x;
    }
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
// threads fill the GPU.  No run is shorter than the width - 1 tokens in front of the next one, which
// would then reach into the initial state: a row's first run may be writing the final state there.
int conv_run(int64_t packs, int32_t batch, int32_t len, int32_t width) {
  const int least = width <= 5 ? 4 : 8;
  int run = 32;
  while (run > least && packs * batch * ((len + run - 1) / run) < 148 * 1024) run >>= 1;
  return run;
}

struct ConvBackPlan {
  int v, run, chunks, packs;
};
ConvBackPlan conv_back_plan(const salt_causal_conv_backward_args& a) {
  ConvBackPlan p;
  const size_t ts = type_size(a.type);
  const bool fits = a.dim % kBackVec == 0 &&
                    pack_rows(a.x, kBackVec, ts, a.x_batch_stride, a.x_stride) &&
                    pack_rows(a.dy, kBackVec, ts, a.dy_batch_stride, a.dy_stride) &&
                    pack_rows(a.dx, kBackVec, ts, a.dx_batch_stride, a.dx_stride);
  p.v = fits ? kBackVec : 1;
  p.packs = (a.dim + kBackLanes * p.v - 1) / (kBackLanes * p.v);
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
  const size_t ts = type_size(a.type);
  auto fits = [&](int v) {
    return a.dim % v == 0 && pack_rows(a.x, v, ts, a.x_batch_stride, a.x_stride) &&
           pack_rows(a.out, v, ts, a.out_batch_stride, a.out_stride);
  };
    const int v = fits(kRowVec) ? kRowVec : 1, packs = a.dim / v;
  const int run = conv_run(packs, a.batch, a.len, a.width);
  const int runs = std::max(1, (a.len + run - 1) / run);  // a row without tokens has a final state
  const int64_t threads = (int64_t)packs * runs * a.batch;
  const unsigned blocks = (unsigned)((threads + 127) / 128);
  const bool w_f32 = a.weight_type == SALT_F32;
  const bool w_vec = pack_rows(a.weight, v, w_f32 ? 4 : ts, 0);
  SALT_WITH_TYPE(a.type, T, SALT_WITH_WIDTH(a.width, {
    if (v == kRowVec)
      causal_conv_kernel<T, kRowVec, W><<<blocks, 128, 0, st>>>(a, packs, runs, run, w_f32, w_vec);
    else
      causal_conv_kernel<T, 1, W><<<blocks, 128, 0, st>>>(a, packs, runs, run, w_f32, w_vec);
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
  const bool w_f32 = a.weight_type == SALT_F32;
  const bool w_vec = pack_rows(a.weight, p.v, w_f32 ? 4 : type_size(a.type), 0);
  float* parts = static_cast<float*>(ws);
  if (a.batch > 0) {
    const unsigned blocks = (unsigned)((int64_t)p.packs * p.chunks * a.batch);
    const dim3 block(kBackLanes, kBackRuns);
    SALT_WITH_TYPE(a.type, T, SALT_WITH_WIDTH(a.width, {
      if (p.v == 1)
        causal_conv_backward_kernel<T, 1, W>
            <<<blocks, block, 0, st>>>(a, p.packs, p.chunks, p.run, w_f32, w_vec, parts);
      else
        causal_conv_backward_kernel<T, kBackVec, W>
            <<<blocks, block, 0, st>>>(a, p.packs, p.chunks, p.run, w_f32, w_vec, parts);
    }));
    ++*launches;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  ++*launches;
  const int64_t dim = a.dim;
  return sum_parts_launch(
      parts, (int64_t)p.chunks * a.batch,
      PartSums{dim * a.width, dim, 0, a.dweight, a.dbias, nullptr, a.width}, st);
}

}  // namespace salt
