// Linear attention with a decay for each head: rows, single tokens, gradients.
//
// All gradients are the operator itself over other arguments: dq over (dout, v, k) in the row's
// order, dk and dv over (v, dout, q) and (k, q, dout) against it.  One pass computes
//   forward:  S = l S + k v^T;  out = scale * q S
//   reverse:  D = C + beta * k v^T;  out = q D;  C = l D   (from the row's end; C starts as given)
#include "sequence.cuh"

namespace salt {
namespace {

struct Rows {
  const void* p;
  int64_t batch, token;
  int share;  // heads that read one head of this array
};
struct Pass {
  Rows q, k, v;
  int dk, dv, heads, len, batch;
  float scale;
  bool reverse;
  const float* log_decay;
  const int32_t* n_real;
  const float* initial;
  bool initial_t;  // initial is (dv, dk)
  void* out;
  int64_t out_batch, out_token;
  float* final;
};

__device__ __forceinline__ float decay_of(const float* g, int h) {
  const float v = g[h];
  return v > 0.f ? 0.f : v < -200.f ? -200.f : v;  // a NaN stays one
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& r, int b, int64_t t, int h, int dim) {
  return static_cast<const T*>(r.p) + b * r.batch + t * r.token + (int64_t)(h / r.share) * dim;
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) attention_simple_kernel(Pass a) {
  __shared__ float red[8][33];
  const int tiles = (a.dv + 31) / 32;
  const int tile = blockIdx.x % tiles, bh = blockIdx.x / tiles, b = bh / a.heads, h = bh % a.heads;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, col = tile * 32 + x;
  const int n = row_tokens(a.n_real, b, a.len);
  const float l = expf(decay_of(a.log_decay, h));
  float s[16];
  for (int i = 0; i < 16; ++i) {
    const int r = y + 8 * i;
    const int64_t base = (int64_t)bh * a.dk * a.dv;
    s[i] = a.initial && r < a.dk && col < a.dv
               ? a.initial[base + (a.initial_t ? (int64_t)col * a.dk + r : (int64_t)r * a.dv + col)]
               : 0.f;
  }
  for (int i = 0; i < n; ++i) {
    const int t = a.reverse ? n - 1 - i : i;
    const T* q = row_of<T>(a.q, b, t, h, a.dk);
    const T* k = row_of<T>(a.k, b, t, h, a.dk);
    const float v = col < a.dv ? to_f32(row_of<T>(a.v, b, t, h, a.dv)[col]) : 0.f;
    float acc = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int r = y + 8 * j;
      if (r >= a.dk) continue;
      const float kv = to_f32(k[r]) * v;
      s[j] = a.reverse ? s[j] + a.scale * kv : l * s[j] + kv;
      acc += to_f32(q[r]) * s[j];
      if (a.reverse) s[j] *= l;
    }
    red[y][x] = acc;
    __syncthreads();
    if (y == 0 && col < a.dv) {
      float o = 0.f;
      for (int j = 0; j < 8; ++j) o += red[j][x];
      static_cast<O*>(a.out)[b * a.out_batch + t * a.out_token + (int64_t)h * a.dv + col] =
          from_f32<O>(a.reverse ? o : a.scale * o);
    }
    __syncthreads();
  }
  if (y == 0 && col < a.dv)
    for (int t = n; t < a.len; ++t)
      static_cast<O*>(a.out)[b * a.out_batch + t * a.out_token + (int64_t)h * a.dv + col] =
          from_f32<O>(0.f);
  if (a.final && col < a.dv)
    for (int j = 0; j < 16; ++j) {
      const int r = y + 8 * j;
      if (r < a.dk) a.final[(int64_t)bh * a.dk * a.dv + (int64_t)r * a.dv + col] = s[j];
    }
}

// Adds up what the heads that share a key head gave: (batch, len, kv, share, dim) of float32 to
// (batch, len, kv, dim), in the heads' order.
template <typename T>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* from, T* to, int64_t tokens,
                                                        int len, int kv, int share, int dim,
                                                        int64_t to_batch, int64_t to_token) {
  const int64_t each = (int64_t)kv * dim, n = tokens * each;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t token = i / each;
    const int at = (int)(i - token * each), h = at / dim, c = at - h * dim;
    const float* p = from + (token * kv + h) * share * dim + c;
    float s = 0.f;
    for (int j = 0; j < share; ++j) s += p[(int64_t)j * dim];
    const int64_t b = token / len;
    to[b * to_batch + (token - b * len) * to_token + at] = from_f32<T>(s);
  }
}

template <typename T, typename O>
cudaError_t run_pass(const Pass& p, cudaStream_t st, int* launches) {
  const int64_t blocks = (int64_t)p.batch * p.heads * ((p.dv + 31) / 32);
  if (!blocks) return cudaSuccess;
  attention_simple_kernel<T, O><<<(unsigned)blocks, 256, 0, st>>>(p);
  ++*launches;
  return cudaGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(128) attention_step_kernel(salt_linear_attention_step_args a) {
  const int bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, share = a.heads / a.kv_heads;
  const int slot = a.slots ? a.slots[b] : b;
  T* out = static_cast<T*>(a.out) + b * a.out_stride + (int64_t)h * a.dim_v;
  const int col = threadIdx.x;
  if (col >= a.dim_v) return;
  if (slot < 0 || slot >= a.n_slots) {
    out[col] = from_f32<T>(0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)h * a.dim_k;
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride + (int64_t)(h / share) * a.dim_k;
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride + (int64_t)(h / share) * a.dim_v;
  float* s = a.pool + ((int64_t)slot * a.heads + h) * a.dim_k * a.dim_v;
  const float l = expf(decay_of(a.log_decay, h)), vc = to_f32(v[col]);
  float acc = 0.f;
  for (int r = 0; r < a.dim_k; ++r) {
    const float x = l * s[r * a.dim_v + col] + to_f32(k[r]) * vc;
    s[r * a.dim_v + col] = x;
    acc += to_f32(q[r]) * x;
  }
  out[col] = from_f32<T>(a.scale * acc);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t linear_attention_bytes(const salt_linear_attention_args&) { return 0; }

cudaError_t linear_attention_launch(const salt_linear_attention_args& a, void*, cudaStream_t st,
                                    int* launches) {
  const int share = a.heads / a.kv_heads;
  Pass p{{a.q, a.q_batch_stride, a.q_stride, 1},
         {a.k, a.k_batch_stride, a.k_stride, share},
         {a.v, a.v_batch_stride, a.v_stride, share},
         a.dim_k, a.dim_v, a.heads, a.len, a.batch, a.scale, false, a.log_decay, a.n_real,
         a.initial_state, false, a.out, a.out_batch_stride, a.out_stride, a.final_state};
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, e = (run_pass<T, T>(p, st, launches)));
  return e;
}

cudaError_t linear_attention_step_launch(const salt_linear_attention_step_args& a, cudaStream_t st,
                                         int* launches) {
  if (!a.batch) return cudaSuccess;
  SALT_WITH_TYPE(a.type, T, attention_step_kernel<T><<<a.batch * a.heads, 128, 0, st>>>(a));
  ++*launches;
  return cudaGetLastError();
}

size_t linear_attention_backward_bytes(const salt_linear_attention_backward_args& a) {
  if (a.heads == a.kv_heads) return 0;
  return align256(4ull * a.batch * a.len * a.heads * std::max(a.dim_k, a.dim_v));
}

cudaError_t linear_attention_backward_launch(const salt_linear_attention_backward_args& a, void* ws,
                                             cudaStream_t st, int* launches) {
  const int share = a.heads / a.kv_heads;
  const Rows q{a.q, a.q_batch_stride, a.q_stride, 1}, k{a.k, a.k_batch_stride, a.k_stride, share},
      v{a.v, a.v_batch_stride, a.v_stride, share}, d{a.dout, a.dout_batch_stride, a.dout_stride, 1};
  const Pass dq{d, v, k, a.dim_v, a.dim_k, a.heads, a.len, a.batch, a.scale, false, a.log_decay,
                a.n_real, a.initial_state, true, a.dq, a.dq_batch_stride, a.dq_stride, nullptr};
  Pass dk{v, d, q, a.dim_v, a.dim_k, a.heads, a.len, a.batch, a.scale, true, a.log_decay, a.n_real,
          a.dfinal, true, a.dk, a.dk_batch_stride, a.dk_stride, nullptr};
  Pass dv{k, q, d, a.dim_k, a.dim_v, a.heads, a.len, a.batch, a.scale, true, a.log_decay, a.n_real,
          a.dfinal, false, a.dv, a.dv_batch_stride, a.dv_stride, a.dinitial};
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, {
    e = run_pass<T, T>(dq, st, launches);
    for (Pass* p : {&dk, &dv}) {
      if (e != cudaSuccess) return e;
      if (share == 1) {
        e = run_pass<T, T>(*p, st, launches);
        continue;
      }
      T* to = static_cast<T*>(p->out);
      const int64_t to_batch = p->out_batch, to_token = p->out_token;
      p->out = ws;
      p->out_token = (int64_t)a.heads * p->dv;
      p->out_batch = p->out_token * a.len;
      e = run_pass<T, float>(*p, st, launches);
      const int64_t n = (int64_t)a.batch * a.len * a.kv_heads * p->dv;
      if (e != cudaSuccess || !n) continue;
      sum_heads_kernel<T><<<(unsigned)std::min<int64_t>((n + 255) / 256, 148 * 8), 256, 0, st>>>(
          static_cast<const float*>(ws), to, (int64_t)a.batch * a.len, a.len, a.kv_heads, share,
          p->dv, to_batch, to_token);
      ++*launches;
      e = cudaGetLastError();
    }
  });
  return e;
}

}  // namespace salt
