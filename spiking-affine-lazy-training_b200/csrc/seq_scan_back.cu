// Gradient of the selective state space scan.
//
// With g = dy * z sigmoid(z), the state's gradient runs from the last token to the first:
//   dh[t] = g[t] C[t] + a[t+1] dh[t+1],  a = exp(s A),
// and everything else is a sum over it: over the states for x, delta and z, over the channels of
// a group for B and C, over the tokens for A, D and delta_bias.  The states h[t] are not kept from
// the forward pass: it leaves one of 16, and a tile of 16 tokens is run again from there into
// registers.  That costs a second exponential for each state and token; the bound is these, the
// multiply-adds (about 14) and the shuffles of the two sums across lanes alike.
#include <algorithm>

#include "seq_scan.cuh"

namespace salt {

namespace {

constexpr int kTile = SALT_SCAN_CHECKPOINT;

// LPC lanes hold a channel's states, 4 each: 16 tokens' states are 64 registers.
template <int LPC_>
struct BackShape {
  static constexpr int NS = 4, LPC = LPC_;
  static constexpr int kThreads = LPC <= 4 ? kScanChannels * LPC : 256;
  static constexpr int kChannels = kThreads / LPC;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kStates = NS * LPC;
  static constexpr int kPack = kTile / LPC;  // neighbouring channels of one token that a thread moves
  static constexpr int kPitch = kChannels + 8;
};

template <class S>
struct BackShared {
  float s[kTile][S::kChannels], sx[kTile][S::kChannels], g[kTile][S::kChannels];
  float y[kTile][S::kPitch], to[kTile][S::kPitch], As[kTile][S::kPitch];
  float B[kTile][S::kStates], C[kTile][S::kStates];
  float part[S::kWarps][kTile][2 * S::kStates];  // each warp's dB and dC
};

struct BackParts {
  float *BC;                 // (blocks, batch, len, 2 state): a block's dB and dC of its channels
  float *A, *D, *bias;       // (batch * chunks, dim, state), (batch * chunks, dim) twice
  int groups_blocks;         // blocks of one group
};

template <typename T, class S>
__global__ void __launch_bounds__(S::kThreads)
selective_scan_backward_kernel(salt_selective_scan_backward_args a, ScanSplit sp, BackParts parts,
                               int blocks, bool vec, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, P = S::kPack, CB = S::kChannels;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  BackShared<S>& sm = *reinterpret_cast<BackShared<S>*>(raw_shared);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.x / (blocks * sp.chunks);
  const int rest = (int)(blockIdx.x - b * blocks * sp.chunks), c = rest / blocks;
  const int block = rest - c * blocks;
  const ScanBlock cb = scan_block(block, a.dim, a.groups, CB);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, end = min(begin + sp.chunk_len, a.len);
  const int stop = min(real, end);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;

  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  float A[NS], carry[NS], dA[NS];
  load_states<NS>(A, a.A + d * a.state + n0, mine ? ns : 0, svec);
#pragma unroll
  for (int i = 0; i < NS; ++i) dA[i] = 0.f;
  // carry = a[t+1] dh[t+1] behind the chunk's last token: [c] holds chunk c + 1's own result, the
  // last live chunk's the gradient of the final state
  if (c >= last) {
    load_states<NS>(carry, a.dfinal + (b * a.dim + d) * a.state + n0,
                    mine && a.dfinal && c == last ? ns : 0, svec);
  } else {
    const int64_t step = (int64_t)a.dim * a.state;
    const float* own = sp.state + (b * sp.chunks * a.dim + d) * a.state + n0;
    load_states<NS>(carry, own + (last - 1) * step, ns, svec);
    for (int k = last - 2; k >= c; --k) {
      float l[NS];
      load_states<NS>(l, own + k * step, ns, svec);
      const float s = sp.steps[(b * sp.chunks + k + 1) * a.dim + d];
#pragma unroll
      for (int i = 0; i < NS; ++i) carry[i] = fmaf(exp_fast(A[i] * s), carry[i], l[i]);
    }
  }

  const int io_t = tid / (CB / P), io_c = tid % (CB / P) * P;
  const int io_d = cb.d0 + io_c, io_n = cb.n - io_c;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + io_d;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + io_d;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + io_d : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + io_d;
  T* dx = static_cast<T*>(a.dx) + b * a.dx_batch_stride + io_d;
  T* ddelta = static_cast<T*>(a.ddelta) + b * a.ddelta_batch_stride + io_d;
  T* dz = z ? static_cast<T*>(a.dz) + b * a.dz_batch_stride + io_d : nullptr;
  const T* B = static_cast<const T*>(a.B) + b * a.B_batch_stride + (int64_t)cb.group * a.state;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  const int64_t per = (a.len + kTile - 1) / kTile;
  float bias[P], skip[P], dbias[P], dskip[P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    bias[k] = a.delta_bias && k < io_n ? a.delta_bias[io_d + k] : 0.f;
    skip[k] = a.D && k < io_n ? a.D[io_d + k] : 0.f;
    dbias[k] = dskip[k] = 0.f;
  }

  // tokens past the row's end
  for (int t = max(stop, begin) / kTile * kTile + io_t; t < end; t += kTile) {
    if (t < stop) continue;
    float zero[P];
#pragma unroll
    for (int k = 0; k < P; ++k) zero[k] = 0.f;
    store_pack<T, P>(dx + t * a.dx_stride, zero, io_n, vec);
    store_pack<T, P>(ddelta + t * a.ddelta_stride, zero, io_n, vec);
    if (dz) store_pack<T, P>(dz + t * a.dz_stride, zero, io_n, vec);
  }

  for (int t0 = stop > begin ? (stop - 1) / kTile * kTile : -1; t0 >= begin; t0 -= kTile) {
    const int t = t0 + io_t;
    const bool live = t < stop;
    Pack<T, P> px, pd, pz, py;
    {
      const int n = live ? io_n : 0;
      px = load_pack<T, P>(x + t * a.x_stride, n, vec);
      pd = load_pack<T, P>(delta + t * a.delta_stride, n, vec);
      py = load_pack<T, P>(dy + t * a.dy_stride, n, vec);
      if (z) pz = load_pack<T, P>(z + t * a.z_stride, n, vec);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float g = to_f32(py.v[k]);
        if (z) {
          const float v = to_f32(pz.v[k]);
          g *= v * sigmoid(v);
        }
        const float s = live ? scan_step(to_f32(pd.v[k]) + bias[k], a.softplus) : 0.f;
        sm.s[io_t][io_c + k] = s;
        sm.sx[io_t][io_c + k] = s * to_f32(px.v[k]);
        sm.g[io_t][io_c + k] = live ? g : 0.f;
      }
      for (int i = tid; i < kTile * S::kStates; i += S::kThreads) {
        const int q = i / S::kStates, n1 = i % S::kStates;
        const bool in = t0 + q < stop && n1 < a.state;
        sm.B[q][n1] = in ? to_f32(B[(t0 + q) * a.B_stride + n1]) : 0.f;
        sm.C[q][n1] = in ? to_f32(C[(t0 + q) * a.C_stride + n1]) : 0.f;
      }
    }
    float h0[NS], hist[kTile][NS];
    load_states<NS>(h0, a.checkpoints + ((b * per + t0 / kTile) * a.dim + d) * a.state + n0,
                    mine ? ns : 0, svec);
    __syncthreads();
    // the tile's states again, and y
    {
      float h[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) h[i] = h0[i];
#pragma unroll
      for (int q0 = 0; q0 < kTile; q0 += 4) {
        float yq[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int q = q0 + k;
          const float s = sm.s[q][ch] * kLog2e, sx = sm.sx[q][ch];
          yq[k] = 0.f;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            h[i] = fmaf(exp2_fast(A[i] * s), h[i], sx * sm.B[q][n0 + i]);
            hist[q][i] = h[i];
            yq[k] = fmaf(h[i], sm.C[q][n0 + i], yq[k]);
          }
        }
        int first = 0;
        lane_sums<4, 1, (LPC < 4 ? LPC : 4)>(yq, lane, first);
#pragma unroll
        for (int o = 4; o < LPC; o <<= 1) yq[0] += __shfl_xor_sync(0xffffffffu, yq[0], o);
        if ((lane & (LPC - 1)) < 4)
#pragma unroll
          for (int k = 0; k < (LPC < 4 ? 4 / LPC : 1); ++k) sm.y[q0 + first + k][ch] = yq[k];
      }
    }
#pragma unroll
    for (int q0 = kTile - 4; q0 >= 0; q0 -= 4) {
      float to[4], As[4];
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        const int q = q0 + k;
        const float s = sm.s[q][ch], sx = sm.sx[q][ch], g = sm.g[q][ch];
        to[k] = As[k] = 0.f;
        float bc[2 * NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float dh = fmaf(g, sm.C[q][n0 + i], carry[i]);
          bc[i] = dh * sx;
          bc[NS + i] = g * hist[q][i];
          to[k] = fmaf(dh, sm.B[q][n0 + i], to[k]);
          carry[i] = exp2_fast(A[i] * (s * kLog2e)) * dh;
          const float m = carry[i] * (q > 0 ? hist[q > 0 ? q - 1 : 0][i] : h0[i]);
          As[k] = fmaf(m, A[i], As[k]);
          dA[i] = fmaf(m, s, dA[i]);
        }
        int first = 0;
        lane_sums<2 * NS, LPC, 32>(bc, lane, first);
        constexpr int DL = 32 / LPC, kept = DL >= 2 * NS ? 1 : 2 * NS / DL;
        // with more lanes than sums the first lanes of each group write
        if (DL <= 2 * NS || lane / (LPC * 2 * NS) == 0)
#pragma unroll
          for (int i = 0; i < kept; ++i) {
            const int v = first + i;
            sm.part[warp][q][(v < NS ? 0 : S::kStates) + n0 + v % NS] = bc[i];
          }
      }
      int first = 0;
      lane_sums<4, 1, (LPC < 4 ? LPC : 4)>(to, lane, first);
      first = 0;
      lane_sums<4, 1, (LPC < 4 ? LPC : 4)>(As, lane, first);
#pragma unroll
      for (int o = 4; o < LPC; o <<= 1) {
        to[0] += __shfl_xor_sync(0xffffffffu, to[0], o);
        As[0] += __shfl_xor_sync(0xffffffffu, As[0], o);
      }
      if ((lane & (LPC - 1)) < 4)
#pragma unroll
        for (int k = 0; k < (LPC < 4 ? 4 / LPC : 1); ++k) {
          sm.to[q0 + first + k][ch] = to[k];
          sm.As[q0 + first + k][ch] = As[k];
        }
    }
    __syncthreads();
    if (live) {
      float ox[P], od[P], oz[P];
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const float xs = to_f32(px.v[k]), g = sm.g[io_t][io_c + k], s = sm.s[io_t][io_c + k];
        const float to = sm.to[io_t][io_c + k];
        ox[k] = fmaf(s, to, g * skip[k]);
        od[k] = fmaf(xs, to, sm.As[io_t][io_c + k]);
        if (a.softplus) od[k] *= sigmoid(to_f32(pd.v[k]) + bias[k]);
        dbias[k] += od[k];
        dskip[k] = fmaf(g, xs, dskip[k]);
        if (z) {
          const float v = to_f32(pz.v[k]), y = fmaf(skip[k], xs, sm.y[io_t][io_c + k]);
          oz[k] = to_f32(py.v[k]) * y * silu_slope(v, sigmoid(v));
        }
      }
      store_pack<T, P>(dx + t * a.dx_stride, ox, io_n, vec);
      store_pack<T, P>(ddelta + t * a.ddelta_stride, od, io_n, vec);
      if (dz) store_pack<T, P>(dz + t * a.dz_stride, oz, io_n, vec);
    }
    // the block's sum of dB and dC over its warps, in order
    for (int i = tid; i < kTile * 2 * a.state; i += S::kThreads) {
      const int q = i / (2 * a.state), v = i - q * 2 * a.state;
      const int at = v < a.state ? v : S::kStates + v - a.state;
      if (t0 + q < stop) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) sum += sm.part[w][q][at];
        parts.BC[(((int64_t)block * a.batch + b) * a.len + t0 + q) * 2 * a.state + v] = sum;
      }
    }
    __syncthreads();
  }

  if (mine) {
    store_states<NS>(parts.A + ((b * sp.chunks + c) * a.dim + d) * a.state + n0, dA, ns, svec);
    if (c == 0 && a.dinitial)
      store_states<NS>(a.dinitial + (b * a.dim + d) * a.state + n0, carry, ns, svec);
  }
  // the 16 tokens' threads of a channel pack add up what they saw, in order
#pragma unroll
  for (int k = 0; k < P; ++k) {
    sm.s[io_t][io_c + k] = dbias[k];
    sm.g[io_t][io_c + k] = dskip[k];
  }
  __syncthreads();
  if (tid < cb.n) {
    float sb = 0.f, ss = 0.f;
#pragma unroll
    for (int q = 0; q < kTile; ++q) {
      sb += sm.s[q][tid];
      ss += sm.g[q][tid];
    }
    const int64_t at = (b * sp.chunks + c) * a.dim + cb.d0 + tid;
    parts.bias[at] = sb;
    parts.D[at] = ss;
  }
}

// The first pass over a split row, from its end: the carry in front of chunk c + 1 with nothing
// behind it (the last live chunk: the final state's gradient) into place c, and the chunk's steps.
template <typename T, class S>
__global__ void __launch_bounds__(S::kThreads)
scan_back_state_kernel(salt_selective_scan_backward_args a, ScanSplit sp, int blocks, bool vec,
                       bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, P = S::kPack, CB = S::kChannels;
  __shared__ float2 step[kTile][CB];
  __shared__ float sC[kTile][S::kStates];
  const int tid = threadIdx.x, run = sp.chunks - 1;
  const int64_t b = blockIdx.x / (blocks * run);
  const int rest = (int)(blockIdx.x - b * blocks * run), c = rest / blocks + 1;
  const ScanBlock cb = scan_block(rest % blocks, a.dim, a.groups, CB);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, stop = min(real, begin + sp.chunk_len);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;
  const int ch = tid / LPC, n0 = tid % LPC * NS, ns = a.state - n0;
  const bool mine = ch < cb.n;
  const int64_t d = cb.d0 + (mine ? ch : 0);
  float A2[NS], carry[NS], sum = 0.f;
  load_states<NS>(A2, a.A + d * a.state + n0, mine ? ns : 0, svec);
#pragma unroll
  for (int i = 0; i < NS; ++i) A2[i] *= kLog2e;
  load_states<NS>(carry, a.dfinal + (b * a.dim + d) * a.state + n0,
                  c == last && mine && a.dfinal ? ns : 0, svec);
  const int io_t = tid / (CB / P), io_c = tid % (CB / P) * P;
  const int io_d = cb.d0 + io_c, io_n = cb.n - io_c;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + io_d;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + io_d : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + io_d;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  float bias[P];
#pragma unroll
  for (int k = 0; k < P; ++k)
    bias[k] = a.delta_bias && k < io_n ? a.delta_bias[io_d + k] : 0.f;
  for (int t0 = stop > begin ? (stop - 1) / kTile * kTile : -1; t0 >= begin; t0 -= kTile) {
    const int t = t0 + io_t, n = t < stop ? io_n : 0;
    const Pack<T, P> pd = load_pack<T, P>(delta + t * a.delta_stride, n, vec);
    const Pack<T, P> py = load_pack<T, P>(dy + t * a.dy_stride, n, vec);
    Pack<T, P> pz;
    if (z) pz = load_pack<T, P>(z + t * a.z_stride, n, vec);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float g = to_f32(py.v[k]);
      if (z) {
        const float v = to_f32(pz.v[k]);
        g *= v * sigmoid(v);
      }
      const bool in = t < stop;
      const float s = in ? scan_step(to_f32(pd.v[k]) + bias[k], a.softplus) : 0.f;
      step[io_t][io_c + k] = make_float2(s, in ? g : 0.f);
    }
    for (int i = tid; i < kTile * S::kStates; i += S::kThreads) {
      const int q = i / S::kStates, n1 = i % S::kStates;
      sC[q][n1] =
          t0 + q < stop && n1 < a.state ? to_f32(C[(t0 + q) * a.C_stride + n1]) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int q = kTile - 1; q >= 0; --q) {
      const float2 st = step[q][ch];
      sum += st.x;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        carry[i] = exp2_fast(A2[i] * st.x) * fmaf(st.y, sC[q][n0 + i], carry[i]);
    }
  }
  if (!mine) return;
  store_states<NS>(sp.state + ((b * sp.chunks + c - 1) * a.dim + d) * a.state + n0, carry, ns,
                   svec);
  if (n0 == 0) sp.steps[(b * sp.chunks + c) * a.dim + d] = sum;
}

// dB and dC of every token: the sum over the blocks of its group, zero past the row's end.
template <typename T>
__global__ void scan_BC_gradient(salt_selective_scan_backward_args a, const float* parts,
                                 int per_group, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int two = 2 * a.state;
  const int64_t row = i / (two * a.groups);
  const int v = (int)(i - row * two * a.groups), group = v / two, at = v - group * two;
  const int64_t b = row / a.len, t = row - b * a.len;
  float sum = 0.f;
  if (t < row_tokens(a.n_real, (int)b, a.len))
    for (int k = 0; k < per_group; ++k)
      sum += parts[(((int64_t)(group * per_group + k) * a.batch + b) * a.len + t) * two + at];
  T* out = static_cast<T*>(at < a.state ? a.dB : a.dC);
  out[(row * a.groups + group) * a.state + (at < a.state ? at : at - a.state)] = from_f32<T>(sum);
}

#define SALT_BACK_SHAPE(state, S, ...) \
  do {                                 \
    if ((state) <= 4) {                \
      using S = BackShape<1>;          \
      __VA_ARGS__;                     \
    } else if ((state) <= 8) {         \
      using S = BackShape<2>;          \
      __VA_ARGS__;                     \
    } else if ((state) <= 16) {        \
      using S = BackShape<4>;          \
      __VA_ARGS__;                     \
    } else if ((state) <= 32) {        \
      using S = BackShape<8>;          \
      __VA_ARGS__;                     \
    } else {                           \
      using S = BackShape<16>;         \
      __VA_ARGS__;                     \
    }                                  \
  } while (0)

int back_channels(int32_t state) { return state <= 16 ? 64 : state <= 32 ? 32 : 16; }

constexpr int kFillBlocks = 148 * 2;

struct BackPlan {
  int blocks, chunks, chunk_len;
  size_t state, steps, BC, A, D, bias, bytes;  // offsets in floats, and the whole in bytes
};

BackPlan back_plan(const salt_selective_scan_backward_args& a) {
  BackPlan p;
  p.blocks = scan_blocks(a.dim, a.groups, back_channels(a.state));
  p.chunks = 1, p.chunk_len = std::max(a.len, 1);
  const int64_t blocks = (int64_t)a.batch * p.blocks;
  if (blocks > 0 && blocks < kFillBlocks) {
    const int want = (int)((2 * kFillBlocks + blocks - 1) / blocks);
    const int each = std::max(128, (a.len + want - 1) / want);
    p.chunk_len = (each + kTile - 1) / kTile * kTile;
    p.chunks = std::max(1, (a.len + p.chunk_len - 1) / p.chunk_len);
  }
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += (n + 63) / 64 * 64;
    return o;
  };
  const size_t rows = (size_t)a.batch * p.chunks * a.dim;
  p.state = take(p.chunks > 1 ? rows * a.state : 0);
  p.steps = take(p.chunks > 1 ? rows : 0);
  p.BC = take((size_t)p.blocks * a.batch * a.len * 2 * a.state);
  p.A = take(rows * a.state);
  p.D = take(rows);
  p.bias = take(rows);
  p.bytes = at * sizeof(float);
  return p;
}

}  // namespace

size_t selective_scan_backward_bytes(const salt_selective_scan_backward_args& a) {
  return back_plan(a).bytes;
}

cudaError_t selective_scan_backward_launch(const salt_selective_scan_backward_args& a, void* ws,
                                           cudaStream_t st, int* launches) {
  const BackPlan p = back_plan(a);
  float* base = static_cast<float*>(ws);
  const ScanSplit sp{p.chunks, p.chunk_len, base + p.state, base + p.steps};
  const BackParts parts{base + p.BC, base + p.A, base + p.D, base + p.bias, p.blocks / a.groups};
  const size_t ts = type_size(a.type);
  const bool vec = (a.groups == 1 || (a.dim / a.groups * ts) % 16 == 0) &&
                   vec_rows(a.x, ts, a.x_batch_stride, a.x_stride) &&
                   vec_rows(a.delta, ts, a.delta_batch_stride, a.delta_stride) &&
                   vec_rows(a.z, ts, a.z_batch_stride, a.z_stride) &&
                   vec_rows(a.dy, ts, a.dy_batch_stride, a.dy_stride) &&
                   vec_rows(a.dx, ts, a.dx_batch_stride, a.dx_stride) &&
                   vec_rows(a.ddelta, ts, a.ddelta_batch_stride, a.ddelta_stride) &&
                   vec_rows(a.dz, ts, a.dz_batch_stride, a.dz_stride);
  const bool svec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.dfinal) &&
                    aligned16(a.dinitial) && aligned16(a.checkpoints);
  cudaError_t e = cudaSuccess;
  if (a.batch > 0) {
    SALT_WITH_TYPE(a.type, T, SALT_BACK_SHAPE(a.state, S, {
      if (p.chunks > 1) {
        scan_back_state_kernel<T, S><<<(unsigned)((int64_t)a.batch * p.blocks * (p.chunks - 1)),
                                       S::kThreads, 0, st>>>(a, sp, p.blocks, vec, svec);
        ++*launches;
        e = cudaGetLastError();
      }
      constexpr size_t shared = sizeof(BackShared<S>);
      if (e == cudaSuccess && shared > 48 * 1024)
        e = cudaFuncSetAttribute(selective_scan_backward_kernel<T, S>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
      if (e == cudaSuccess) {
        selective_scan_backward_kernel<T, S>
            <<<(unsigned)((int64_t)a.batch * p.blocks * p.chunks), S::kThreads, shared, st>>>(
                a, sp, parts, p.blocks, vec, svec);
        ++*launches;
        e = cudaGetLastError();
      }
    }));
    const int64_t n = (int64_t)a.batch * a.len * a.groups * 2 * a.state;
    if (e == cudaSuccess && n > 0) {
      SALT_WITH_TYPE(a.type, T, {
        scan_BC_gradient<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            a, parts.BC, parts.groups_blocks, n);
      });
      ++*launches;
      e = cudaGetLastError();
    }
  }
  const int64_t rows = (int64_t)a.batch * p.chunks;
  if (e == cudaSuccess) {
    e = sum_parts_launch(parts.A, rows, (int64_t)a.dim * a.state, a.dA, st);
    ++*launches;
  }
  if (e == cudaSuccess && a.dD) {
    e = sum_parts_launch(parts.D, rows, a.dim, a.dD, st);
    ++*launches;
  }
  if (e == cudaSuccess && a.ddelta_bias) {
    e = sum_parts_launch(parts.bias, rows, a.dim, a.ddelta_bias, st);
    ++*launches;
  }
  return e;
}

}  // namespace salt
