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

constexpr int kTile = SALT_SCAN_CHECKPOINT;  // tokens
constexpr int kGroup = 4;                    // tokens whose states are in registers at a time
constexpr int kGroups = kTile / kGroup;

// LPC lanes hold a channel's states, 4 each, and CPT channels each: what a lane reads of B and C,
// and its sums for their gradients, serve both.  A thread moves P neighbouring channels of a token.
template <int LPC_, int CPT_, int CHANNELS>
struct BackShape {
  static constexpr int NS = 4, LPC = LPC_, CPT = CPT_, kChannels = CHANNELS;
  static constexpr int kThreads = kChannels * LPC / CPT;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kStates = NS * LPC;
  static constexpr int P = kTile * kChannels / kThreads;
  static constexpr int kIo = kChannels / P;  // threads of one token
  static constexpr int kStepPitch = kChannels + 64 / P, kPitch = kChannels + 8;
};

// As in the forward kernel: channel P v + k lies at place kIo k + v.
template <class S>
__device__ __forceinline__ int back_channel(int place) {
  return place % S::kIo * S::P + place / S::kIo;
}

template <typename T, class S>
struct BackShared {
  struct Raw {
    alignas(16) T x[kTile][S::kChannels], delta[kTile][S::kChannels], z[kTile][S::kChannels],
        dy[kTile][S::kChannels];
    alignas(16) T bc[2][kTile][S::kStates];
  } raw[2];  // this tile and the next, as they were loaded
  alignas(16) float2 step[kTile][S::kStepPitch];  // s and s * x
  alignas(16) float g[kTile][S::kPitch];
  alignas(16) float y[kTile][S::kPitch], to[kTile][S::kPitch], As[kTile][S::kPitch];
  alignas(16) float B[kTile][S::kStates], C[kTile][S::kStates];
  alignas(16) float part[S::kWarps][kTile][2 * S::kStates];    // each warp's dB and dC
  float4 start[kGroups - 1][S::CPT][S::kThreads];  // the states in front of groups 1, 2, 3
  float4 dA[S::CPT][S::kThreads];                  // the sum over the tiles so far
  alignas(8) float bias[S::kChannels], skip[S::kChannels];
};

struct BackParts {
  float* BC;            // (blocks, batch, len, 2 state): a block's dB and dC of its channels
  float *A, *D, *bias;  // (batch * chunks, dim, state), (batch * chunks, dim) twice
  int per_group;        // blocks of one group
};

template <typename T, class S, int COPY>
__global__ void __launch_bounds__(S::kThreads, 384 / S::kThreads)
selective_scan_backward_kernel(salt_selective_scan_backward_args a, ScanSplit sp, BackParts parts,
                               int blocks, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, CPT = S::CPT, P = S::P, H = NS / 2;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  BackShared<T, S>& sm = *reinterpret_cast<BackShared<T, S>*>(raw_shared);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.x / (blocks * sp.chunks);
  const int rest = (int)(blockIdx.x - b * blocks * sp.chunks), c = rest / blocks;
  const int block = rest - c * blocks;
  const ScanBlock cb = scan_block(block, a.dim, a.groups, S::kChannels);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, end = min(begin + sp.chunk_len, a.len);
  const int stop = min(real, end);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;

  const int at = tid / LPC * CPT, n0 = tid % LPC * NS, ns = a.state - n0;
  bool mine[CPT];
  int64_t d[CPT];
  f32x2 A[CPT][H], carry[CPT][H];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int ch = back_channel<S>(at + j);
    mine[j] = ch < cb.n;
    d[j] = cb.d0 + (mine[j] ? ch : 0);
    float f[NS], r[NS];
    load_states<NS>(f, a.A + d[j] * a.state + n0, mine[j] ? ns : 0, svec);
    // carry = a[t+1] dh[t+1] behind the chunk's last token: [c] holds chunk c + 1's own result, the
    // last live chunk's the gradient of the final state
    if (c >= last) {
      load_states<NS>(r, a.dfinal + (b * a.dim + d[j]) * a.state + n0,
                      mine[j] && a.dfinal && c == last ? ns : 0, svec);
    } else {
      const int64_t step = (int64_t)a.dim * a.state;
      const float* own = sp.state + (b * sp.chunks * a.dim + d[j]) * a.state + n0;
      load_states<NS>(r, own + (last - 1) * step, ns, svec);
      for (int k = last - 2; k >= c; --k) {
        float l[NS];
        load_states<NS>(l, own + k * step, ns, svec);
        const float s = sp.steps[(b * sp.chunks + k + 1) * a.dim + d[j]];
#pragma unroll
        for (int i = 0; i < NS; ++i) r[i] = fmaf(exp_fast(f[i] * s), r[i], l[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {
      A[j][i] = pair(f[2 * i] * kLog2e, f[2 * i + 1] * kLog2e);
      carry[j][i] = pair(r[2 * i], r[2 * i + 1]);
    }
    sm.dA[j][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  const int io_t = tid / S::kIo, io_v = tid % S::kIo;
  const int io_d = cb.d0 + io_v * P, io_n = cb.n - io_v * P;
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
  constexpr bool WIDE = COPY == kCopy16;
  for (int i = tid; i < S::kChannels; i += S::kThreads) {
    sm.bias[i] = a.delta_bias && i < cb.n ? a.delta_bias[cb.d0 + i] : 0.f;
    sm.skip[i] = a.D && i < cb.n ? a.D[cb.d0 + i] : 0.f;
  }
  float dbias[P], dskip[P];
#pragma unroll
  for (int k = 0; k < P; ++k) dbias[k] = dskip[k] = 0.f;

  // tokens past the row's end
  for (int t = max(stop, begin) / kTile * kTile + io_t; t < end; t += kTile) {
    if (t < stop) continue;
    float zero[P];
#pragma unroll
    for (int k = 0; k < P; ++k) zero[k] = 0.f;
    scan_store<T, P, WIDE>(dx + t * a.dx_stride, zero, io_n);
    scan_store<T, P, WIDE>(ddelta + t * a.ddelta_stride, zero, io_n);
    if (dz) scan_store<T, P, WIDE>(dz + t * a.dz_stride, zero, io_n);
  }

  constexpr int kPacks = kTile * S::kStates / 4;
  auto load = [&](int t0) {  // each thread copies what it converts itself
    auto& raw = sm.raw[t0 / kTile % 2];
    const int t = t0 + io_t, n = t < stop ? io_n : 0;
    copy_pack<COPY, P>(&raw.x[io_t][io_v * P], x + t * a.x_stride, n);
    copy_pack<COPY, P>(&raw.delta[io_t][io_v * P], delta + t * a.delta_stride, n);
    copy_pack<COPY, P>(&raw.dy[io_t][io_v * P], dy + t * a.dy_stride, n);
    if (z) copy_pack<COPY, P>(&raw.z[io_t][io_v * P], z + t * a.z_stride, n);
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      const int left = t0 + q < stop ? a.state - n1 : 0;
      copy_pack<COPY, 4>(&raw.bc[0][q][n1], B + (t0 + q) * a.B_stride + n1, left);
      copy_pack<COPY, 4>(&raw.bc[1][q][n1], C + (t0 + q) * a.C_stride + n1, left);
    }
    copies_commit();
  };

  const int first_tile = stop > begin ? (stop - 1) / kTile * kTile : -1;
  if (first_tile >= begin) load(first_tile);
  __syncthreads();  // bias and skip
  for (int t0 = first_tile; t0 >= begin; t0 -= kTile) {
    const int t = t0 + io_t;
    const bool live = t < stop;
    const auto& raw = sm.raw[t0 / kTile % 2];
    const T *rx = &raw.x[io_t][io_v * P], *rd = &raw.delta[io_t][io_v * P];
    const T *rz = &raw.z[io_t][io_v * P], *ry = &raw.dy[io_t][io_v * P];
    f32x2 h[CPT][H];  // the state in front of the tile
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      float f[NS];
      load_states<NS>(f, a.checkpoints + ((b * per + t0 / kTile) * a.dim + d[j]) * a.state + n0,
                      mine[j] ? ns : 0, svec);
      h[j][0] = pair(f[0], f[1]), h[j][1] = pair(f[2], f[3]);
    }
    if (t0 - kTile >= begin) {
      load(t0 - kTile);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float g = to_f32(ry[k]), s = 0.f;
      if (z) {
        const float v = to_f32(rz[k]);
        g *= v * sigmoid(v);
      }
      if (live) s = scan_step(to_f32(rd[k]) + sm.bias[io_v * P + k], a.softplus);
      sm.step[io_t][k * S::kIo + io_v] = make_float2(s, s * to_f32(rx[k]));
      sm.g[io_t][k * S::kIo + io_v] = g;  // 0 past the end, as dy there
    }
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      const T *p = &raw.bc[0][q][n1], *r = &raw.bc[1][q][n1];
      *reinterpret_cast<float4*>(&sm.B[q][n1]) =
          make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
      *reinterpret_cast<float4*>(&sm.C[q][n1]) =
          make_float4(to_f32(r[0]), to_f32(r[1]), to_f32(r[2]), to_f32(r[3]));
    }
    __syncthreads();

    auto step_of = [&](int q, float2 (&st)[CPT]) {
      if constexpr (CPT == 2) {
        const float4 v = *reinterpret_cast<const float4*>(&sm.step[q][at]);
        st[0] = make_float2(v.x, v.y), st[1] = make_float2(v.z, v.w);
      } else {
        st[0] = sm.step[q][at];
      }
    };
    // the states in front of each group but the first
#pragma unroll 1
    for (int u = 0; u < kGroups - 1; ++u) {
#pragma unroll
      for (int q = 0; q < kGroup; ++q) {
        float2 st[CPT];
        step_of(u * kGroup + q, st);
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&sm.B[u * kGroup + q][n0]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const f32x2 s = pair(st[j].x, st[j].x), sx = pair(st[j].y, st[j].y);
          h[j][0] = fma2(exp2_fast2(mul2(A[j][0], s)), h[j][0], mul2(sx, bn.x));
          h[j][1] = fma2(exp2_fast2(mul2(A[j][1], s)), h[j][1], mul2(sx, bn.y));
        }
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        *reinterpret_cast<ulonglong2*>(&sm.start[u][j][tid]) = make_ulonglong2(h[j][0], h[j][1]);
    }
    f32x2 dA[CPT][H] = {};
#pragma unroll 1
    for (int u = kGroups - 1; u >= 0; --u) {
      f32x2 ea[kGroup][CPT][H], hs[kGroup][CPT][H], h0[CPT][H];
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        if (u > 0) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.start[u - 1][j][tid]);
          h0[j][0] = v.x, h0[j][1] = v.y;
        } else {
          float f[NS];  // the checkpoint once more: from L1
          load_states<NS>(f, a.checkpoints + ((b * per + t0 / kTile) * a.dim + d[j]) * a.state + n0,
                          mine[j] ? ns : 0, svec);
          h0[j][0] = pair(f[0], f[1]), h0[j][1] = pair(f[2], f[3]);
        }
      }
#pragma unroll
      for (int q = 0; q < kGroup; ++q) {
        float2 st[CPT];
        step_of(u * kGroup + q, st);
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&sm.B[u * kGroup + q][n0]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const f32x2 s = pair(st[j].x, st[j].x), sx = pair(st[j].y, st[j].y);
          const f32x2* before = q ? hs[q ? q - 1 : 0][j] : h0[j];
          ea[q][j][0] = exp2_fast2(mul2(A[j][0], s));
          ea[q][j][1] = exp2_fast2(mul2(A[j][1], s));
          hs[q][j][0] = fma2(ea[q][j][0], before[0], mul2(sx, bn.x));
          hs[q][j][1] = fma2(ea[q][j][1], before[1], mul2(sx, bn.y));
        }
      }
      float sums[3][kGroup * CPT];  // y, sum of dh B, sum of m A: over this lane's states
#pragma unroll
      for (int q = kGroup - 1; q >= 0; --q) {
        const int row = u * kGroup + q;
        float2 st[CPT];
        float g[CPT];
        step_of(row, st);
        if constexpr (CPT == 2) {
          const float2 v = *reinterpret_cast<const float2*>(&sm.g[row][at]);
          g[0] = v.x, g[1] = v.y;
        } else {
          g[0] = sm.g[row][at];
        }
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&sm.B[row][n0]);
        const ulonglong2 cn = *reinterpret_cast<const ulonglong2*>(&sm.C[row][n0]);
        f32x2 dB[H] = {}, dC[H] = {};
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const f32x2 s = pair(st[j].x, st[j].x), sx = pair(st[j].y, st[j].y), gg = pair(g[j], g[j]);
          const f32x2* before = q ? hs[q ? q - 1 : 0][j] : h0[j];
          f32x2 y2 = 0, to2 = 0, As2 = 0;
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const f32x2 bi = i ? bn.y : bn.x, ci = i ? cn.y : cn.x;
            const f32x2 dh = fma2(gg, ci, carry[j][i]);
            y2 = fma2(hs[q][j][i], ci, y2);
            to2 = fma2(dh, bi, to2);
            dB[i] = fma2(dh, sx, dB[i]);
            dC[i] = fma2(gg, hs[q][j][i], dC[i]);
            carry[j][i] = mul2(ea[q][j][i], dh);
            const f32x2 m = mul2(carry[j][i], before[i]);
            As2 = fma2(m, A[j][i], As2);
            dA[j][i] = fma2(m, s, dA[j][i]);
          }
          const f32x2 all[3] = {y2, to2, As2};
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const float2 v = halves(all[k]);
            sums[k][q * CPT + j] = v.x + v.y;
          }
        }
        float bc[2 * NS];
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float2 v = halves(dB[i]), w = halves(dC[i]);
          bc[2 * i] = v.x, bc[2 * i + 1] = v.y;
          bc[NS + 2 * i] = w.x, bc[NS + 2 * i + 1] = w.y;
        }
        int first = 0;
        lane_sums<2 * NS, LPC, 32>(bc, lane, first);
        constexpr int DL = 32 / LPC, kept = DL >= 2 * NS ? 1 : 2 * NS / DL;
        // with more lanes than sums the first lanes of each group write
        if (DL <= 2 * NS || lane / (LPC * 2 * NS) == 0)
#pragma unroll
          for (int i = 0; i < kept; ++i) {
            const int v = first + i;
            sm.part[warp][row][(v < NS ? 0 : S::kStates) + n0 + v % NS] = bc[i];
          }
      }
      constexpr int values = kGroup * CPT;
      constexpr int left = LPC <= values ? values / LPC : 1;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        int first = 0;
        lane_sums<values, 1, LPC>(sums[k], lane, first);
        float(*out)[S::kPitch] = k == 0 ? sm.y : k == 1 ? sm.to : sm.As;
        if (LPC <= values || (lane & (LPC - 1)) < values)
#pragma unroll
          for (int i = 0; i < left; ++i)
            out[u * kGroup + (first + i) / CPT][at + (first + i) % CPT] = sums[k][i];
      }
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      // tile by tile: a sum of sums loses fewer digits than one long sum
      const float2 v = halves(dA[j][0]), w = halves(dA[j][1]);
      float4 f = sm.dA[j][tid];
      f.x += v.x, f.y += v.y, f.z += w.x, f.w += w.y;
      sm.dA[j][tid] = f;
    }
    __syncthreads();
    if (live) {
      float ox[P], od[P], oz[P];
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int place = k * S::kIo + io_v;
        const float xs = to_f32(rx[k]), g = sm.g[io_t][place], s = sm.step[io_t][place].x;
        const float to = sm.to[io_t][place], skip = sm.skip[io_v * P + k];
        ox[k] = fmaf(s, to, g * skip);
        // A held log2(e) times A
        od[k] = fmaf(xs, to, sm.As[io_t][place] * (1.f / kLog2e));
        if (a.softplus) od[k] *= sigmoid(to_f32(rd[k]) + sm.bias[io_v * P + k]);
        dbias[k] += od[k];
        dskip[k] = fmaf(g, xs, dskip[k]);
        if (z) {
          const float v = to_f32(rz[k]), y = fmaf(skip, xs, sm.y[io_t][place]);
          oz[k] = to_f32(ry[k]) * y * silu_slope(v, sigmoid(v));
        }
      }
      scan_store<T, P, WIDE>(dx + t * a.dx_stride, ox, io_n);
      scan_store<T, P, WIDE>(ddelta + t * a.ddelta_stride, od, io_n);
      if (dz) scan_store<T, P, WIDE>(dz + t * a.dz_stride, oz, io_n);
    }
    // the block's sum of dB and dC over its warps, in order
    for (int i = tid; i < kTile * 2 * a.state; i += S::kThreads) {
      const int q = i / (2 * a.state), v = i - q * 2 * a.state;
      const int from = v < a.state ? v : S::kStates + v - a.state;
      if (t0 + q < stop) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) sum += sm.part[w][q][from];
        parts.BC[(((int64_t)block * a.batch + b) * a.len + t0 + q) * 2 * a.state + v] = sum;
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    if (!mine[j]) continue;
    const float4 v = sm.dA[j][tid];
    const float f[NS] = {v.x, v.y, v.z, v.w};
    store_states<NS>(parts.A + ((b * sp.chunks + c) * a.dim + d[j]) * a.state + n0, f, ns, svec);
    if (c == 0 && a.dinitial) {
      const float2 lo = halves(carry[j][0]), hi = halves(carry[j][1]);
      const float r[NS] = {lo.x, lo.y, hi.x, hi.y};
      store_states<NS>(a.dinitial + (b * a.dim + d[j]) * a.state + n0, r, ns, svec);
    }
  }
  // the 16 tokens' threads of a channel pack add up what they saw, in order
#pragma unroll
  for (int k = 0; k < P; ++k) {
    sm.y[io_t][io_v * P + k] = dbias[k];
    sm.g[io_t][io_v * P + k] = dskip[k];
  }
  __syncthreads();
  for (int i = tid; i < cb.n; i += S::kThreads) {
    float sb = 0.f, ss = 0.f;
#pragma unroll
    for (int q = 0; q < kTile; ++q) {
      sb += sm.y[q][i];
      ss += sm.g[q][i];
    }
    const int64_t to = (b * sp.chunks + c) * a.dim + cb.d0 + i;
    parts.bias[to] = sb;
    parts.D[to] = ss;
  }
}

// The first pass over a split row, from its end: the carry in front of chunk c + 1 with nothing
// behind it (the last live chunk: the final state's gradient) into place c, and the chunk's steps.
template <typename T, class S, int COPY>
__global__ void __launch_bounds__(S::kThreads)
scan_back_state_kernel(salt_selective_scan_backward_args a, ScanSplit sp, int blocks, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, CPT = S::CPT, P = S::P, H = NS / 2;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  struct Shared {
    struct Raw {
      alignas(16) T delta[kTile][S::kChannels], z[kTile][S::kChannels], dy[kTile][S::kChannels];
      alignas(16) T c[kTile][S::kStates];
    } raw[2];
    alignas(16) float2 step[kTile][S::kStepPitch];  // s and g
    alignas(16) float C[kTile][S::kStates];
    float bias[S::kChannels];
  };
  static_assert(sizeof(Shared) <= sizeof(BackShared<T, S>), "");
  Shared& sm = *reinterpret_cast<Shared*>(raw_shared);
  const int tid = threadIdx.x, run = sp.chunks - 1;
  const int64_t b = blockIdx.x / (blocks * run);
  const int rest = (int)(blockIdx.x - b * blocks * run), c = rest / blocks + 1;
  const ScanBlock cb = scan_block(rest % blocks, a.dim, a.groups, S::kChannels);
  const int real = row_tokens(a.n_real, (int)b, a.len);
  const int begin = c * sp.chunk_len, stop = min(real, begin + sp.chunk_len);
  const int last = real > 0 ? (real - 1) / sp.chunk_len : 0;
  const int at = tid / LPC * CPT, n0 = tid % LPC * NS, ns = a.state - n0;
  bool mine[CPT];
  int64_t d[CPT];
  f32x2 A2[CPT][H], carry[CPT][H];
  float sum[CPT] = {};
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int ch = back_channel<S>(at + j);
    mine[j] = ch < cb.n;
    d[j] = cb.d0 + (mine[j] ? ch : 0);
    float f[NS], r[NS];
    load_states<NS>(f, a.A + d[j] * a.state + n0, mine[j] ? ns : 0, svec);
    load_states<NS>(r, a.dfinal + (b * a.dim + d[j]) * a.state + n0,
                    c == last && mine[j] && a.dfinal ? ns : 0, svec);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      A2[j][i] = pair(f[2 * i] * kLog2e, f[2 * i + 1] * kLog2e);
      carry[j][i] = pair(r[2 * i], r[2 * i + 1]);
    }
  }
  const int io_t = tid / S::kIo, io_v = tid % S::kIo;
  const int io_d = cb.d0 + io_v * P, io_n = cb.n - io_v * P;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + io_d;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + io_d : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + io_d;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  for (int i = tid; i < S::kChannels; i += S::kThreads)
    sm.bias[i] = a.delta_bias && i < cb.n ? a.delta_bias[cb.d0 + i] : 0.f;
  constexpr int kPacks = kTile * S::kStates / 4;
  auto load = [&](int t0) {
    auto& raw = sm.raw[t0 / kTile % 2];
    const int t = t0 + io_t, n = t < stop ? io_n : 0;
    copy_pack<COPY, P>(&raw.delta[io_t][io_v * P], delta + t * a.delta_stride, n);
    copy_pack<COPY, P>(&raw.dy[io_t][io_v * P], dy + t * a.dy_stride, n);
    if (z) copy_pack<COPY, P>(&raw.z[io_t][io_v * P], z + t * a.z_stride, n);
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      copy_pack<COPY, 4>(&raw.c[q][n1], C + (t0 + q) * a.C_stride + n1,
                         t0 + q < stop ? a.state - n1 : 0);
    }
    copies_commit();
  };
  const int first_tile = stop > begin ? (stop - 1) / kTile * kTile : -1;
  if (first_tile >= begin) load(first_tile);
  for (int t0 = first_tile; t0 >= begin; t0 -= kTile) {
    const int t = t0 + io_t;
    const auto& raw = sm.raw[t0 / kTile % 2];
    if (t0 - kTile >= begin) {
      load(t0 - kTile);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();  // the last tile's readers; the first time, bias
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float g = to_f32(raw.dy[io_t][io_v * P + k]), s = 0.f;
      if (z) {
        const float v = to_f32(raw.z[io_t][io_v * P + k]);
        g *= v * sigmoid(v);
      }
      if (t < stop)
        s = scan_step(to_f32(raw.delta[io_t][io_v * P + k]) + sm.bias[io_v * P + k], a.softplus);
      sm.step[io_t][k * S::kIo + io_v] = make_float2(s, g);
    }
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      const T* p = &raw.c[q][n1];
      *reinterpret_cast<float4*>(&sm.C[q][n1]) =
          make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
    }
    __syncthreads();
#pragma unroll 4
    for (int q = kTile - 1; q >= 0; --q) {
      const ulonglong2 cn = *reinterpret_cast<const ulonglong2*>(&sm.C[q][n0]);
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const float2 st = sm.step[q][at + j];
        sum[j] += st.x;
        const f32x2 s = pair(st.x, st.x), g = pair(st.y, st.y);
        carry[j][0] = mul2(exp2_fast2(mul2(A2[j][0], s)), fma2(g, cn.x, carry[j][0]));
        carry[j][1] = mul2(exp2_fast2(mul2(A2[j][1], s)), fma2(g, cn.y, carry[j][1]));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    if (!mine[j]) continue;
    const float2 lo = halves(carry[j][0]), hi = halves(carry[j][1]);
    const float r[NS] = {lo.x, lo.y, hi.x, hi.y};
    store_states<NS>(sp.state + ((b * sp.chunks + c - 1) * a.dim + d[j]) * a.state + n0, r, ns,
                     svec);
    if (n0 == 0) sp.steps[(b * sp.chunks + c) * a.dim + d[j]] = sum[j];
  }
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

using Back4 = BackShape<1, 1, 64>;
using Back8 = BackShape<2, 1, 64>;
#ifndef BCPT
#define BCPT 2
#endif
using Back16 = BackShape<4, BCPT, 64>;
using Back32 = BackShape<8, 2, 64>;
using Back64 = BackShape<16, 2, 32>;
#define SALT_BACK_SHAPE(state, S, ...) \
  SALT_BY_STATE(state, S, Back4, Back8, Back16, Back32, Back64, __VA_ARGS__)
int back_channels(int32_t state) {
  return state <= 32 ? Back16::kChannels : Back64::kChannels;
}

#ifndef BENOUGH
#define BENOUGH 3
#define BFILL 9
#endif
constexpr int kEnoughBlocks = 148 * BENOUGH;  // rows are not split
constexpr int kFillBlocks = 148 * BFILL;    // and otherwise into about so many

template <typename T, class S, int COPY>
cudaError_t back_launch(const salt_selective_scan_backward_args& a, const ScanSplit& sp,
                        const BackParts& parts, int blocks, bool svec, cudaStream_t st,
                        int* launches) {
  constexpr size_t shared = sizeof(BackShared<T, S>);
  const auto first = scan_back_state_kernel<T, S, COPY>;
  const auto main = selective_scan_backward_kernel<T, S, COPY>;
  cudaError_t e = cudaSuccess;
  if (shared > 48 * 1024) {
    const auto limit = cudaFuncAttributeMaxDynamicSharedMemorySize;
    e = cudaFuncSetAttribute(main, limit, (int)shared);
    if (e == cudaSuccess && sp.chunks > 1) e = cudaFuncSetAttribute(first, limit, (int)shared);
  }
  const int64_t rows = (int64_t)a.batch * blocks;
  if (e == cudaSuccess && sp.chunks > 1) {
    first<<<(unsigned)(rows * (sp.chunks - 1)), S::kThreads, shared, st>>>(a, sp, blocks, svec);
    ++*launches;
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    main<<<(unsigned)(rows * sp.chunks), S::kThreads, shared, st>>>(a, sp, parts, blocks, svec);
    ++*launches;
    e = cudaGetLastError();
  }
  return e;
}

struct BackPlan {
  int blocks, chunks, chunk_len;
  size_t state, steps, BC, A, D, bias, bytes;  // offsets in floats, and the whole in bytes
};

BackPlan back_plan(const salt_selective_scan_backward_args& a) {
  BackPlan p;
  p.blocks = scan_blocks(a.dim, a.groups, back_channels(a.state));
  p.chunks = 1, p.chunk_len = std::max(a.len, 1);
  const int64_t blocks = (int64_t)a.batch * p.blocks;
  if (blocks > 0 && blocks < kEnoughBlocks) {
    const int want = (int)(kFillBlocks / blocks);
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
  // the widest copies that no row's start and end stand against
  auto fits = [&](int64_t bytes) {
    const int64_t few = std::min<int64_t>(bytes, 4 * ts);
    const int pack = a.state <= 4 ? Back4::P : kVec;  // channels of the largest pack
    return (a.dim / a.groups) % (bytes == 16 ? pack : (int)(bytes / ts)) == 0 &&
           a.state % (few / ts) == 0 && packed_rows(a.x, bytes, ts, a.x_batch_stride, a.x_stride) &&
           packed_rows(a.delta, bytes, ts, a.delta_batch_stride, a.delta_stride) &&
           (!a.z || (packed_rows(a.z, bytes, ts, a.z_batch_stride, a.z_stride) &&
                     packed_rows(a.dz, bytes, ts, a.dz_batch_stride, a.dz_stride))) &&
           packed_rows(a.dy, bytes, ts, a.dy_batch_stride, a.dy_stride) &&
           packed_rows(a.dx, bytes, ts, a.dx_batch_stride, a.dx_stride) &&
           packed_rows(a.ddelta, bytes, ts, a.ddelta_batch_stride, a.ddelta_stride) &&
           packed_rows(a.B, few, ts, a.B_batch_stride, a.B_stride) &&
           packed_rows(a.C, few, ts, a.C_batch_stride, a.C_stride);
  };
  const int copy = fits(16) ? kCopy16 : fits(4) ? kCopy4 : kCopyPlain;
  const bool svec = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.dfinal) &&
                    aligned16(a.dinitial) && aligned16(a.checkpoints);
  cudaError_t e = cudaSuccess;
  if (a.batch > 0) {
    SALT_WITH_TYPE(a.type, T, SALT_BACK_SHAPE(a.state, S, {
      e = copy == kCopy16  ? back_launch<T, S, kCopy16>(a, sp, parts, p.blocks, svec, st, launches)
          : copy == kCopy4 ? back_launch<T, S, kCopy4>(a, sp, parts, p.blocks, svec, st, launches)
                           : back_launch<T, S, kCopyPlain>(a, sp, parts, p.blocks, svec, st,
                                                           launches);
    }));
    const int64_t n = (int64_t)a.batch * a.len * a.groups * 2 * a.state;
    if (e == cudaSuccess && n > 0) {
      SALT_WITH_TYPE(a.type, T, {
        scan_BC_gradient<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            a, parts.BC, parts.per_group, n);
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
