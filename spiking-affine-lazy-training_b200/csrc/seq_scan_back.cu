// Gradient of the selective state space scan.
//
// With g = dy * z sigmoid(z), the state's gradient runs from the last token to the first:
//   dh[t] = g[t] C[t] + a[t+1] dh[t+1],  a = exp(s A),
// and everything else is a sum over it: over the states for x, delta and z, over the channels of a
// group for B and C, over the tokens for A, D and delta_bias.  The states h[t] are not kept from
// the forward pass: it leaves one of 16, and a tile of 16 tokens is run again from there into
// registers, 4 tokens at a time.  That costs 1.75 exponentials for each state and token; these,
// about 22 instructions and the shuffles of the two sums across lanes bound it alike.  Forward and
// backward of 4 rows of 2048 tokens x 2048 channels x 16 states in bf16 take 752 us, of which the
// main kernel here has 432 us: 12 warps on an SM (168 registers) issue an instruction in every
// second cycle. The first form, with a tile's states in 64 registers of one channel a lane, took
// 1612 us; one channel a lane in this form 880 to 950 us (25 reads of shared memory to 18), 128
// registers 842 us.
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
  alignas(16) float2 step[kTile][S::kStepPitch];  // s and s * x; at last s and y
  alignas(16) float g[kTile][S::kPitch], to[kTile][S::kPitch], As[kTile][S::kPitch];
  alignas(16) float B[4][kTile][S::kStates], C[4][kTile][S::kStates];  // in every lane order
  alignas(16) float part[S::kWarps][kTile][2 * S::kStates];    // each warp's dB and dC
  float4 start[kGroups - 1][S::CPT][S::kThreads];  // the states in front of groups 1, 2, 3
  float4 dA[S::CPT][S::kThreads];                  // the sum over the tiles so far
  alignas(8) float bias[S::kChannels], skip[S::kChannels];
};

// The sums over channels, of dB and dC, halve what a lane holds at each step across lanes: it keeps
// one half and sends the other.  So that no lane has to choose between registers, the lanes hold
// their 4 states in different orders, always keep what lies first and send what lies second: lane
// bit LPC swaps the pairs of states, bit 2 LPC the two of a pair (where the warp has such bits).
// Likewise bit 1 swaps a lane's two channels for the sums over states.
template <class S>
struct LaneOrder {
  int pairs, halves, channels;  // 0 or 1 each
  __device__ __forceinline__ explicit LaneOrder(int lane)
      : pairs(S::LPC < 32 ? lane / S::LPC % 2 : 0),
        halves(2 * S::LPC < 32 ? lane / (2 * S::LPC) % 2 : 0),
        channels(S::CPT == 2 && S::LPC > 1 ? lane % 2 : 0) {}
  // memory order to lane order, or back (either is its own inverse)
  __device__ __forceinline__ void turn(float (&f)[4]) const {
    const float p0 = pairs ? f[2] : f[0], p1 = pairs ? f[3] : f[1];
    const float q0 = pairs ? f[0] : f[2], q1 = pairs ? f[1] : f[3];
    f[0] = halves ? p1 : p0, f[1] = halves ? p0 : p1;
    f[2] = halves ? q1 : q0, f[3] = halves ? q0 : q1;
  }
};

__device__ __forceinline__ f32x2 shuffle2(f32x2 v, int mask) {
  const float2 h = salt::halves(v);
  return pair(__shfl_xor_sync(0xffffffffu, h.x, mask), __shfl_xor_sync(0xffffffffu, h.y, mask));
}

// BC is what the workspace holds most of: 8 bytes a token and state for every block of 64 channels
// (32 of them over 32 states), so at 64 states 16 bytes a token and channel, written and read once.
struct BackParts {
  float* BC;            // (blocks, batch, len, 2 state): a block's dB and dC of its channels
  float* sums;          // (batch * chunks, dim * (state + 2)): dA, dD and ddelta_bias
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

  const LaneOrder<S> order(lane);
  const int n0 = tid % LPC * NS, ns = a.state - n0;
  int at[CPT];  // places of the lane's channels
  bool mine[CPT];
  int64_t d[CPT];
  f32x2 A[CPT][H], carry[CPT][H];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    at[j] = tid / LPC * CPT + (j ^ order.channels);
    const int ch = back_channel<S>(at[j]);
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
    order.turn(f);
    order.turn(r);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      A[j][i] = pair(f[2 * i] * kLog2e, f[2 * i + 1] * kLog2e);
      carry[j][i] = pair(r[2 * i], r[2 * i + 1]);
    }
    sm.dA[j][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  const int io_t = tid / S::kIo, io_v = tid % S::kIo;
  const int io_n = cb.n - io_v * P;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch_stride + cb.d0;
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + cb.d0;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + cb.d0 : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + cb.d0;
  T* dx = static_cast<T*>(a.dx) + b * a.dx_batch_stride + cb.d0;
  T* ddelta = static_cast<T*>(a.ddelta) + b * a.ddelta_batch_stride + cb.d0;
  T* dz = z ? static_cast<T*>(a.dz) + b * a.dz_batch_stride + cb.d0 : nullptr;
  const T* B = static_cast<const T*>(a.B) + b * a.B_batch_stride + (int64_t)cb.group * a.state;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  const int64_t per = (a.len + kTile - 1) / kTile;
  constexpr bool WIDE = COPY == kCopy16;
  for (int i = tid; i < S::kChannels; i += S::kThreads) {
    sm.bias[i] = a.delta_bias && i < cb.n ? a.delta_bias[cb.d0 + i] : 0.f;
    sm.skip[i] = a.D && i < cb.n ? a.D[cb.d0 + i] : 0.f;
  }
  f32x2 dbias[P / 2] = {}, dskip[P / 2] = {};

  // tokens past the row's end
  for (int t = max(stop, begin) / kTile * kTile + io_t; t < end; t += kTile) {
    if (t < stop) continue;
    const float zero[P] = {};
    store_pack<T, P>(dx + t * a.dx_stride + io_v * P, zero, io_n, WIDE);
    store_pack<T, P>(ddelta + t * a.ddelta_stride + io_v * P, zero, io_n, WIDE);
    if (dz) store_pack<T, P>(dz + t * a.dz_stride + io_v * P, zero, io_n, WIDE);
  }

  constexpr int kPacks = kTile * S::kStates / 4;
  auto load = [&](int t0) {  // in copies of 16 bytes each thread copies what it converts itself
    auto& raw = sm.raw[t0 / kTile % 2];
    auto tile = [&](T(*to)[S::kChannels], const T* from, int64_t stride) {
      copy_tile<COPY, P, kTile, S::kChannels, S::kThreads>(to, from, stride, t0, stop, cb.n);
    };
    tile(raw.x, x, a.x_stride);
    tile(raw.delta, delta, a.delta_stride);
    tile(raw.dy, dy, a.dy_stride);
    if (z) tile(raw.z, z, a.z_stride);
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
    auto& raw = sm.raw[t0 / kTile % 2];
    f32x2 h[CPT][H];  // the state in front of the tile
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      float f[NS];
      load_states<NS>(f, a.checkpoints + ((b * per + t0 / kTile) * a.dim + d[j]) * a.state + n0,
                      mine[j] ? ns : 0, svec);
      order.turn(f);
      h[j][0] = pair(f[0], f[1]), h[j][1] = pair(f[2], f[3]);
    }
    if (t0 - kTile >= begin) {
      load(t0 - kTile);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    if (!WIDE) __syncthreads();
    {
      const auto px = pack_at<P>(&raw.x[io_t][io_v * P]);
      const auto pd = pack_at<P>(&raw.delta[io_t][io_v * P]);
      const auto pz = pack_at<P>(&raw.z[io_t][io_v * P]), py = pack_at<P>(&raw.dy[io_t][io_v * P]);
#pragma unroll
      for (int k = 0; k < P; k += 2) {
        f32x2 g2 = pair_of(py, k);
        if (z) {
          const f32x2 v = pair_of(pz, k);
          g2 = mul2(g2, mul2(v, sigmoid2(v)));
        }
        const f32x2 in =
            add2(pair_of(pd, k), pair(sm.bias[io_v * P + k], sm.bias[io_v * P + k + 1]));
        const f32x2 s2 = live ? scan_step2(in, a.softplus) : 0;
        const float2 s = halves(s2), sx = halves(mul2(s2, pair_of(px, k))), g = halves(g2);
        sm.step[io_t][k * S::kIo + io_v] = make_float2(s.x, sx.x);
        sm.step[io_t][(k + 1) * S::kIo + io_v] = make_float2(s.y, sx.y);
        sm.g[io_t][k * S::kIo + io_v] = g.x;  // 0 past the end, as dy there
        sm.g[io_t][(k + 1) * S::kIo + io_v] = g.y;
      }
    }
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const auto p = pack_at<4>(&raw.bc[k][q][n1]);
        const float2 lo = halves(pair_of(p, 0)), hi = halves(pair_of(p, 2));
        auto to = k ? sm.C : sm.B;
        *reinterpret_cast<float4*>(&to[0][q][n1]) = make_float4(lo.x, lo.y, hi.x, hi.y);
        *reinterpret_cast<float4*>(&to[1][q][n1]) = make_float4(hi.x, hi.y, lo.x, lo.y);
        *reinterpret_cast<float4*>(&to[2][q][n1]) = make_float4(lo.y, lo.x, hi.y, hi.x);
        *reinterpret_cast<float4*>(&to[3][q][n1]) = make_float4(hi.y, hi.x, lo.y, lo.x);
      }
    }
    __syncthreads();

    const float(*Bo)[S::kStates] = sm.B[order.pairs + 2 * order.halves];
    const float(*Co)[S::kStates] = sm.C[order.pairs + 2 * order.halves];
    // the states in front of each group but the first
#pragma unroll 1
    for (int u = 0; u < kGroups - 1; ++u) {
#pragma unroll
      for (int q = 0; q < kGroup; ++q) {
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&Bo[u * kGroup + q][n0]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const float2 st = sm.step[u * kGroup + q][at[j]];
          const f32x2 s = both(st.x), sx = both(st.y);
          h[j][0] = fma2(decay2(A[j][0], s), h[j][0], mul2(sx, bn.x));
          h[j][1] = fma2(decay2(A[j][1], s), h[j][1], mul2(sx, bn.y));
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
          order.turn(f);
          h0[j][0] = pair(f[0], f[1]), h0[j][1] = pair(f[2], f[3]);
        }
      }
#pragma unroll
      for (int q = 0; q < kGroup; ++q) {
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&Bo[u * kGroup + q][n0]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const float2 st = sm.step[u * kGroup + q][at[j]];
          const f32x2 s = both(st.x), sx = both(st.y);
          const f32x2* before = q ? hs[q ? q - 1 : 0][j] : h0[j];
          ea[q][j][0] = decay2(A[j][0], s);
          ea[q][j][1] = decay2(A[j][1], s);
          hs[q][j][0] = fma2(ea[q][j][0], before[0], mul2(sx, bn.x));
          hs[q][j][1] = fma2(ea[q][j][1], before[1], mul2(sx, bn.y));
        }
      }
      float sums[3][CPT][kGroup];  // y, sum of dh B, sum of m A: over this lane's states
#pragma unroll
      for (int q = kGroup - 1; q >= 0; --q) {
        const int row = u * kGroup + q;
        const ulonglong2 bn = *reinterpret_cast<const ulonglong2*>(&Bo[row][n0]);
        const ulonglong2 cn = *reinterpret_cast<const ulonglong2*>(&Co[row][n0]);
        f32x2 dB[H] = {}, dC[H] = {};
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const float2 st = sm.step[row][at[j]];
          const f32x2 s = both(st.x), sx = both(st.y), gg = both(sm.g[row][at[j]]);
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
            sums[k][j][q] = v.x + v.y;
          }
        }
        // what is left of dB and dC on this lane after the halvings: of pair order.pairs, its
        // half order.halves, and one of the two
        float* to = &sm.part[warp][row][n0 + 2 * order.pairs];
        dB[0] = add2(dB[0], shuffle2(dB[1], LPC));
        dC[0] = add2(dC[0], shuffle2(dC[1], LPC));
        const float2 vb = halves(dB[0]), vc = halves(dC[0]);
        if constexpr (2 * LPC >= 32) {
          *reinterpret_cast<float2*>(to) = vb;
          *reinterpret_cast<float2*>(to + S::kStates) = vc;
        } else {
          const float kb = vb.x + __shfl_xor_sync(0xffffffffu, vb.y, 2 * LPC);
          const float kc = vc.x + __shfl_xor_sync(0xffffffffu, vc.y, 2 * LPC);
          to += order.halves;
          if constexpr (4 * LPC >= 32) {
            to[0] = kb;
            to[S::kStates] = kc;
          } else {
            const bool up = lane & (4 * LPC);
            float v = (up ? kc : kb) + __shfl_xor_sync(0xffffffffu, up ? kb : kc, 4 * LPC);
#pragma unroll
            for (int o = 8 * LPC; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane < 8 * LPC) to[up ? S::kStates : 0] = v;
          }
        }
      }
      __syncwarp();  // the group's s x has been read
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        float* v = sums[k][0];
        if constexpr (CPT == 2 && LPC > 1) {
#pragma unroll
          for (int q = 0; q < kGroup; ++q)
            v[q] += __shfl_xor_sync(0xffffffffu, sums[k][CPT - 1][q], 1);
        }
        // the rest of the channel's lanes, over the group's tokens
        int first = 0;
        constexpr int from = CPT == 2 ? 2 : 1, lanes = LPC / from;
        constexpr int left = lanes >= kGroup ? 1 : lanes > 1 ? kGroup / lanes : kGroup;
        lane_sums<kGroup, from, LPC>(v, lane, first);
        if (lanes <= kGroup || (lane & (LPC - 1)) / from < kGroup)
#pragma unroll
          for (int i = 0; i < left; ++i) {
            const int row = u * kGroup + first + i;
            if (k == 0)
              sm.step[row][at[0]].y = v[i];
            else
              (k == 1 ? sm.to : sm.As)[row][at[0]] = v[i];
          }
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
      const auto px = pack_at<P>(&raw.x[io_t][io_v * P]);
      const auto pd = pack_at<P>(&raw.delta[io_t][io_v * P]);
      const auto pz = pack_at<P>(&raw.z[io_t][io_v * P]), py = pack_at<P>(&raw.dy[io_t][io_v * P]);
      float ox[P], od[P], oz[P];
#pragma unroll
      for (int k = 0; k < P; k += 2) {
        const int p0 = k * S::kIo + io_v, p1 = p0 + S::kIo;
        const f32x2 xs = pair_of(px, k), g = pair(sm.g[io_t][p0], sm.g[io_t][p1]);
        const f32x2 s = pair(sm.step[io_t][p0].x, sm.step[io_t][p1].x);
        const f32x2 to = pair(sm.to[io_t][p0], sm.to[io_t][p1]);
        const f32x2 skip = pair(sm.skip[io_v * P + k], sm.skip[io_v * P + k + 1]);
        float2 f = halves(fma2(s, to, mul2(g, skip)));
        ox[k] = f.x, ox[k + 1] = f.y;
        // A held log2(e) times A
        f32x2 dd = fma2(xs, to, mul2(pair(sm.As[io_t][p0], sm.As[io_t][p1]), both(1.f / kLog2e)));
        if (a.softplus)
          dd = mul2(dd, sigmoid2(add2(pair_of(pd, k), pair(sm.bias[io_v * P + k],
                                                           sm.bias[io_v * P + k + 1]))));
        f = halves(dd);
        od[k] = f.x, od[k + 1] = f.y;
        dbias[k / 2] = add2(dbias[k / 2], dd);
        dskip[k / 2] = fma2(g, xs, dskip[k / 2]);
        if (z) {
          const f32x2 v = pair_of(pz, k);
          const f32x2 y = fma2(skip, xs, pair(sm.step[io_t][p0].y, sm.step[io_t][p1].y));
          f = halves(mul2(mul2(pair_of(py, k), y), silu_slope2(v, sigmoid2(v))));
          oz[k] = f.x, oz[k + 1] = f.y;
        }
      }
      const int at = io_v * P;
      scan_store<T, P, WIDE>(dx + t * a.dx_stride + at, &raw.x[io_t][at], ox, io_n);
      scan_store<T, P, WIDE>(ddelta + t * a.ddelta_stride + at, &raw.delta[io_t][at], od, io_n);
      if (dz) scan_store<T, P, WIDE>(dz + t * a.dz_stride + at, &raw.z[io_t][at], oz, io_n);
    }
    if (!WIDE) {
      __syncthreads();
      auto back = [&](T* to, T(*from)[S::kChannels], int64_t stride) {
        store_tile<COPY, kTile, S::kChannels, S::kThreads>(to, from, stride, t0, stop, cb.n);
      };
      back(dx, raw.x, a.dx_stride);
      back(ddelta, raw.delta, a.ddelta_stride);
      if (dz) back(dz, raw.z, a.dz_stride);
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

  float* sums = parts.sums + (b * sp.chunks + c) * a.dim * (a.state + 2);
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    if (!mine[j]) continue;
    const float4 v = sm.dA[j][tid];
    float f[NS] = {v.x, v.y, v.z, v.w};
    order.turn(f);
    // a row of sums has dim * (state + 2) values
    store_states<NS>(sums + d[j] * a.state + n0, f, ns, svec && a.dim % 2 == 0);
    if (c == 0 && a.dinitial) {
      const float2 lo = halves(carry[j][0]), hi = halves(carry[j][1]);
      float r[NS] = {lo.x, lo.y, hi.x, hi.y};
      order.turn(r);
      store_states<NS>(a.dinitial + (b * a.dim + d[j]) * a.state + n0, r, ns, svec);
    }
  }
  // the 16 tokens' threads of a channel pack add up what they saw, in order
#pragma unroll
  for (int k = 0; k < P; k += 2) {
    *reinterpret_cast<f32x2*>(&sm.to[io_t][io_v * P + k]) = dbias[k / 2];
    *reinterpret_cast<f32x2*>(&sm.g[io_t][io_v * P + k]) = dskip[k / 2];
  }
  __syncthreads();
  for (int i = tid; i < cb.n; i += S::kThreads) {
    float sb = 0.f, ss = 0.f;
#pragma unroll
    for (int q = 0; q < kTile; ++q) {
      sb += sm.to[q][i];
      ss += sm.g[q][i];
    }
    float* to = sums + (int64_t)a.dim * a.state + cb.d0 + i;
    to[0] = ss;
    to[a.dim] = sb;
  }
}

template <typename T, class S>
struct BackStateShared {
  struct Raw {
    alignas(16) T delta[kTile][S::kChannels], z[kTile][S::kChannels], dy[kTile][S::kChannels];
    alignas(16) T c[kTile][S::kStates];
  } raw[2];
  alignas(16) float2 step[kTile][S::kStepPitch];  // s and g
  alignas(16) float C[kTile][S::kStates];
  float bias[S::kChannels];
};

// The first pass over a split row, from its end: the carry in front of chunk c + 1 with nothing
// behind it (the last live chunk: the final state's gradient) into place c, and the chunk's steps.
template <typename T, class S, int COPY>
__global__ void __launch_bounds__(S::kThreads)
scan_back_state_kernel(salt_selective_scan_backward_args a, ScanSplit sp, int blocks, bool svec) {
  constexpr int NS = S::NS, LPC = S::LPC, CPT = S::CPT, P = S::P, H = NS / 2;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  BackStateShared<T, S>& sm = *reinterpret_cast<BackStateShared<T, S>*>(raw_shared);
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
  const T* delta = static_cast<const T*>(a.delta) + b * a.delta_batch_stride + cb.d0;
  const T* z = a.z ? static_cast<const T*>(a.z) + b * a.z_batch_stride + cb.d0 : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch_stride + cb.d0;
  const T* C = static_cast<const T*>(a.C) + b * a.C_batch_stride + (int64_t)cb.group * a.state;
  for (int i = tid; i < S::kChannels; i += S::kThreads)
    sm.bias[i] = a.delta_bias && i < cb.n ? a.delta_bias[cb.d0 + i] : 0.f;
  constexpr int kPacks = kTile * S::kStates / 4;
  auto load = [&](int t0) {
    auto& raw = sm.raw[t0 / kTile % 2];
    auto tile = [&](T(*to)[S::kChannels], const T* from, int64_t stride) {
      copy_tile<COPY, P, kTile, S::kChannels, S::kThreads>(to, from, stride, t0, stop, cb.n);
    };
    tile(raw.delta, delta, a.delta_stride);
    tile(raw.dy, dy, a.dy_stride);
    if (z) tile(raw.z, z, a.z_stride);
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
    {
      const auto pd = pack_at<P>(&raw.delta[io_t][io_v * P]);
      const auto pz = pack_at<P>(&raw.z[io_t][io_v * P]), py = pack_at<P>(&raw.dy[io_t][io_v * P]);
#pragma unroll
      for (int k = 0; k < P; k += 2) {
        f32x2 g2 = pair_of(py, k);
        if (z) {
          const f32x2 v = pair_of(pz, k);
          g2 = mul2(g2, mul2(v, sigmoid2(v)));
        }
        const f32x2 in =
            add2(pair_of(pd, k), pair(sm.bias[io_v * P + k], sm.bias[io_v * P + k + 1]));
        const float2 s = halves(t < stop ? scan_step2(in, a.softplus) : 0), g = halves(g2);
        sm.step[io_t][k * S::kIo + io_v] = make_float2(s.x, g.x);
        sm.step[io_t][(k + 1) * S::kIo + io_v] = make_float2(s.y, g.y);
      }
    }
    for (int i = tid; i < kPacks; i += S::kThreads) {
      const int q = i / (S::kStates / 4), n1 = i % (S::kStates / 4) * 4;
      widen4(&sm.C[q][n1], &raw.c[q][n1]);
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
        carry[j][0] = mul2(decay2(A2[j][0], s), fma2(g, cn.x, carry[j][0]));
        carry[j][1] = mul2(decay2(A2[j][1], s), fma2(g, cn.y, carry[j][1]));
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
using Back8 = BackShape<2, 2, 64>;
using Back16 = BackShape<4, 2, 64>;
using Back32 = BackShape<8, 2, 64>;
using Back64 = BackShape<16, 2, 32>;
#define SALT_BACK_SHAPE(state, S, ...) \
  SALT_BY_STATE(state, S, Back4, Back8, Back16, Back32, Back64, __VA_ARGS__)
int back_channels(int32_t state) {
  return state <= 8    ? Back8::kChannels
         : state <= 16 ? Back16::kChannels
         : state <= 32 ? Back32::kChannels
                       : Back64::kChannels;
}

// As in the forward pass both constants are those of 9 to 16 states in 16 bits.  In 32 bits two of the
// blocks fit an SM, yet counting two took 245 us instead of 224 for 3 ragged rows of 1021 x 1002 x
// 12, 896 instead of 861 for 4 x 2048 x 2048 x 16 and 218 instead of 253 for one row of 2048 x 1536.
// Of 17 states and more one block fits.  Forward and backward of 4 rows of 2048 tokens x 2048
// channels in bf16: 506, 630, 1390 and 2790 us at 4, 8, 32 and 64 states.
constexpr int kSlots = 148 * 3;      // blocks of 128 threads at 168 registers
constexpr float kFirstPass = 0.22f;  // its time, of the second pass's

template <typename T, class S, int COPY>
cudaError_t back_launch(const salt_selective_scan_backward_args& a, const ScanSplit& sp,
                        const BackParts& parts, int blocks, bool svec, cudaStream_t st,
                        int* launches) {
  constexpr size_t shared = sizeof(BackShared<T, S>), few = sizeof(BackStateShared<T, S>);
  const auto first = scan_back_state_kernel<T, S, COPY>;
  const auto main = selective_scan_backward_kernel<T, S, COPY>;
  const auto limit = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaSuccess;
  if (shared > 48 * 1024) e = cudaFuncSetAttribute(main, limit, (int)shared);
  if (few > 48 * 1024 && e == cudaSuccess) e = cudaFuncSetAttribute(first, limit, (int)few);
  const int64_t rows = (int64_t)a.batch * blocks;
  if (e == cudaSuccess && sp.chunks > 1) {
    first<<<(unsigned)(rows * (sp.chunks - 1)), S::kThreads, few, st>>>(a, sp, blocks, svec);
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
  size_t state, steps, BC, sums, bytes;  // offsets in floats, and the whole in bytes
};

BackPlan back_plan(const salt_selective_scan_backward_args& a) {
  BackPlan p;
  p.blocks = scan_blocks(a.dim, a.groups, back_channels(a.state));
  const ScanSplit split = scan_split((int64_t)a.batch * p.blocks, kSlots, a.len, kFirstPass);
  p.chunks = split.chunks, p.chunk_len = split.chunk_len;
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
  p.sums = take(rows * (a.state + 2));
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
  const BackParts parts{base + p.BC, base + p.sums, p.blocks / a.groups};
  const size_t ts = type_size(a.type);
  // the widest copies that no row's start and end stand against
  auto fits = [&](int64_t bytes) {
    const int64_t few = std::min<int64_t>(bytes, 4 * ts);
    const int pack = a.state <= 8 ? Back4::P : kVec;  // channels of the largest pack
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
  if (e == cudaSuccess) {
    const int64_t dim = a.dim;
    e = sum_parts_launch(parts.sums, (int64_t)a.batch * p.chunks,
                         PartSums{dim * a.state, dim, dim, a.dA, a.dD, a.ddelta_bias, 0}, st);
    ++*launches;
  }
  return e;
}

}  // namespace salt
