// Linear attention with a decay for each head: rows, single tokens, gradients.
//
// All gradients are the operator itself over other arguments: dq over (dout, v, k) in the row's
// order, dk and dv over (v, dout, q) and (k, q, dout) against it.  One pass computes
//   forward:  S = l S + k v^T;  out = scale * q S
//   reverse:  D = C + beta * k v^T;  out = q D;  C = l D   (from the row's end; C starts as given)
#include <type_traits>

#include "sequence.cuh"
#include "tc.cuh"

namespace salt {
namespace {

struct Pass {
  int q_share, k_share, v_share;  // heads that read one head of an array
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
  // set by the launch
  int segments, seg_chunks;  // segments of a row that run side by side, chunks of each
  float* seg_states;         // (batch, heads, segments, dk, dv): what each adds to the state
  bool copies_out;
};

__device__ __forceinline__ float decay_of(const float* g, int h) {
  const float v = g[h];
  return v > 0.f ? 0.f : v < -200.f ? -200.f : v;  // a NaN stays one
}

constexpr int kTile = 64;      // columns of v that a block takes
constexpr int kWorkers = 512;  // 16 warps: four for each 32 rows of tensor memory
constexpr int kThreads = kWorkers + 32;  // and one for the copies and the products
constexpr int kParts = 3;      // of what is computed in 32 bits: a weighted v, a state, a weight in a chunk

// A type's values in parts of bfloat16, 8 bits each: what the tensor cores multiply.
template <typename T>
constexpr int parts_of() { return sizeof(T) == 4 ? 3 : std::is_same<T, __half>::value ? 2 : 1; }
// Tokens of a chunk: 64 where 128 do not fit into shared memory.
constexpr int chunk_of(int parts, int panels) {
  return parts == 1 || (parts == 2 && panels == 1) ? 128 : 64;
}

// Shared memory, all operands in rows of 128 bytes (tc::operand): q and k in panels of 64 columns,
// part after part; k and v twice, for copies a chunk further ahead, where there is room.  A chunk's
// outputs leave through memory of their own, or, where that does not fit (bfloat16 heads over 64), through
// the chunk's values, which no product reads any more.
template <int P, int PANELS, typename O>
struct Layout {
  static constexpr int C = chunk_of(P, PANELS), B = P == 3 || (P == 2 && C == 128) ? 1 : 2;
  static constexpr int kPanel = C * 128, kKeys = P * PANELS * kPanel, kValues = P * kPanel;
  static constexpr int kState = PANELS * 64 * 128;  // a part of the state
  // a warp's 32 rows of out, 32 bytes each at a time
  static constexpr int kStaged = 1024, kOutColumns = 32 / sizeof(O), kOut = kWorkers / 32 * kStaged;
  static constexpr bool out_in_values = P == 1 && PANELS == 2;
  static_assert(!out_in_values || (B == 2 && kValues == kOut), "outputs through the values' place");
  static constexpr int q = 0, k = q + kKeys, v = k + B * kKeys, weighted = v + B * kValues,
                       state = weighted + kParts * kPanel, out = state + kParts * kState,
                       bytes = out + (out_in_values ? 0 : kOut) + 1024;
  // the pass that wants the states alone has weighted values of two chunks instead
  static constexpr int state_bytes = weighted + 2 * kParts * kPanel + 1024;
  static_assert(bytes <= 225 * 1024 && state_bytes <= 225 * 1024, "2 KB are the kernel's own");
};

// The next part of two values, their upper 8 bits each, taken out of them.  (The sign goes over with the
// upper bits.)
__device__ __forceinline__ uint32_t next_part(f32x2& v) {
  const float2 x = halves(v);
  v = add2(v, pair(__uint_as_float((__float_as_uint(x.x) & 0xffff0000u) ^ 0x80000000u),
                   __uint_as_float((__float_as_uint(x.y) & 0xffff0000u) ^ 0x80000000u)));
  return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
}
// Two values in parts of bfloat16: one holds bfloat16's 8 bits, two float16's 11, three all 24.
template <int N>
__device__ __forceinline__ void split2(uint32_t (&to)[N], f32x2 v) {
#pragma unroll
  for (int i = 0; i < N; ++i) to[i] = next_part(v);
}
template <int N>
__device__ __forceinline__ void split2(uint32_t (&to)[N], float x, float y) {
  split2<N>(to, pair(x, y));
}
// Arrays (batch, len, heads, dim) of T in planes of bfloat16 parts (part, batch, len, heads, dim rounded
// up to 8), zero past the rows' ends: what tensor copies can take of every type, alignment and size.
// blockIdx.y is the array.  Bound by memory.
struct ToPlanes {
  const void* from;
  int64_t batch_stride, stride;
  uint4* to;
  int heads, dim;
  bool vec;
};
struct AllToPlanes {
  ToPlanes a[4];
};
template <typename T>
__global__ void __launch_bounds__(256) planes_kernel(const AllToPlanes all, int batch, int len,
                                                     const int32_t* n_real) {
  tc::let_next_begin();
  tc::wait_for_earlier();
  constexpr int P = parts_of<T>();
  const ToPlanes x = all.a[blockIdx.y];
  const int units = (x.dim + 7) / 8, each = x.heads * units;
  const int64_t n = (int64_t)batch * len * each;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t token = n >> 32 ? i / each : (unsigned)i / (unsigned)each;
    const int in = (int)(i - token * each), h = in / units, at = (in - h * units) * 8;
    const int b = (int)(n >> 32 ? token / len : (unsigned)token / (unsigned)len);
    const int t = (int)(token - (int64_t)b * len);
    const Pack<T, 8> p = load_pack<T, 8>(
        static_cast<const T*>(x.from) + b * x.batch_stride + t * x.stride + (int64_t)h * x.dim + at,
        t < row_tokens(n_real, b, len) ? x.dim - at : 0, x.vec);
    uint32_t parts[4][P];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2<P>(parts[k], to_f32(p.v[2 * k]), to_f32(p.v[2 * k + 1]));
#pragma unroll
    for (int j = 0; j < P; ++j)
      x.to[j * n + i] = make_uint4(parts[0][j], parts[1][j], parts[2][j], parts[3][j]);
  }
}

// One pass over chunks of C tokens (natural order; from the last one where `reverse`):
//   out = row weight * (q S) + (q k^T under a triangle of decays) v;
//   S = l^tokens S + k^T (weights * v)
// as four products of the tensor cores.  Per chunk and head, with c = C tokens: 2 c^2 dk + 2 c^2 dv +
// 4 c dk dv operations, against the 5 dk dv a token of the recurrence itself.
//
// A block has a row's head and 64 columns of v.  Sixteen warps write operands and take results, one warp
// copies and multiplies:
//   values' weights -> [q S, k^T (weights v)] -> the state -> the next chunk's values' weights
//   [q k^T] -> triangle -> [its product with v] -> out, a chunk behind
//
// What is rounded: every operand is bfloat16, in parts of 8 bits.  Inputs are exact (bfloat16 in one
// part, float16 in two, float32 in three); what is computed in 32 bits, the weighted values, states and
// the triangle, has three parts, which hold its 24 bits, whatever the outputs' type (two for outputs of
// 16 bits took 125 us instead of 141 below, and lost what is left where an output's terms cancel).  Sums
// and states are float32; the state is carried in registers.  The tensor cores cut their sums off after
// every instruction, so the parts'
// products go from the smallest to the largest: in the other order float32's outputs were off by 2.5e-6
// instead of 3.5e-7.
//
// What bounds it: the threads' work on operands.  8 rows of 2048 x 16 heads of 128 in bfloat16 take 141
// us, 2.0 TB/s, 3.3 times their bytes' time: 256 blocks are two rounds of 16 chunks of some 8000 cycles,
// of which the tensor cores work 3500 (an instruction of 128 x 64 x 16 takes 48 cycles, 30 with an
// operand in tensor memory), and an instruction issues in every other cycle.  One row of 32768 takes 346
// us: 9 segments, 98 of it the states' pass.  float16 heads of 128 and float32 have chunks of 64 tokens,
// since shared memory holds no more of their parts: the long row in float16 takes 880 us, in float32 1265.
// 17 warps leave 96 registers to a thread, and most instances keep some values in local memory: 4 and 24
// bytes for bfloat16 heads up to 64 and over, 28 for float16 heads over 64, 56 and 104 for float32.
// A call's kernels set themselves up while the one in front ends (tc::follow): a backward pass of 10
// small launches (3 x 1021 x 12 heads of 64 x 100, 4 key heads, float16; 166 us) gained 20 us.
// Measured and left: eight warps (269 us when sixteen took 189), all products' warps in step with the
// others (189 us when this was 133), roles for the warps, eight for triangle and out, four for the state
// and four for the values (180 us when this was 139: four warps wait too long for their own
// instructions), the direction as a template parameter (5 % for heads of 100 x 77, 1 % slower for heads
// of 128 backward).
template <int P, typename O, int PANELS, bool STATE>
__global__ void __launch_bounds__(kThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_out, const Pass a) {
  using L = Layout<P, PANELS, O>;
  constexpr int C = L::C, B = L::B, DK = PANELS * 64;
  constexpr int VB = STATE ? B + PANELS : B;  // places for values, also where q is not needed
  constexpr int kPanel = L::kPanel;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = raw + (1024 - tc::shared_at(raw) % 1024) % 1024;
  __shared__ uint64_t loaded_q, loaded_k[B], loaded_v[VB];  // copies
  // Products, and operands that threads wrote.  (Who waits at a barrier has to see every phase of it:
  // the next one ends only after all of them went on.  STATE runs a chunk ahead of its products, and
  // takes two barriers in turn.)
  constexpr int R = STATE ? 2 : 1;
  __shared__ uint64_t done_scores, done_q, done_state[R], done_out, ready_chunk[R], ready_triangle;
  __shared__ uint64_t out_gone;  // out_in_values: the outputs of the chunk in front left the values' place
  __shared__ uint64_t drained;  // every product issued
  __shared__ uint32_t tmem_at, gave_up;
  __shared__ float powers[32 + C + 1];        // l^i from place 32 on
  __shared__ __align__(16) float column[32];  // of a column within its 32
  __shared__ int bad[3][kTile];               // the outermost token whose v is not finite
  __shared__ int any_bad[3];
  float* power = powers + 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;

  const int tiles = (a.dv + kTile - 1) / kTile;
  int id = blockIdx.x;
  const int tile = id % tiles;
  id /= tiles;
  const int seg = id % a.segments, bh = id / a.segments, b = bh / a.heads, h = bh - b * a.heads;
  const int n = row_tokens(a.n_real, b, a.len), chunks = (n + C - 1) / C;
  const int c0 = min(seg * a.seg_chunks, chunks);
  // (nobody needs what the last segment alone adds to the state)
  const bool needed = !STATE || seg != (a.reverse ? 0 : a.segments - 1);
  const int c1 = needed ? min(c0 + a.seg_chunks, chunks) : c0, steps = c1 - c0;
  const int col0 = tile * kTile, cols = min(kTile, a.dv - col0);
  const float g = decay_of(a.log_decay, h) * kLog2e;
  const int64_t state_at = (int64_t)bh * a.dk * a.dv;
  const auto chunk = [&](int i) { return a.reverse ? c1 - 1 - i : c0 + i; };
  const auto tokens = [&](int c) { return min(C, n - c * C); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < B; ++i) tc::barrier_init(&loaded_k[i], 1);
    for (int i = 0; i < VB; ++i) tc::barrier_init(&loaded_v[i], 1);
    for (uint64_t* x : {&loaded_q, &done_q, &done_scores, &done_out, &drained})
      tc::barrier_init(x, 1);
    for (int i = 0; i < R; ++i) {
      tc::barrier_init(&done_state[i], 1);
      tc::barrier_init(&ready_chunk[i], kWorkers / 32);
    }
    tc::barrier_init(&ready_triangle, kWorkers / 32);
    tc::barrier_init(&out_gone, kWorkers / 32);
    gave_up = 0;
    tc::barrier_init_fence();
  }
  if (warp == 0) tc::tmem_alloc(&tmem_at, 512);
  for (int i = (int)threadIdx.x - 32; i <= C; i += kThreads)
    power[i] = i <= 0 ? 1.f : exp2f(g * (float)i);  // (in front of place 0: any number)
  if (threadIdx.x < 32) {
    const int i = a.reverse ? threadIdx.x : 31 - threadIdx.x;
    column[threadIdx.x] = i == 0 ? 1.f : exp2f(g * (float)i);
  }
  for (int i = threadIdx.x; i < 3 * kTile; i += kThreads) bad[i / kTile][i % kTile] = -1;
  if (threadIdx.x < 3) any_bad[threadIdx.x] = 0;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  tc::let_next_begin();
  tc::wait_for_earlier();
  const uint32_t tmem = tmem_at, mine = tmem + ((uint32_t)(quarter * 32) << 16);
  // columns of tensor memory
  constexpr int kScores = 0, kTriangle = 128, kFromState = 256, kOut = 384, kAdded = 448;
  const auto added = [&](int i) { return STATE ? (i & 1) * kTile : kAdded; };
  // Parts of chunk i's triangle.  With 128 tokens the third lies where the outputs from the state of the
  // chunk in front were: each warp has read its columns of them before it writes the same ones.
  constexpr bool kAway = C == 128;
  const auto triangle = [&](int i, int x) {
    return kAway && x == 2 ? kFromState + (~i & 1) * kTile : kTriangle + x * (C / 2);
  };
  const auto value_place = [&](int i) {
    return i % VB < B ? L::v + i % VB * L::kValues : L::q + (i % VB - B) * L::kValues;
  };
  const auto values = [&](int i) { return STATE ? (i & 1) * kParts * kPanel : 0; };
  uint32_t tries = tc::kTries;

  if (warp == kWorkers / 32) {
    if (tc::one_lane() && steps > 0) {
      const auto fetch = [&](int to, const CUtensorMap* map, int panels, int col, int head, int i,
                             uint64_t* barrier) {
        tc::barrier_expect(barrier, P * panels * kPanel);
        for (int x = 0; x < P * panels; ++x)
          tc::load_box4(sm + to + x * kPanel, map, col + x % panels * 64, head, chunk(i) * C,
                        x / panels * a.batch + b, barrier);
      };
      int asked_q = 0, asked_k = 0, asked_v = 0;  // chunks so far
      const auto fetch_q = [&](int i) {
        if (i < steps) fetch(L::q, &map_q, PANELS, 0, h / a.q_share, i, &loaded_q), ++asked_q;
      };
      const auto fetch_k = [&](int i) {
        if (i < steps)
          fetch(L::k + i % B * L::kKeys, &map_k, PANELS, 0, h / a.k_share, i, &loaded_k[i % B]),
              ++asked_k;
      };
      const auto fetch_v = [&](int i) {
        if (i < steps)
          fetch(value_place(i), &map_v, 1, col0, h / a.v_share, i, &loaded_v[i % VB]), ++asked_v;
      };
      const auto wait = [&](uint64_t* barrier, uint32_t parity) {
        tc::barrier_wait(barrier, parity, tries, &gave_up);
        return tries > 0;
      };
      const int depth = (a.dk + 15) / 16;
      const uint64_t q = tc::operand(sm + L::q, 1024), state = tc::operand(sm + L::state, 1024),
                     weighted = tc::operand(sm + L::weighted, 1024);
      const auto scores = [&](int i) {
        const uint64_t k = tc::operand(sm + L::k + i % B * L::kKeys, 1024);
        bool add = false;
#pragma unroll
        for (int o = 2; o >= 0; --o)
#pragma unroll
          for (int x = 0; x < P; ++x) {
            const int y = o - x;
            if (y < 0 || y >= P) continue;
            for (int d = 0; d < depth; ++d) {
              const uint32_t off = (d >> 2) * kPanel + (d & 3) * 32;
              tc::product_16(tmem + kScores, tc::further(q, x * PANELS * kPanel + off),
                             tc::further(k, y * PANELS * kPanel + off), tc::shape(128, C, 1), add);
              add = true;
            }
          }
        tc::products_done(&done_scores);
      };
      const auto work = [&] {  // until a wait is given up
        for (int i = 0; i < VB; ++i) {
          fetch_v(i);
          if (i < B) fetch_k(i);
          if (!STATE && i == 0) fetch_q(0);
        }
        if (!wait(&loaded_k[0], 0)) return;
        if (!STATE) {
          if (!wait(&loaded_q, 0)) return;
          scores(0);
        }
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
          if (!wait(&ready_chunk[i % R], i / R & 1)) return;
          tc::fence_after();
          if (STATE) fetch_v(i + VB);
          if (!STATE) {
            bool add = false;
#pragma unroll
            for (int o = 2; o >= 0; --o)
#pragma unroll
              for (int x = 0; x < P; ++x) {
                const int y = o - x;
                if (y < 0 || y >= kParts) continue;
                for (int d = 0; d < depth; ++d) {
                  const uint32_t off = (d >> 2) * kPanel + (d & 3) * 32;
                  tc::product_16(tmem + kFromState + (i & 1) * kTile,
                                 tc::further(q, x * PANELS * kPanel + off),
                                 tc::further(state, y * L::kState + d * 2048),
                                 tc::shape(128, kTile, 1, false, true), add);
                  add = true;
                }
              }
            tc::products_done(&done_q);
          }
          {
            const uint64_t k = tc::operand(sm + L::k + i % B * L::kKeys, 1024, kPanel);
            bool add = false;
#pragma unroll
            for (int o = 2; o >= 0; --o)
#pragma unroll
              for (int x = 0; x < P; ++x) {
                const int y = o - x;
                if (y < 0 || y >= kParts) continue;
#pragma unroll
                for (int d = 0; d < C / 16; ++d) {
                  tc::product_16(tmem + added(i), tc::further(k, x * PANELS * kPanel + d * 2048),
                                 tc::further(weighted, values(i) + y * kPanel + d * 2048),
                                 tc::shape(128, kTile, 1, true, true), add);
                  add = true;
                }
              }
            tc::products_done(&done_state[i % R]);
          }
          if (!STATE) {
            if (!wait(&done_q, i & 1)) return;
            fetch_q(i + 1);
            if (L::out_in_values && i > 0) {
              if (!wait(&out_gone, (i - 1) & 1)) return;
              fetch_v(i + 1);
            }
            if (!wait(&ready_triangle, i & 1)) return;
            tc::fence_after();
            const uint64_t v = tc::operand(sm + L::v + i % B * L::kValues, 1024);
            bool add = false;
#pragma unroll
            for (int o = 2; o >= 0; --o)
#pragma unroll
              for (int x = 0; x < kParts; ++x) {
                const int y = o - x;
                if (y < 0 || y >= P) continue;
#pragma unroll
                for (int d = 0; d < C / 16; ++d) {
                  tc::product_16_from_tmem(tmem + kOut, tmem + triangle(i, x) + d * 8,
                                           tc::further(v, y * kPanel + d * 2048),
                                           tc::shape(128, kTile, 1, false, true), add);
                  add = true;
                }
              }
            tc::products_done(&done_out);
          }
          if (i + 1 == steps) break;
          const auto next = [&] {
            if (!wait(&loaded_k[(i + 1) % B], (i + 1) / B & 1)) return false;
            if (STATE) return true;
            if (!wait(&loaded_q, (i + 1) & 1)) return false;
            scores(i + 1);
            return true;
          };
          if (B == 2 && !next()) return;
          if (!wait(&done_state[i % R], i / R & 1)) return;
          fetch_k(i + B);
          if (!STATE) {
            if (!wait(&done_out, i & 1)) return;
            if (!L::out_in_values) fetch_v(i + B);
          }
          if (B == 1 && !next()) return;
        }
      };
      work();
      // nothing may be under way when the block ends
      uint32_t more = tc::kTries;
      tc::products_done(&drained);
      tc::barrier_wait(&drained, 0, more, &gave_up);
      if (tc::marked(&gave_up)) {
        for (int i = max(0, asked_v - VB); i < asked_v; ++i)
          tc::barrier_wait(&loaded_v[i % VB], i / VB & 1, more, &gave_up);
        for (int i = max(0, asked_k - B); i < asked_k; ++i)
          tc::barrier_wait(&loaded_k[i % B], i / B & 1, more, &gave_up);
        if (asked_q > 0) tc::barrier_wait(&loaded_q, (asked_q - 1) & 1, more, &gave_up);
      }
    }
    __syncwarp();
  } else {
    // this thread's part of the state: row `row`, 16 columns
    f32x2 s[8];
    const int sc0 = col0 + part * 16;
    const bool joined = a.segments > 1 && !STATE;
    const float* from =
        joined ? a.seg_states + ((int64_t)bh * a.segments + seg) * a.dk * a.dv
               : a.initial ? a.initial + state_at : nullptr;
    const bool across = a.initial_t && !joined;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const auto load = [&](int c) {
        return from && row < a.dk && c < a.dv
                   ? from[across ? (int64_t)c * a.dk + row : (int64_t)row * a.dv + c]
                   : 0.f;
      };
      s[j / 2] = pair(load(sc0 + j), load(sc0 + j + 1));
    }
    const auto store_state = [&] {  // as an operand
      if (row >= DK) return;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t x[4][kParts];
#pragma unroll
        for (int k = 0; k < 4; ++k) split2<kParts>(x[k], s[4 * u + k]);
#pragma unroll
        for (int j = 0; j < kParts; ++j)
          *reinterpret_cast<uint4*>(sm + L::state + j * L::kState + row * 128 +
                                    (((part * 2 + u) ^ (row & 7)) << 4)) =
              make_uint4(x[0][j], x[1][j], x[2][j], x[3][j]);
      }
    };
    if (!STATE && steps > 0) store_state();

    // Chunk i's operands: rows past the end made zero, values weighted.
    const auto begin = [&](int i) {
      const int count = tokens(chunk(i));
      uint8_t* k = sm + L::k + i % B * L::kKeys;
      uint8_t* v = sm + value_place(i);
      tc::barrier_wait_warp(&loaded_v[i % VB], i / VB & 1, tries, &gave_up);
      if (P == 1 && count < C) {  // (planes hold zeros there)
        tc::barrier_wait_warp(&loaded_k[i % B], i / B & 1, tries, &gave_up);
        for (int x = threadIdx.x; x < (C - count) * PANELS * 8; x += kWorkers) {
          const int r = count + x / (PANELS * 8), u = x % (PANELS * 8);
          *reinterpret_cast<uint4*>(k + (u >> 3) * kPanel + r * 128 + ((u & 7) << 4)) =
              make_uint4(0, 0, 0, 0);
        }
      }
      // A thread has the same 8 columns of N rows; all of its loads go out before its first store.
      constexpr int N = C * 8 / kWorkers, kApart = kWorkers / 8;
      const int r0 = threadIdx.x >> 3, u = threadIdx.x & 7;
      uint8_t* place = v + r0 * 128 + ((u ^ (r0 & 7)) << 4);  // kApart is a multiple of 8
      uint32_t in[N][P][4], carry = 0;  // (carry: from an exponent of all ones)
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const uint4 y = *reinterpret_cast<const uint4*>(place + x * kApart * 128 + j * kPanel);
          in[x][j][0] = y.x, in[x][j][1] = y.y, in[x][j][2] = y.z, in[x][j][3] = y.w;
        }
      if (count < C) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
          if (r0 + x * kApart < count) continue;
#pragma unroll
          for (int j = 0; j < P; ++j) {
            in[x][j][0] = in[x][j][1] = in[x][j][2] = in[x][j][3] = 0;
            *reinterpret_cast<uint4*>(place + x * kApart * 128 + j * kPanel) =
                make_uint4(0, 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int m = 0; m < 4; ++m) carry |= (in[x][0][m] & 0x7f807f80u) + 0x00800080u;
      if (carry & 0x80008000u) {
        // A value that is not finite would reach the tokens on the triangle's other side, as 0 * it:
        // it becomes zero here, and its column NaN from its token on.
        any_bad[i % 3] = 1;
#pragma unroll
        for (int x = 0; x < N; ++x) {
          const int r = r0 + x * kApart;
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            const uint32_t mask = 0xffffu << (m & 1) * 16, exponent = 0x7f80u << (m & 1) * 16;
            if ((in[x][0][m / 2] & exponent) != exponent) continue;
            atomicMax(&bad[i % 3][u * 8 + m], a.reverse ? r : C - 1 - r);
#pragma unroll
            for (int j = 0; j < P; ++j) in[x][j][m / 2] &= ~mask;
          }
#pragma unroll
          for (int j = 0; j < P; ++j)
            *reinterpret_cast<uint4*>(place + x * kApart * 128 + j * kPanel) =
                make_uint4(in[x][j][0], in[x][j][1], in[x][j][2], in[x][j][3]);
        }
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const int r = r0 + x * kApart;
        // (rows past the end are zero, whatever their weight; power has 32 places in front)
        const float w = power[a.reverse ? r + 1 : max(count - 1 - r, 0)];
        uint32_t out[4][kParts];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          f32x2 y = 0;
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const f32x2 one = pair(__uint_as_float(in[x][j][m] << 16),
                                   __uint_as_float(in[x][j][m] & 0xffff0000u));
            y = j == 0 ? one : add2(y, one);
          }
          split2<kParts>(out[m], mul2(y, both(w)));
        }
        uint8_t* to = sm + L::weighted + values(i) + (place - v) + x * kApart * 128;
#pragma unroll
        for (int j = 0; j < kParts; ++j)
          *reinterpret_cast<uint4*>(to + j * kPanel) =
              make_uint4(out[0][j], out[1][j], out[2][j], out[3][j]);
      }
      tc::fence_shared();
      tc::fence_before();
      __syncwarp();
      tc::barrier_arrive_if_zero(&ready_chunk[i % R], lane);
    };
    // Chunk i's output, once its products are there.
    const auto finish = [&](int i) {
      const int c = chunk(i), count = tokens(c);
      tc::barrier_wait_warp(&done_out, i & 1, tries, &gave_up);
      tc::fence_after();
      uint32_t x[16], y[16];
      tc::tmem_load<16>(x, mine + kFromState + (i & 1) * kTile + part * 16);
      tc::tmem_load<16>(y, mine + kOut + part * 16);
      tc::loads_done();
      const bool live = row < count;
      const float by = !live ? 0.f : a.reverse ? power[count - 1 - row] : a.scale * power[row + 1];
      float f[16];
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const float2 o =
            halves(fma2(pair(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), both(by),
                        mul2(pair(__uint_as_float(y[j]), __uint_as_float(y[j + 1])), both(a.scale))));
        f[j] = live ? o.x : 0.f, f[j + 1] = live ? o.y : 0.f;
      }
      const bool lost = tc::marked(&gave_up);  // a result that nobody can take for one
      if (any_bad[i % 3] || lost) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int first = bad[i % 3][part * 16 + j];
          if (live && ((first >= 0 && (a.reverse ? row <= first : row >= C - 1 - first)) || lost))
            f[j] = __int_as_float(0x7fffffff);
        }
      }
      // 32 bytes a row, through shared memory: as stores from here every 16 bytes would be a line of
      // their own
      constexpr int W = L::kOutColumns;
      O* to = reinterpret_cast<O*>(sm + (L::out_in_values ? value_place(i) : L::out) +
                                   warp * L::kStaged);
#pragma unroll
      for (int y = 0; y < 16; y += W) {
        if (a.copies_out && lane == 0) tc::stores_read();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < W; j += 8) store_pack<O, 8>(to + lane * W + j, f + y + j, 8, true);
        if (a.copies_out) {
          // rows past the end are zero anyway; those past `len` are left out
          tc::fence_shared();
          __syncwarp();
          if (lane == 0 && quarter * 32 < min(C, a.len - c * C) && sc0 + y < a.dv)
            tc::store_box4(&map_out, to, sc0 + y, h, c * C + quarter * 32, b);
        } else {
          __syncwarp();
          const int col = lane % W;
          O* out = static_cast<O*>(a.out) + b * a.out_batch + (int64_t)h * a.dv + sc0 + y + col;
          if (sc0 + y + col < a.dv) {
            for (int r = lane / W; r < min(32, count - quarter * 32); r += 32 / W)
              out[((int64_t)c * C + quarter * 32 + r) * a.out_token] = to[r * W + col];
          }
        }
      }
    };

    // The chunk in front's outputs are on their way out of the values' place.
    const auto leave_values = [&] {
      if (!L::out_in_values) return;
      if (a.copies_out) {
        if (lane == 0) tc::stores_read();
      } else {
        tc::fence_shared();
      }
      __syncwarp();
      tc::barrier_arrive_if_zero(&out_gone, lane);
    };

    if (STATE && steps > 0) begin(0);
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const int count = tokens(chunk(i));
      if (!STATE)
        begin(i);
      else if (i + 1 < steps)
        begin(i + 1);  // while this chunk's product runs
      if (!STATE) {
        if (i > 0) finish(i - 1);
        // the triangle's weights
        tc::barrier_wait_warp(&done_scores, i & 1, tries, &gave_up);
        tc::fence_after();
        // blocks on the other side hold the zeros that the first chunk left there (but a part away)
        const bool beside = a.reverse ? part < quarter : part > quarter;
        if (part < C / 32 && quarter < C / 32) {
          const bool none = beside || (a.reverse && part * 32 >= count);
          const bool diagonal = part == quarter;
          // against time, columns past the end lie on the triangle's side
          const bool cut = a.reverse && part * 32 + 32 > count;
          const float f = none || diagonal || cut
                              ? 0.f
                              : power[a.reverse ? part * 32 - row : row - part * 32 - 31];
          // (as a loop: unrolled, 8 x 2048 x 16 heads of 128 took 145 us instead of 141)
#pragma unroll 1
          for (int y = 0; y < 32; y += 16) {
            f32x2 x[8];
            if (none) {
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = 0;
            } else {
              uint32_t r[16];
              tc::tmem_load<16>(r, mine + kScores + part * 32 + y);
              tc::loads_done();
              if (cut) {
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                  const int at = part * 32 + y + j, d = at - row;
                  const float w0 = power[max(d, 0)], w1 = power[max(d + 1, 0)];
                  x[j / 2] = pair(d >= 0 && at < count ? __uint_as_float(r[j]) * w0 : 0.f,
                                  d >= -1 && at + 1 < count ? __uint_as_float(r[j + 1]) * w1 : 0.f);
                }
              } else if (diagonal) {
                // (weights of the other side are loaded and left: a branch a value would cost more)
                const float* w = a.reverse ? power - lane + y : power + lane - y;
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                  const int c0 = y + j, c1 = c0 + 1;
                  const float p0 = __uint_as_float(r[j]) * w[a.reverse ? j : -j],
                              p1 = __uint_as_float(r[j + 1]) * w[a.reverse ? j + 1 : -j - 1];
                  x[j / 2] = pair((a.reverse ? c0 >= lane : c0 <= lane) ? p0 : 0.f,
                                  (a.reverse ? c1 >= lane : c1 <= lane) ? p1 : 0.f);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const float4 w = *reinterpret_cast<const float4*>(column + y + j);
                  x[j / 2] = mul2(pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1])),
                                  mul2(pair(w.x, w.y), both(f)));
                  x[j / 2 + 1] = mul2(pair(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])),
                                      mul2(pair(w.z, w.w), both(f)));
                }
              }
            }
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
              if (beside && i > 0 && !(kAway && k == 2)) continue;
              uint32_t o[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = next_part(x[j]);
              tc::tmem_store(mine + triangle(i, k) + part * 16 + y / 2, o);
            }
            if (y == 0 && i > 0) leave_values();
          }
          tc::stores_to_tmem_done();
        }
        tc::fence_before();
        __syncwarp();
        tc::barrier_arrive_if_zero(&ready_triangle, lane);
      }
      // the state behind the chunk
      tc::barrier_wait_warp(&done_state[i % R], i / R & 1, tries, &gave_up);
      tc::fence_after();
      uint32_t x[16];
      tc::tmem_load<16>(x, mine + added(i) + part * 16);
      tc::loads_done();
      tc::fence_before();
      const float l = power[count], by = a.reverse ? a.scale : 1.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s[j] = fma2(s[j], both(l),
                    mul2(pair(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), both(by)));
      if (any_bad[i % 3]) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (bad[i % 3][part * 16 + j] < 0) continue;
          const float2 y = halves(s[j / 2]);
          const float nan = __int_as_float(0x7fffffff);
          s[j / 2] = j % 2 ? pair(y.x, nan) : pair(nan, y.y);
        }
      }
      if (i + 1 < steps) {
        if (!STATE) {
          tc::barrier_wait_warp(&done_q, i & 1, tries, &gave_up);
          store_state();
        }
        // every warp is past the chunk before (STATE: past this one): its marks are free
        tc::named_sync(1, kWorkers);
        constexpr int kFree = STATE ? 0 : 2;
        if (threadIdx.x < kTile) bad[(i + kFree) % 3][threadIdx.x] = -1;
        if (threadIdx.x == 0) any_bad[(i + kFree) % 3] = 0;
      }
    }
    // the state goes out while the last outputs' product runs
    const bool last = a.reverse ? seg == 0 : (c1 == chunks && (c0 < chunks || seg == 0));
    float* to = STATE ? a.seg_states + ((int64_t)bh * a.segments + seg) * a.dk * a.dv
                      : last && a.final ? a.final + state_at : nullptr;
    if (to && row < a.dk) {
      const float nan = __int_as_float(0x7fffffff);
      const bool lost = tc::marked(&gave_up);
      to += (int64_t)row * a.dv + sc0;
      if (sc0 + 16 <= a.dv && a.dv % 4 == 0 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float2 x = halves(s[j]), y = halves(s[j + 1]);
          reinterpret_cast<float4*>(to)[j / 2] =
              lost ? make_float4(nan, nan, nan, nan) : make_float4(x.x, x.y, y.x, y.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (sc0 + j < a.dv) {
            const float2 y = halves(s[j / 2]);
            to[j] = lost ? nan : j % 2 ? y.y : y.x;
          }
      }
    }
    if (!STATE && steps > 0) finish(steps - 1);
    if (!STATE && lane == 0) tc::stores_done();
    __syncwarp();
    if (!STATE) {
      // tokens behind the row's end
      const int end = min(a.len, (seg + 1) * a.seg_chunks * C);
      for (int64_t t = max(a.copies_out ? chunks * C : n, seg * a.seg_chunks * C) + warp; t < end;
           t += kWorkers / 32)
        for (int j = lane; j < cols; j += 32)
          static_cast<O*>(a.out)[b * a.out_batch + t * a.out_token + (int64_t)h * a.dv + col0 + j] =
              from_f32<O>(0.f);
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_free(tmem, 512);
  }
}

// The states in front of a row's segments, in place of what each adds from zero: one value a thread,
// from segment to segment (against time from the last one).
__global__ void __launch_bounds__(256) join_segments_kernel(const Pass a, int chunk) {
  tc::let_next_begin();
  tc::wait_for_earlier();
  const int each = a.dk * a.dv, i = blockIdx.x * 256 + threadIdx.x, bh = blockIdx.y;
  if (i >= each) return;
  const int b = bh / a.heads, n = row_tokens(a.n_real, b, a.len);
  const float g = decay_of(a.log_decay, bh - b * a.heads) * kLog2e;
  const int row = i / a.dv, col = i - row * a.dv;
  float s = a.initial ? a.initial[(int64_t)bh * each + (a.initial_t ? col * a.dk + row : i)] : 0.f;
  float* at = a.seg_states + (int64_t)bh * a.segments * each + i;
  const auto place = [&](int x) { return at + (int64_t)(a.reverse ? a.segments - 1 - x : x) * each; };
  for (int x0 = 0; x0 < a.segments; x0 += 8) {
    float added[8];  // (loaded before the first store, which the compiler would keep in front of them)
#pragma unroll
    for (int x = 0; x < 8; ++x) added[x] = x0 + x + 1 < a.segments ? *place(x0 + x) : 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      if (x0 + x >= a.segments) break;
      const int seg = a.reverse ? a.segments - 1 - x0 - x : x0 + x;
      const int first = seg * a.seg_chunks * chunk,
                count = min(first + a.seg_chunks * chunk, n) - first;
      *place(x0 + x) = s;
      if (count > 0) s = fmaf(s, exp2f(g * (float)count), added[x]);
    }
  }
}

// Adds up what the heads that share a key head gave: (batch, len, kv, share, dim) of float32 to
// (batch, len, kv, dim), in the heads' order.
template <typename T>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* from, T* to, int64_t tokens,
                                                        int len, int kv, int share, int dim,
                                                        int64_t to_batch, int64_t to_token) {
  tc::let_next_begin();
  tc::wait_for_earlier();
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

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// An array (batch, len, heads, dim) of the call, or its planes.
struct Array {
  const void* p;
  int64_t batch_stride, stride;  // in elements
  int heads, dim;
};

// Boxes of `high` tokens x `columns` of one head of an array of elements of `size` bytes, if tensor
// copies can take it.
bool head_map(CUtensorMap* map, const Array& x, size_t size, int len, int batch, int high, int columns,
              bool swizzled) {
  const tc::EncodeTiled f = tc::encoder();
  const int64_t token = len > 1 ? x.stride * (int64_t)size : 16,
                row = batch > 1 ? x.batch_stride * (int64_t)size : 16;
  if (!f || !aligned16(x.p) || x.dim * size % 16 || token % 16 || row % 16 || token < 16 || row < 16 ||
      token >= tc::kMostStride || row >= tc::kMostStride)
    return false;
  const cuuint64_t dims[4] = {(cuuint64_t)x.dim, (cuuint64_t)x.heads, (cuuint64_t)len,
                              (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)(x.dim * size), (cuuint64_t)token, (cuuint64_t)row};
  const cuuint32_t box[4] = {(cuuint32_t)columns, 1, (cuuint32_t)high, 1}, unit[4] = {1, 1, 1, 1};
  return f(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
           const_cast<void*>(x.p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
           swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
           CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The call's arrays as the pass takes them: bfloat16 as it lies where tensor copies can, else planes.
template <typename T>
bool as_it_lies(const Array& x, int len, int batch) {
  CUtensorMap map;
  return parts_of<T>() == 1 && head_map(&map, x, 2, len, batch, 128, 64, true);
}
template <typename T>
size_t planes_bytes(const Array& x, int len, int batch) {
  if (!len || !batch || as_it_lies<T>(x, len, batch)) return 0;
  return align256((size_t)parts_of<T>() * batch * len * x.heads * ((x.dim + 7) / 8) * 16);
}
template <typename T, int N>
cudaError_t take(Array* const (&all)[N], int len, int batch, const int32_t* n_real, uint8_t*& ws,
                 cudaStream_t st, int* launches) {
  AllToPlanes to = {};
  int count = 0;
  int64_t most = 0;
  for (Array* x : all) {
    if (!len || !batch || as_it_lies<T>(*x, len, batch)) continue;
    const size_t bytes = planes_bytes<T>(*x, len, batch);
    const int units = (x->dim + 7) / 8;
    to.a[count++] = {x->p, x->batch_stride, x->stride, reinterpret_cast<uint4*>(ws), x->heads, x->dim,
                     x->dim % 8 == 0 && pack_rows(x->p, 8, sizeof(T), x->batch_stride, x->stride)};
    most = std::max(most, (int64_t)batch * len * x->heads * units);
    x->p = ws;
    x->dim = units * 8;
    x->stride = (int64_t)x->heads * x->dim;
    x->batch_stride = x->stride * len;
    ws += bytes;
  }
  if (!count) return cudaSuccess;
  return tc::follow((*launches)++, planes_kernel<T>,
                    dim3((unsigned)std::min<int64_t>((most + 255) / 256, 148 * 8), count), 256, 0, st,
                    to, batch, len, n_real);
}

template <int P, typename O, int PANELS, bool STATE>
cudaError_t start(const CUtensorMap (&maps)[4], const Pass& p, int64_t blocks, cudaStream_t st,
                  int* launches) {
  const auto kernel = attention_kernel<P, O, PANELS, STATE>;
  constexpr int bytes = STATE ? Layout<P, PANELS, O>::state_bytes : Layout<P, PANELS, O>::bytes;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = tc::allow_shared(reinterpret_cast<const void*>(kernel), bytes, allowed);
  if (e != cudaSuccess) return e;
  return tc::follow((*launches)++, kernel, dim3((unsigned)blocks), kThreads, bytes, st, maps[0], maps[1],
                    maps[2], maps[3], p);
}

// Segments of a row: the number that needs the least time in rounds of resident blocks (one an SM),
// counted in chunks of the main pass.  A block takes about as long as a chunk to begin and end; the
// first pass, over all but the last segment, takes about half of a chunk's time for each, and with the
// joining of its states two more.
int segments_of(int64_t blocks, int chunks) {
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 64 && s <= chunks && blocks * s <= 148 * 8; ++s) {
    const int each = (chunks + s - 1) / s;
    const double rounds = (double)((blocks * s + 147) / 148);
    const double time = rounds * (each + 1) + (s > 1 ? rounds * (0.55 * each + 1) + 2 : 0);
    if (time < least) least = time, best = s;
  }
  return best;
}
template <typename T>
int pass_segments(int batch, int heads, int dk, int dv, int len) {
  const int C = chunk_of(parts_of<T>(), dk <= 64 ? 1 : 2);
  const int64_t blocks = (int64_t)batch * heads * ((dv + kTile - 1) / kTile);
  return blocks ? segments_of(blocks, (len + C - 1) / C) : 1;
}
template <typename T>
size_t segment_bytes(int batch, int heads, int dk, int dv, int len) {
  const int s = pass_segments<T>(batch, heads, dk, dv, len);
  return s == 1 ? 0 : align256(sizeof(float) * batch * heads * s * dk * dv);
}

template <int P, typename O, int PANELS>
cudaError_t run_panels(const CUtensorMap (&maps)[4], const Pass& p, int64_t blocks, cudaStream_t st,
                       int* launches) {
  if (p.segments > 1) {
    Pass first = p;
    first.initial = nullptr;
    // (nothing of out is touched: its type is any)
    cudaError_t e = start<P, float, PANELS, true>(maps, first, blocks * p.segments, st, launches);
    if (e != cudaSuccess) return e;
    // (rows and heads: at most 2^24, and where segments are used few)
    e = tc::follow((*launches)++, join_segments_kernel,
                   dim3((p.dk * p.dv + 255) / 256, p.batch * p.heads), 256, 0, st, p,
                   chunk_of(P, PANELS));
    if (e != cudaSuccess) return e;
  }
  return start<P, O, PANELS, false>(maps, p, blocks * p.segments, st, launches);
}

// One pass over arrays that `take` brought into shape; `ws` holds segment_bytes.
template <typename T, typename O>
cudaError_t run_pass(Pass p, const Array& q, const Array& k, const Array& v, void* ws, cudaStream_t st,
                     int* launches) {
  constexpr int P = parts_of<T>();
  const int C = chunk_of(P, p.dk <= 64 ? 1 : 2);
  const int64_t blocks = (int64_t)p.batch * p.heads * ((p.dv + kTile - 1) / kTile);
  if (!blocks) return cudaSuccess;
  p.q_share = p.heads / q.heads, p.k_share = p.heads / k.heads, p.v_share = p.heads / v.heads;
  const int chunks = (p.len + C - 1) / C;
  p.segments = pass_segments<T>(p.batch, p.heads, p.dk, p.dv, p.len);
  p.seg_chunks = std::max(1, (chunks + p.segments - 1) / p.segments);
  p.seg_states = static_cast<float*>(ws);
  CUtensorMap maps[4] = {};
  p.copies_out = false;
  if (p.len > 0) {
    if (!head_map(&maps[0], q, 2, p.len, p.batch * P, C, 64, true) ||
        !head_map(&maps[1], k, 2, p.len, p.batch * P, C, 64, true) ||
        !head_map(&maps[2], v, 2, p.len, p.batch * P, C, 64, true))
      return cudaErrorInvalidValue;
    p.copies_out = head_map(&maps[3], {p.out, p.out_batch, p.out_token, p.heads, p.dv}, sizeof(O),
                            p.len, p.batch, 32, 32 / sizeof(O), false);
  }
  return p.dk <= 64 ? run_panels<P, O, 1>(maps, p, blocks, st, launches)
                    : run_panels<P, O, 2>(maps, p, blocks, st, launches);
}

// One token of a row's head: S = l S + k v^T; out = scale * q S.  A block has a head; its 8 warps take
// every eighth row of the state, a lane four columns (side by side with VEC, 32 apart without), and all
// of a thread's loads go out before its first store, which the compiler may not put behind loads of the
// same array.  Bound by memory, 8 bytes a value of the state.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 2) attention_step_kernel(salt_linear_attention_step_args a) {
  __shared__ __align__(16) float parts[8][128];
  const int bh = blockIdx.x, b = bh / a.heads, h = bh - b * a.heads, share = a.heads / a.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = a.slots ? a.slots[b] : b;
  T* out = static_cast<T*>(a.out) + b * a.out_stride + (int64_t)h * a.dim_v;
  if (slot < 0 || slot >= a.n_slots) {  // the whole block
    if (threadIdx.x < a.dim_v) out[threadIdx.x] = from_f32<T>(0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)h * a.dim_k;
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride + (int64_t)(h / share) * a.dim_k;
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride + (int64_t)(h / share) * a.dim_v;
  float* s = a.pool + ((int64_t)slot * a.heads + h) * a.dim_k * a.dim_v;
  const auto column = [&](int j) { return VEC ? lane * 4 + j : lane + 32 * j; };
  float x[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = warp + 8 * i;
    if (VEC) {
      if (row < a.dim_k && lane * 4 < a.dim_v)
        *reinterpret_cast<float4*>(x[i]) =
            *reinterpret_cast<const float4*>(s + row * a.dim_v + lane * 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row < a.dim_k && column(j) < a.dim_v) x[i][j] = s[row * a.dim_v + column(j)];
    }
  }
  const float l = expf(decay_of(a.log_decay, h));
  float w[4], sum[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = column(j) < a.dim_v ? to_f32(v[column(j)]) : 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = warp + 8 * i;
    if (row >= a.dim_k) break;
    const float kr = to_f32(k[row]), qr = to_f32(q[row]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[i][j] = fmaf(l, x[i][j], kr * w[j]);
      sum[j] = fmaf(qr, x[i][j], sum[j]);
    }
    if (VEC) {
      if (lane * 4 < a.dim_v)
        *reinterpret_cast<float4*>(s + row * a.dim_v + lane * 4) = *reinterpret_cast<float4*>(x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (column(j) < a.dim_v) s[row * a.dim_v + column(j)] = x[i][j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) parts[warp][column(j)] = sum[j];
  __syncthreads();
  if (threadIdx.x < a.dim_v) {
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o += parts[i][threadIdx.x];
    out[threadIdx.x] = from_f32<T>(a.scale * o);
  }
}

struct Arrays {
  Array q, k, v, d;
};
template <class A>
Arrays arrays_of(const A& a) {
  return {{a.q, a.q_batch_stride, a.q_stride, a.heads, a.dim_k},
          {a.k, a.k_batch_stride, a.k_stride, a.kv_heads, a.dim_k},
          {a.v, a.v_batch_stride, a.v_stride, a.kv_heads, a.dim_v},
          {}};
}
Arrays arrays_of_backward(const salt_linear_attention_backward_args& a) {
  Arrays x = arrays_of(a);
  x.d = {a.dout, a.dout_batch_stride, a.dout_stride, a.heads, a.dim_v};
  return x;
}
template <typename T>
size_t forward_bytes(const salt_linear_attention_args& a) {
  const Arrays x = arrays_of(a);
  return planes_bytes<T>(x.q, a.len, a.batch) + planes_bytes<T>(x.k, a.len, a.batch) +
         planes_bytes<T>(x.v, a.len, a.batch) +
         segment_bytes<T>(a.batch, a.heads, a.dim_k, a.dim_v, a.len);
}
// Backward: planes, segments' states of one pass after the other, and what the heads that share a key
// head give to dk, then to dv.
template <typename T>
size_t backward_states(const salt_linear_attention_backward_args& a) {
  return std::max(segment_bytes<T>(a.batch, a.heads, a.dim_v, a.dim_k, a.len),
                  segment_bytes<T>(a.batch, a.heads, a.dim_k, a.dim_v, a.len));
}
template <typename T>
size_t backward_bytes(const salt_linear_attention_backward_args& a) {
  const Arrays x = arrays_of_backward(a);
  size_t n = backward_states<T>(a);
  for (const Array* y : {&x.q, &x.k, &x.v, &x.d}) n += planes_bytes<T>(*y, a.len, a.batch);
  if (a.heads != a.kv_heads)
    n += align256(sizeof(float) * a.batch * a.len * a.heads * std::max(a.dim_k, a.dim_v));
  return n;
}

template <typename T>
cudaError_t forward(const salt_linear_attention_args& a, uint8_t* ws, cudaStream_t st, int* launches) {
  Arrays x = arrays_of(a);
  const cudaError_t e = take<T, 3>({&x.q, &x.k, &x.v}, a.len, a.batch, a.n_real, ws, st, launches);
  if (e != cudaSuccess) return e;
  const Pass p{0, 0, 0, a.dim_k, a.dim_v, a.heads, a.len, a.batch, a.scale, false, a.log_decay,
               a.n_real, a.initial_state, false, a.out, a.out_batch_stride, a.out_stride,
               a.final_state};
  return run_pass<T, T>(p, x.q, x.k, x.v, ws, st, launches);
}

template <typename T>
cudaError_t backward(const salt_linear_attention_backward_args& a, uint8_t* ws, cudaStream_t st,
                     int* launches) {
  Arrays x = arrays_of_backward(a);
  cudaError_t e =
      take<T, 4>({&x.q, &x.k, &x.v, &x.d}, a.len, a.batch, a.n_real, ws, st, launches);
  if (e != cudaSuccess) return e;
  float* parts = reinterpret_cast<float*>(ws + backward_states<T>(a));
  const Pass dq{0, 0, 0, a.dim_v, a.dim_k, a.heads, a.len, a.batch, a.scale, false, a.log_decay,
                a.n_real, a.initial_state, true, a.dq, a.dq_batch_stride, a.dq_stride, nullptr};
  Pass dk{0, 0, 0, a.dim_v, a.dim_k, a.heads, a.len, a.batch, a.scale, true, a.log_decay, a.n_real,
          a.dfinal, true, a.dk, a.dk_batch_stride, a.dk_stride, nullptr};
  Pass dv{0, 0, 0, a.dim_k, a.dim_v, a.heads, a.len, a.batch, a.scale, true, a.log_decay, a.n_real,
          a.dfinal, false, a.dv, a.dv_batch_stride, a.dv_stride, a.dinitial};
  e = run_pass<T, T>(dq, x.d, x.v, x.k, ws, st, launches);
  const int share = a.heads / a.kv_heads;
  for (Pass* p : {&dk, &dv}) {
    if (e != cudaSuccess) return e;
    T* to = static_cast<T*>(p->out);
    const int64_t to_batch = p->out_batch, to_token = p->out_token;
    if (share > 1) {
      p->out = parts;
      p->out_token = (int64_t)a.heads * p->dv;
      p->out_batch = p->out_token * a.len;
    }
    const Array &q = p == &dk ? x.v : x.k, &k = p == &dk ? x.d : x.q, &v = p == &dk ? x.q : x.d;
    e = share > 1 ? run_pass<T, float>(*p, q, k, v, ws, st, launches)
                  : run_pass<T, T>(*p, q, k, v, ws, st, launches);
    const int64_t n = (int64_t)a.batch * a.len * a.kv_heads * p->dv;
    if (e != cudaSuccess || share == 1 || !n) continue;
    e = tc::follow((*launches)++, sum_heads_kernel<T>,
                   dim3((unsigned)std::min<int64_t>((n + 255) / 256, 148 * 8)), 256, 0, st, parts, to,
                   (int64_t)a.batch * a.len, a.len, a.kv_heads, share, p->dv, to_batch, to_token);
  }
  return e;
}

}  // namespace

size_t linear_attention_bytes(const salt_linear_attention_args& a) {
  size_t n = 0;
  SALT_WITH_TYPE(a.type, T, n = forward_bytes<T>(a));
  return n;
}

cudaError_t linear_attention_launch(const salt_linear_attention_args& a, void* ws, cudaStream_t st,
                                    int* launches) {
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, e = forward<T>(a, static_cast<uint8_t*>(ws), st, launches));
  return e;
}

cudaError_t linear_attention_step_launch(const salt_linear_attention_step_args& a, cudaStream_t st,
                                         int* launches) {
  if (!a.batch) return cudaSuccess;
  const bool vec = aligned16(a.pool) && a.dim_v % 4 == 0;
  SALT_WITH_TYPE(a.type, T, {
    const auto kernel = vec ? attention_step_kernel<T, true> : attention_step_kernel<T, false>;
    kernel<<<a.batch * a.heads, 256, 0, st>>>(a);
  });
  ++*launches;
  return cudaGetLastError();
}

size_t linear_attention_backward_bytes(const salt_linear_attention_backward_args& a) {
  size_t n = 0;
  SALT_WITH_TYPE(a.type, T, n = backward_bytes<T>(a));
  return n;
}

cudaError_t linear_attention_backward_launch(const salt_linear_attention_backward_args& a, void* ws,
                                             cudaStream_t st, int* launches) {
  cudaError_t e = cudaSuccess;
  SALT_WITH_TYPE(a.type, T, e = backward<T>(a, static_cast<uint8_t*>(ws), st, launches));
  return e;
}

}  // namespace salt
