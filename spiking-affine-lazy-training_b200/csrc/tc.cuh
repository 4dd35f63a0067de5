// Tensor cores of sm_100a (tcgen05, accumulators in tensor memory), tensor copies (TMA) and the
// barriers between them, as the sequence operators' products use them.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace salt::tc {

__device__ __forceinline__ uint32_t shared_at(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// ---------------------------------------------------------------- barriers in shared memory

__device__ __forceinline__ void barrier_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_at(b)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* b, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(shared_at(b)), "r"(parity)
      : "memory");
  return done;
}
// Waits for the barrier's phase of that parity to end.  Gives up after `tries` looks, which only a
// fault elsewhere can bring about (a look that finds nothing takes some 4 us: about a second in
// all), and leaves tries = 0 behind: later waits then look once.  Others' waits may still end well, so
// who gave up arrives at no barrier any more, and what waits for it gives up in turn ...
constexpr uint32_t kTries = 1u << 18;
__device__ __forceinline__ void barrier_wait(uint64_t* b, uint32_t parity, uint32_t& tries) {
  for (uint32_t i = tries; !barrier_try(b, parity); --i)
    if (i == 0) {
      tries = 0;
      break;
    }
}
// The same by a whole warp, whose lanes stay together.
__device__ __forceinline__ void barrier_wait_warp(uint64_t* b, uint32_t parity, uint32_t& tries) {
  for (uint32_t i = tries; !__all_sync(0xffffffffu, barrier_try(b, parity)); --i)
    if (i == 0) {
      tries = 0;
      break;
    }
}
// ... or leaves a mark that the block's threads share, at which each looks before it writes results.
__device__ __forceinline__ void barrier_wait(uint64_t* b, uint32_t parity, uint32_t& tries,
                                             uint32_t* gave_up) {
  for (uint32_t i = tries; !barrier_try(b, parity); --i)
    if (i == 0) {
      tries = 0;
      *reinterpret_cast<volatile uint32_t*>(gave_up) = 1;
      break;
    }
}
__device__ __forceinline__ void barrier_wait_warp(uint64_t* b, uint32_t parity, uint32_t& tries,
                                                  uint32_t* gave_up) {
  for (uint32_t i = tries; !__all_sync(0xffffffffu, barrier_try(b, parity)); --i)
    if (i == 0) {
      tries = 0;
      *reinterpret_cast<volatile uint32_t*>(gave_up) = 1;
      break;
    }
}
__device__ __forceinline__ bool marked(const uint32_t* gave_up) {
  return *reinterpret_cast<const volatile uint32_t*>(gave_up) != 0;
}
// An arrival of the lanes that hold 0, without a branch.
__device__ __forceinline__ void barrier_arrive_if_zero(uint64_t* b, int lane) {
  asm volatile(
      "{\n .reg .pred p;\n setp.eq.s32 p, %1, 0;\n @p mbarrier.arrive.shared::cta.b64 _, [%0];\n}" ::"r"(
          shared_at(b)),
      "r"(lane)
      : "memory");
}
// Threads of part of a block.
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// A warpgroup's share of the registers that the block was launched with.
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---------------------------------------------------------------- tensor copies

// Box (inner, outer) from column x (in elements; its bytes a multiple of 16) and row y.
__device__ __forceinline__ void load_box(void* to, const CUtensorMap* map, int x, int y,
                                         uint64_t* barrier) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(shared_at(to)),
      "l"(map), "r"(x), "r"(y), "r"(shared_at(barrier))
      : "memory");
}
// A box of shared memory to column x and row y, what lies past the array's edges left out.  The memory
// may be written again after stores_read, and given up after stores_done, by the same thread.
__device__ __forceinline__ void store_box(const CUtensorMap* map, const void* from, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(x), "r"(y), "r"(shared_at(from))
      : "memory");
}
__device__ __forceinline__ void store_box4(const CUtensorMap* map, const void* from, int x, int y, int z,
                                           int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];\n"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(x), "r"(y), "r"(z), "r"(w), "r"(shared_at(from))
      : "memory");
}
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void stores_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// The same of an array of four axes: box (inner, 1, rows, 1) from (x, y, z, w).
__device__ __forceinline__ void load_box4(void* to, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint64_t* barrier) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4, %5}], [%6];" ::"r"(shared_at(to)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(shared_at(barrier))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// 4 bytes by the calling thread; the barrier counts the thread once all its copies so far are there.
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_at(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* barrier) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_at(barrier))
               : "memory");
}
// The same in groups: all but the thread's last N groups are there.
__device__ __forceinline__ void copies_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---------------------------------------------------------------- tensor memory

// By one whole warp; `columns` a power of two, 32 to 512.
__device__ __forceinline__ void tmem_alloc(uint32_t* at, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   shared_at(at)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Shared memory that threads wrote, for the tensor cores to read.
__device__ __forceinline__ void fence_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void loads_done() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// N columns of the warp's 32 rows: a register each.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t (&r)[N], uint32_t at) {
  static_assert(N == 8 || N == 16, "columns of one load");
  if constexpr (N == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(at));
  }
}

__device__ __forceinline__ void stores_to_tmem_done() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// 8 columns of the warp's 32 rows from registers.
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// ---------------------------------------------------------------- products

// An operand in shared memory in rows of 128 bytes, swizzled by 128 bytes (the 16-byte unit of row r
// at place unit ^ (r & 7)), 1024-byte aligned.  Along its depth (`step` bytes between groups of 8
// rows, of the operand's other axis), or, for 16-bit types, across it (rows are the depth, `step`
// between groups of 8, `panel` bytes between panels of 64 elements of the other axis).
__device__ __forceinline__ uint64_t operand(const void* p, uint32_t step, uint32_t panel = 16) {
  return (uint64_t)((shared_at(p) & 0x3ffff) >> 4) | (uint64_t)(panel >> 4) << 16 |
         (uint64_t)(step >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The descriptor of an operand `bytes` further on.
__device__ __forceinline__ uint64_t further(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }

// Shape and types of a product with 32-bit sums: M x N; formats 0 e4m3 or float16, 1 bfloat16;
// `across` for operands whose rows are the depth.
__host__ __device__ constexpr uint32_t shape(int m, int n, int format, bool a_across = false,
                                             bool b_across = false) {
  return 1u << 4 | (uint32_t)format << 7 | (uint32_t)format << 10 | (uint32_t)a_across << 15 |
         (uint32_t)b_across << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// d (+)= a b over a depth of 32 bytes, by one thread.
__device__ __forceinline__ void product_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t shape,
                                             bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void product_16(uint32_t d, uint64_t a, uint64_t b, uint32_t shape,
                                           bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
      : "memory");
}
// The same with a in tensor memory: a row a lane, two 16-bit values a column.
__device__ __forceinline__ void product_16_from_tmem(uint32_t d, uint32_t a, uint64_t b,
                                                     uint32_t shape, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
      : "memory");
}
// The barrier's arrival once all products that this thread issued are done.
__device__ __forceinline__ void products_done(uint64_t* barrier) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   shared_at(barrier))
               : "memory");
}
// Kernels of one call that follow one another on a stream (`follow` below): the next may set itself up
// once every block of this one runs, and every thread waits for the whole kernel in front, and all that
// it wrote, before it touches memory that kernels of the call write or have written.  (Every kernel of
// the call waits, so the one in front ends after all those before it.)
__device__ __forceinline__ void let_next_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_earlier() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ bool one_lane() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(is));
  return is;
}

// ---------------------------------------------------------------- host

// Launches a kernel that calls `wait_for_earlier`; the call's first one (`follows` false) starts behind
// all that the stream holds.
template <typename... Params, typename... Args>
cudaError_t follow(bool follows, void (*kernel)(Params...), dim3 grid, int threads, size_t shared,
                   cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = shared;
  c.stream = st;
  cudaLaunchAttribute overlap = {};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &overlap;
  c.numAttrs = follows ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, static_cast<Params>(args)...);
  return e == cudaSuccess ? e : cudaGetLastError();
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder of tensor maps; NULL where it has none.
inline EncodeTiled encoder() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}
// Lets a kernel have that much dynamic shared memory: asked of the runtime once a device (`done` is the
// kernel's own, a bit a device).
inline cudaError_t allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
constexpr int64_t kMostStride = 1ll << 39;  // bytes: a tensor map's strides lie under 2^40

}  // namespace salt::tc
