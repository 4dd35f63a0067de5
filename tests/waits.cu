// A block whose first warp waits at a barrier and then lets the second warp's barrier end, as a kernel's
// product thread does with its products: the second warp's own wait always ends well.
#include "tc.cuh"

using namespace salt;

__global__ void two_waits(int* out, bool arrives, uint32_t limit) {
  __shared__ uint64_t first, second;
  __shared__ uint32_t gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::barrier_init(&first, 1);
    tc::barrier_init(&second, 1);
    gave_up = 0;
    tc::barrier_init_fence();
  }
  __syncthreads();
  uint32_t tries = warp == 0 ? limit : tc::kTries;
  if (warp == 0) {
    if (lane == 0) {
      tc::barrier_wait(&first, 0, tries, &gave_up);
      tc::barrier_arrive_if_zero(&second, 0);
      out[0] = tries > 0;
    }
  } else if (warp == 1) {
    tc::barrier_wait_warp(&second, 0, tries, &gave_up);
    const bool lost = tc::marked(&gave_up);
    if (lane == 0) out[1] = tries > 0, out[2] = lost;
  } else if (arrives) {
    tc::barrier_arrive_if_zero(&first, lane);
  }
}

// One whole warp that waits where nobody arrives: (tries left, the mark).
__global__ void one_wait(int* out, uint32_t limit) {
  __shared__ uint64_t never;
  __shared__ uint32_t gave_up;
  if (threadIdx.x == 0) {
    tc::barrier_init(&never, 1);
    gave_up = 0;
    tc::barrier_init_fence();
  }
  __syncthreads();
  uint32_t tries = limit;
  tc::barrier_wait_warp(&never, 0, tries, &gave_up);
  tc::barrier_wait_warp(&never, 0, tries, &gave_up);  // looks once
  const bool lost = tc::marked(&gave_up);
  if (threadIdx.x == 0) out[0] = tries > 0, out[1] = lost;
}

extern "C" int run_waits(int arrives, unsigned limit, int* host) {
  int* out = nullptr;
  cudaError_t e = cudaMalloc(&out, 5 * sizeof(int));
  if (e == cudaSuccess) {
    two_waits<<<1, 96>>>(out, arrives != 0, limit);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    one_wait<<<1, 32>>>(out + 3, limit);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(host, out, 5 * sizeof(int), cudaMemcpyDeviceToHost);
  cudaFree(out);
  return (int)e;
}
