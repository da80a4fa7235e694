// What the paged-KV kernels share on the device.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "paged_kv.h"

namespace ppb {
namespace dev {

// ---- copies of 16 bytes into shared memory, in groups ---------------------------
// Without `valid` nothing is read and the place is filled with zeros.
__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- a kernel and the one behind it in the stream -----------------------------------
// The one behind may start before this one is done; before it reads what this one
// writes (and in every thread, so that it does not end first) it waits for its end.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_parent() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- requests -------------------------------------------------------------------------
// Tokens of request b, cut to its table.
__device__ __forceinline__ int length_of(const KvRequests& r, int block, int b) {
  const long long most = static_cast<long long>(r.width) * block;
  return max(0, static_cast<int>(min(static_cast<long long>(r.lens[b]), most)));
}

// first[b] = sum of count(c) over c < b for b = 0 .. n, by the whole CTA; scratch
// has a place for each warp.
template <typename Count>
__device__ __forceinline__ void running_sums(int n, Count count, uint32_t* first, uint32_t* scratch) {
  const int per = (n + blockDim.x - 1) / blockDim.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int b0 = min(n, static_cast<int>(threadIdx.x) * per), b1 = min(n, b0 + per);
  uint32_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    first[b] = mine;
    mine += count(b);
  }
  uint32_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, x);
    if (lane >= x) upto += v;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  uint32_t before = upto - mine;
  for (int i = 0; i < warp; ++i) before += scratch[i];
  for (int b = b0; b < b1; ++b) first[b] += before;
  if (threadIdx.x == blockDim.x - 1) first[n] = before + mine;
  __syncthreads();
}

// The last b with first[b] <= at < first[n]; it has a count above 0.
__device__ __forceinline__ int request_of(const uint32_t* first, int n, uint32_t at) {
  int lo = 0, hi = n;  // first[lo] <= at < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= at)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

}  // namespace dev

// A kernel that may be resident before the one ahead of it in the stream is done
// (it waits for it itself).
template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), unsigned ctas, int threads, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(threads);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

inline cudaError_t sm_count(int* sms, int* device) {
  cudaError_t rc = cudaGetDevice(device);
  return rc != cudaSuccess ? rc : cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *device);
}

}  // namespace ppb
