// Which blocks of a paged KV cache matter: key bounds of its pages, the choice of
// blocks by those bounds, and eviction by accumulated attention weight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "paged_kv.h"

namespace ppb {
namespace {

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

__device__ __forceinline__ int length_of(const KvRequests& r, int block, int b) {
  return max(0, (int)min((long long)r.lens[b], (long long)r.width * block));
}

// ---- key bounds -------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(128) bounds_kernel(PagedKv kv, KvRequests r, int new_tokens, T* __restrict__ bounds) {
  const int b = blockIdx.y, len = length_of(r, kv.block, b);
  const int first = new_tokens < 0 ? 0 : max(0, len - new_tokens) / kv.block;
  const int j = first + blockIdx.x;
  if ((long long)j * kv.block >= len) return;
  const int page = r.table[b * r.table_stride + j], n = min(kv.block, len - j * kv.block);
  if (page < 0 || page >= kv.pages) return;
  for (int c = threadIdx.x; c < kv.kv_heads * kv.dim; c += blockDim.x) {
    const int g = c / kv.dim, d = c % kv.dim;
    const T* k = (const T*)kv.base + page * kv.page_stride + g * kv.head_stride + d;
    T lo = k[0], hi = k[0];
    for (int t = 1; t < n; ++t) {
      lo = __hmin(lo, k[t * kv.token_stride]);
      hi = __hmax(hi, k[t * kv.token_stride]);
    }
    T* o = bounds + ((long long)page * kv.kv_heads + g) * 2 * kv.dim + d;
    o[0] = lo;
    o[kv.dim] = hi;
  }
}

// ---- scores -------------------------------------------------------------------------
// score = sum over the group's heads of sum_d max(q_d lo_d, q_d hi_d): a warp for each
// (block, key head).
template <typename T>
__global__ void __launch_bounds__(128) score_kernel(KvSelect s) {
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x % 32;
  const int n = (length_of(s.req, s.block, b) + s.block - 1) / s.block, G = s.heads / s.kv_heads;
  for (int j = blockIdx.x * 4 + threadIdx.x / 32; j < n; j += gridDim.x * 4) {
    const int page = s.req.table[b * s.req.table_stride + j];
    if (page < 0 || page >= s.pages) continue;
    const T* lo = (const T*)s.bounds + ((long long)page * s.kv_heads + g) * 2 * s.dim;
    double sum = 0;
    for (int d = lane; d < s.dim; d += 32) {
      const double x = to_f(lo[d]), y = to_f(lo[s.dim + d]);
      for (int h = 0; h < G; ++h) {
        const double q = to_f(((const T*)s.q)[b * s.q_stride + (g * G + h) * s.q_head_stride + d]);
        sum += fmax(q * x, q * y);
      }
    }
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) s.scores[((long long)b * s.kv_heads + g) * s.req.width + j] = (float)sum;
  }
}

// ---- the highest of a row --------------------------------------------------------------
constexpr int kRowThreads = 512;

// Unsigned keys in the order of the values: not a number is the lowest value, both
// zeros are equal.  0 is left for what cannot be taken, all ones for what must be.
__device__ __forceinline__ unsigned key_of(float v) {
  if (v != v) return 1u;
  const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int block_sum(int v, int* scratch) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
  __syncthreads();
  int s = 0;
  for (int i = 0; i < kRowThreads / 32; ++i) s += scratch[i];
  return s;
}

// Number of true `flag`s of lower threads, and of all in `total`.
__device__ __forceinline__ int block_rank(bool flag, int* scratch, int& total) {
  const unsigned m = __ballot_sync(0xffffffffu, flag);
  const int warp = threadIdx.x / 32;
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[warp] = __popc(m);
  __syncthreads();
  int before = __popc(m & ((1u << threadIdx.x % 32) - 1));
  total = 0;
  for (int i = 0; i < kRowThreads / 32; ++i) {
    if (i < warp) before += scratch[i];
    total += scratch[i];
  }
  return before;
}

struct Chosen {
  unsigned least;  // every key above it is taken
  int ties;        // and so many equal to it, from the lowest index
};

// The `want` highest keys of n, bit by bit from the top.
template <typename Key>
__device__ __forceinline__ Chosen choose(Key key, int n, int want, int* scratch) {
  int can = 0;
  for (int j = threadIdx.x; j < n; j += kRowThreads) can += key(j) != 0;
  can = block_sum(can, scratch);
  want = min(want, can);
  if (want == 0) return {0xffffffffu, 0};
  unsigned t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned c = t | 1u << bit;
    int m = 0;
    for (int j = threadIdx.x; j < n; j += kRowThreads) m += key(j) >= c;
    if (block_sum(m, scratch) >= want) t = c;
  }
  int above = 0;
  for (int j = threadIdx.x; j < n; j += kRowThreads) above += key(j) > t;
  return {t, want - block_sum(above, scratch)};
}

__global__ void __launch_bounds__(kRowThreads) select_kernel(KvSelect s) {
  __shared__ int scratch[kRowThreads / 32];
  const int b = blockIdx.y, g = blockIdx.x;
  const int n = (length_of(s.req, s.block, b) + s.block - 1) / s.block;
  const float* score = s.scores + ((long long)b * s.kv_heads + g) * s.req.width;
  const int* table = s.req.table + b * s.req.table_stride;
  auto key = [&](int j) -> unsigned {
    if (table[j] < 0 || table[j] >= s.pages) return 0u;
    return j < s.sink || j >= n - s.recent ? 0xffffffffu : key_of(score[j]);
  };
  const Chosen c = choose(key, n, s.keep, scratch);
  int* out = s.out + ((long long)b * s.kv_heads + g) * s.keep;
  int done = 0, ties = 0;
  for (int base = 0; base < n; base += kRowThreads) {
    const int j = base + threadIdx.x;
    const unsigned k = j < n ? key(j) : 0u;
    int nt, nk;
    const int rt = block_rank(k != 0 && k == c.least, scratch, nt);
    const bool take = k > c.least || (k != 0 && k == c.least && ties + rt < c.ties);
    const int rk = block_rank(take, scratch, nk);
    if (take) out[done + rk] = j;
    ties += nt;
    done += nk;
  }
  for (int j = done + threadIdx.x; j < s.keep; j += kRowThreads) out[j] = -1;
}

__global__ void __launch_bounds__(kRowThreads) evict_kernel(KvEvict e) {
  __shared__ int scratch[kRowThreads / 32];
  const int b = blockIdx.x, width = e.req.width, len = length_of(e.req, e.block, b);
  const int n = (len + e.block - 1) / e.block;
  const float* mass = e.mass + b * e.mass_stride;
  const int* table = e.req.table + b * e.req.table_stride;
  auto key = [&](int j) -> unsigned {
    if (table[j] < 0) return 0u;
    return j < e.sink || j >= n - e.recent ? 0xffffffffu : key_of(mass[j]);
  };
  const Chosen c = choose(key, n, e.budget, scratch);
  const long long row = (long long)b * width;
  int kept = 0, gone = 0, ties = 0, tokens = 0;
  for (int base = 0; base < n; base += kRowThreads) {
    const int j = base + threadIdx.x;
    const unsigned k = j < n ? key(j) : 0u;
    int nt, nk, ng;
    const int rt = block_rank(k != 0 && k == c.least, scratch, nt);
    const bool take = k > c.least || (k != 0 && k == c.least && ties + rt < c.ties);
    const int rk = block_rank(take, scratch, nk), rg = block_rank(k != 0 && !take, scratch, ng);
    if (take) {
      e.new_table[row + kept + rk] = table[j];
      e.new_mass[row + kept + rk] = mass[j];
      tokens += min(e.block, len - j * e.block);
    } else if (k != 0) {
      e.evicted[row + gone + rg] = table[j];
      e.evicted_at[row + gone + rg] = j;
    }
    ties += nt;
    kept += nk;
    gone += ng;
  }
  for (int j = kept + threadIdx.x; j < width; j += kRowThreads) e.new_table[row + j] = -1, e.new_mass[row + j] = 0.f;
  for (int j = gone + threadIdx.x; j < width; j += kRowThreads) e.evicted[row + j] = -1, e.evicted_at[row + j] = -1;
  tokens = block_sum(tokens, scratch);
  if (threadIdx.x == 0) {
    e.new_lens[b] = tokens;
    e.evicted_count[b] = gone;
  }
}

}  // namespace

cudaError_t paged_kv_bounds(const PagedKv& kv, const KvRequests& req, int new_tokens, void* bounds,
                            cudaStream_t stream) {
  const int blocks = new_tokens < 0 ? req.width
                                    : static_cast<int>(std::min((long long)req.width, (new_tokens + kv.block - 2ll) / kv.block + 1));
  if (req.requests == 0 || blocks == 0 || new_tokens == 0) return cudaSuccess;
  const dim3 grid(blocks, req.requests);
  if (kv.type == kKvBf16)
    bounds_kernel<<<grid, 128, 0, stream>>>(kv, req, new_tokens, static_cast<__nv_bfloat16*>(bounds));
  else
    bounds_kernel<<<grid, 128, 0, stream>>>(kv, req, new_tokens, static_cast<__half*>(bounds));
  return cudaGetLastError();
}

cudaError_t paged_kv_select(const KvSelect& s, cudaStream_t stream) {
  if (s.req.requests == 0) return cudaSuccess;
  if (s.req.width) {
    const dim3 grid((s.req.width + 31) / 32, s.kv_heads, s.req.requests);
    if (s.type == kKvBf16)
      score_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(s);
    else
      score_kernel<__half><<<grid, 128, 0, stream>>>(s);
  }
  select_kernel<<<dim3(s.kv_heads, s.req.requests), kRowThreads, 0, stream>>>(s);
  return cudaGetLastError();
}

cudaError_t paged_kv_evict(const KvEvict& e, cudaStream_t stream) {
  if (e.req.requests == 0) return cudaSuccess;
  evict_kernel<<<e.req.requests, kRowThreads, 0, stream>>>(e);
  return cudaGetLastError();
}

}  // namespace ppb
