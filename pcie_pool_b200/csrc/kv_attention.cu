// Attention of one new token per request over a paged KV cache.
//
//   s_t = scale * <q, K_t>,  out = sum_t exp(s_t - lse) V_t,  lse = log sum_t exp(s_t)
//   mass_j += sum over heads and the tokens t of block j of exp(s_t - lse)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "paged_kv.h"

namespace ppb {
namespace {

constexpr int kTile = 16;  // tokens of a step; the mass is gathered by tiles

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(__half& o, float v) { o = __float2half_rn(v); }

// Blocks of request b that are read: all that hold tokens, or the listed ones.
__device__ __forceinline__ int slots_of(const KvAttention& a, int len) {
  const int n = (len + a.kv.block - 1) / a.kv.block;
  return a.blocks != nullptr && a.blocks_width < n ? a.blocks_width : n;
}

// One CTA for each query head of a request, four warps that take tiles in turn.
template <typename T>
__global__ void __launch_bounds__(128) attention_kernel(KvAttention a, float* __restrict__ z, int max_tiles) {
  const int b = blockIdx.y, h = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int D = a.kv.dim, g = h / (a.heads / a.kv.kv_heads);
  const long long most = (long long)a.req.width * a.kv.block;
  const int len = max(0, (int)min((long long)a.req.lens[b], most));
  const int slots = slots_of(a, len), tiles = (int)(((long long)slots * a.kv.block + kTile - 1) / kTile);
  const T* qp = (const T*)a.q + b * a.q_stride + h * a.q_head_stride;
  const T* kp = (const T*)a.kv.base + g * a.kv.head_stride;
  float q[8], o[8], m = -INFINITY, l = 0.f;
  for (int i = 0; i < 8; ++i) {
    q[i] = lane + 32 * i < D ? to_f(qp[lane + 32 * i]) : 0.f;
    o[i] = 0.f;
  }
  for (int tile = warp; tile < tiles; tile += 4) {
    float zm = -INFINITY, zl = 0.f;
    for (int r = 0; r < kTile; ++r) {
      const long long t = (long long)tile * kTile + r;
      const int slot = (int)(t / a.kv.block), off = (int)(t % a.kv.block);
      if (slot >= slots) break;
      const int lb = a.blocks ? a.blocks[((long long)b * a.kv.kv_heads + g) * a.blocks_width + slot] : slot;
      if (lb < 0 || (long long)lb * a.kv.block + off >= len) continue;
      const int page = a.req.table[b * a.req.table_stride + lb];
      if (page < 0 || page >= a.kv.pages) continue;
      const T* k = kp + page * a.kv.page_stride + off * a.kv.token_stride;
      float s = 0.f;
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < D) s += q[i] * to_f(k[lane + 32 * i]);
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= a.scale;
      if (s == -INFINITY) continue;
      const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
      m = mn;
      l = l * c + p;
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < D) o[i] = o[i] * c + p * to_f(k[a.kv.lane_stride + lane + 32 * i]);
      const float zn = fmaxf(zm, s);
      zl = (zm == -INFINITY ? 0.f : zl * expf(zm - zn)) + expf(s - zn);
      zm = zn;
    }
    if (z && lane == 0) z[((long long)b * max_tiles + tile) * a.heads + h] = zm + logf(zl);
  }
  __shared__ float sm[4], sl[4], so[4][256];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < D) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float w[4], total = 0.f;
  for (int i = 0; i < 4; ++i) {
    w[i] = sm[i] == -INFINITY ? 0.f : expf(sm[i] - top);
    total += w[i] * sl[i];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.f;
    for (int i = 0; i < 4; ++i) v += w[i] * so[i][d];
    from_f(((T*)a.out)[((long long)b * a.heads + h) * D + d], total == 0.f ? 0.f : v / total);
  }
  if (threadIdx.x == 0) a.lse[(long long)b * a.heads + h] = total == 0.f ? -INFINITY : top + logf(total);
}

// A warp for each block: the tiles' log-sums of every head, weighed by the head's total.
__global__ void __launch_bounds__(128) mass_kernel(KvAttention a, const float* __restrict__ z, int max_tiles) {
  const int b = blockIdx.y, j = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long most = (long long)a.req.width * a.kv.block;
  const int len = max(0, (int)min((long long)a.req.lens[b], most));
  if (j >= (len + a.kv.block - 1) / a.kv.block) return;
  const int per = a.kv.block / kTile, last = (len + kTile - 1) / kTile;
  float sum = 0.f;
  for (int t = j * per; t < min((j + 1) * per, last); ++t)
    for (int h = lane; h < a.heads; h += 32) {
      const float v = z[((long long)b * max_tiles + t) * a.heads + h];
      if (v != -INFINITY) sum += expf(v - a.lse[(long long)b * a.heads + h]);
    }
  for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if (lane == 0) a.mass[b * a.mass_stride + j] += sum;
}

int max_tiles(const KvAttention& a) {
  return static_cast<int>(((long long)a.req.width * a.kv.block + kTile - 1) / kTile);
}

}  // namespace

uint64_t paged_kv_attention_work(const KvAttention& a, int) {
  return a.mass ? uint64_t(a.req.requests) * max_tiles(a) * a.heads * 4 : 0;
}

cudaError_t paged_kv_attention(const KvAttention& a, cudaStream_t stream) {
  if (a.req.requests == 0) return cudaSuccess;
  float* z = a.mass ? static_cast<float*>(a.work) : nullptr;
  const dim3 grid(a.heads, a.req.requests);
  if (a.kv.type == kKvBf16)
    attention_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a, z, max_tiles(a));
  else
    attention_kernel<__half><<<grid, 128, 0, stream>>>(a, z, max_tiles(a));
  if (a.mass && a.req.width)
    mass_kernel<<<dim3((a.req.width + 3) / 4, a.req.requests), 128, 0, stream>>>(a, z, max_tiles(a));
  return cudaGetLastError();
}

}  // namespace ppb
