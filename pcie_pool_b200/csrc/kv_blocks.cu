// Which blocks of a paged KV cache matter: key bounds of its pages, the choice of
// blocks by those bounds, and eviction by accumulated attention weight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "paged_kv.h"

namespace ppb {
namespace {

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

__device__ __forceinline__ int length_of(const KvRequests& r, int block, int b) {
  return max(0, (int)min((long long)r.lens[b], (long long)r.width * block));
}

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <>
struct Pair<__half> {
  using type = __half2;
};

// Smaller and larger of packed pairs; a value that is not a number gives way to the other.
template <typename T>
__device__ __forceinline__ uint32_t least2(uint32_t x, uint32_t y) {
  using P = typename Pair<T>::type;
  P r = __hmin2(reinterpret_cast<P&>(x), reinterpret_cast<P&>(y));
  return reinterpret_cast<uint32_t&>(r);
}
template <typename T>
__device__ __forceinline__ uint32_t most2(uint32_t x, uint32_t y) {
  using P = typename Pair<T>::type;
  P r = __hmax2(reinterpret_cast<P&>(x), reinterpret_cast<P&>(y));
  return reinterpret_cast<uint32_t&>(r);
}
template <typename T>
__device__ __forceinline__ float2 floats(uint32_t v) {
  const T* p = reinterpret_cast<const T*>(&v);
  return make_float2(to_f(p[0]), to_f(p[1]));
}

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_parent() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- key bounds -------------------------------------------------------------------
// A CTA for each block: a thread takes 8 channels of all its tokens, 16 bytes a load,
// eight loads in flight; the keys' bytes bound it.
template <typename T>
__global__ void __launch_bounds__(256) bounds_kernel(const __grid_constant__ PagedKv kv, const __grid_constant__ KvRequests r,
                                                     int new_tokens, T* __restrict__ bounds) {
  const int b = blockIdx.y, len = length_of(r, kv.block, b);
  const int j = (new_tokens < 0 ? 0 : max(0, len - new_tokens) / kv.block) + blockIdx.x;
  if (static_cast<long long>(j) * kv.block >= len) return;
  const int page = r.table[b * r.table_stride + j], n = min(kv.block, len - j * kv.block);
  if (page < 0 || page >= kv.pages) return;
  const int per = kv.dim / 8;
  for (int c = threadIdx.x; c < kv.kv_heads * per; c += blockDim.x) {
    const int g = c / per, d = c % per * 8;
    const T* k = static_cast<const T*>(kv.base) + page * kv.page_stride + g * kv.head_stride + d;
    uint4 lo = __ldcs(reinterpret_cast<const uint4*>(k)), hi = lo;
#pragma unroll 8
    for (int t = 1; t < n; ++t) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(k + t * kv.token_stride));
      lo = make_uint4(least2<T>(lo.x, v.x), least2<T>(lo.y, v.y), least2<T>(lo.z, v.z), least2<T>(lo.w, v.w));
      hi = make_uint4(most2<T>(hi.x, v.x), most2<T>(hi.y, v.y), most2<T>(hi.z, v.z), most2<T>(hi.w, v.w));
    }
    T* o = bounds + (static_cast<long long>(page) * kv.kv_heads + g) * 2 * kv.dim + d;
    *reinterpret_cast<uint4*>(o) = lo;
    *reinterpret_cast<uint4*>(o + kv.dim) = hi;
  }
}

// ---- scores -------------------------------------------------------------------------
// score = sum over the group's heads h and the channels d of max(q_hd lo_d, q_hd hi_d)
//       = sum_d A_d hi_d + B_d lo_d,  A = sum_h max(q_h, 0),  B = sum_h min(q_h, 0),
// so a group costs as much as one head.  The sums are taken in 64 bits: products of
// two 8- or 11-bit numbers and their sums are then exact for all but far-flung
// exponents, and the order of blocks does not hang on the order of summation.  A
// warp takes eight blocks of one key head at a time (their loads are in flight
// together, and their sums are reduced together); it reads `kReach` channels of
// lower and upper bounds with 8 bytes a lane each.  The bounds' bytes bound it.
constexpr int kScoreWarps = 8, kScoreBlocks = 16, kTogether = 8, kReach = 128;

template <typename T, int PARTS>  // PARTS: dim / kReach, rounded up
__global__ void __launch_bounds__(kScoreWarps * 32) score_kernel(const __grid_constant__ KvSelect s) {
  const int b = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, G = s.heads / s.kv_heads;
  launch_dependents();
  const int n = (length_of(s.req, s.block, b) + s.block - 1) / s.block;
  const int from = blockIdx.x * kScoreBlocks;
  if (from >= n) return;
  const int batches = (min(kScoreBlocks, n - from) + kTogether - 1) / kTogether;
  const int* table = s.req.table + b * s.req.table_stride;
  double above[PARTS][4], below[PARTS][4];
  uint32_t above_on[PARTS][2], below_on[PARTS][2];  // channels that count: 0 * inf shall be nothing
  int have = -1;
  for (int unit = warp; unit < s.kv_heads * batches; unit += kScoreWarps) {
    const int g = unit % s.kv_heads, j0 = from + unit / s.kv_heads * kTogether;
    int page = lane < kTogether && j0 + lane < n ? table[j0 + lane] : -1;
    if (page >= s.pages) page = -1;
    uint2 lo[kTogether][PARTS], hi[kTogether][PARTS];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int at = __shfl_sync(0xffffffffu, page, i);
      const T* row = static_cast<const T*>(s.bounds) + (static_cast<long long>(max(at, 0)) * s.kv_heads + g) * 2 * s.dim;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const int d = p * kReach + lane * 4;
        lo[i][p] = hi[i][p] = make_uint2(0, 0);
        if (at >= 0 && d < s.dim) {
          lo[i][p] = *reinterpret_cast<const uint2*>(row + d);
          hi[i][p] = *reinterpret_cast<const uint2*>(row + s.dim + d);
        }
      }
    }
    if (have != g) {
      have = g;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) above[p][i] = below[p][i] = 0;
        const int d = p * kReach + lane * 4;
        if (d < s.dim) {
          const T* q = static_cast<const T*>(s.q) + b * s.q_stride + g * G * s.q_head_stride + d;
          for (int h = 0; h < G; ++h, q += s.q_head_stride) {
            const float2 x = floats<T>(*reinterpret_cast<const uint32_t*>(q)), y = floats<T>(*reinterpret_cast<const uint32_t*>(q + 2));
            const float v[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) (v[i] < 0.f ? below : above)[p][i] += v[i];
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          above_on[p][i] = (above[p][2 * i] != 0 ? 0xffffu : 0u) | (above[p][2 * i + 1] != 0 ? 0xffff0000u : 0u);
          below_on[p][i] = (below[p][2 * i] != 0 ? 0xffffu : 0u) | (below[p][2 * i + 1] != 0 ? 0xffff0000u : 0u);
        }
      }
    }
    double sum[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      sum[i] = 0;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const uint32_t l[2] = {lo[i][p].x, lo[i][p].y}, u[2] = {hi[i][p].x, hi[i][p].y};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 top = floats<T>(most2<T>(l[x], u[x]) & above_on[p][x]);
          const float2 low = floats<T>(least2<T>(l[x], u[x]) & below_on[p][x]);
          sum[i] += above[p][2 * x] * top.x;
          sum[i] += above[p][2 * x + 1] * top.y;
          sum[i] += below[p][2 * x] * low.x;
          sum[i] += below[p][2 * x + 1] * low.y;
        }
      }
    }
    // halve the eight sums while the lanes are added: lane bits 4, 3 and 2 choose the block
#pragma unroll
    for (int width = kTogether / 2, bit = 16; width > 0; width /= 2, bit /= 2)
#pragma unroll
      for (int i = 0; i < width; ++i) {
        const bool upper = lane & bit;
        const double give = upper ? sum[i] : sum[i + width], keep = upper ? sum[i + width] : sum[i];
        sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 2);
    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
    const int j = j0 + (lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1);
    if ((lane & 3) == 0 && j < n)
      s.scores[(static_cast<long long>(b) * s.kv_heads + g) * s.req.width + j] = static_cast<float>(sum[0]);
  }
}

// ---- the highest of a row --------------------------------------------------------------
// A CTA for each row.  A thread holds ITEMS neighbours as unsigned keys in the order
// of the values; the border is found bit by bit from the top, counting the keys
// above it, and the row is written in order by a scan over the threads.  Rows longer
// than THREADS * ITEMS are read again in every pass.

// Not a number is the lowest value, both zeros are equal.  0 is left for what cannot
// be taken, all ones for what must be.
__device__ __forceinline__ unsigned key_of(float v) {
  if (v != v) return 1u;
  const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int THREADS>
struct Counter {
  static constexpr int kWarps = THREADS / 32;
  int (*scratch)[32];  // two rows in turn, so that one barrier a count is enough
  int turn = 0;

  __device__ int sum(int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    int* row = scratch[turn ^= 1];
    if (threadIdx.x % 32 == 0) row[threadIdx.x / 32] = v;
    __syncthreads();
    const int lane = threadIdx.x % 32;
    return __reduce_add_sync(0xffffffffu, lane < kWarps ? row[lane] : 0);
  }
  // Sum of the lower threads' v; `total` of all.
  __device__ int before(int v, int& total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int upto = v;
#pragma unroll
    for (int x = 1; x < 32; x *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, upto, x);
      if (lane >= x) upto += u;
    }
    int* row = scratch[turn ^= 1];
    if (lane == 31) row[warp] = upto;
    __syncthreads();
    const int w = lane < kWarps ? row[lane] : 0;
    total = __reduce_add_sync(0xffffffffu, w);
    return upto - v + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
  }
};

// Keys of a row of values whose table entries lie in [0, pages).
struct ValueKey {
  const float* value;
  const int* table;
  int pages, n, sink, recent;

  struct Raw {
    float value;
    int page;
  };
  __device__ Raw read(int j) const { return {value[j], table[j]}; }
  __device__ unsigned make(int j, Raw r) const {
    if (r.page < 0 || r.page >= pages) return 0u;
    return j < sink || j >= n - recent ? 0xffffffffu : key_of(r.value);
  }
};

struct Border {
  unsigned above;  // every key above it is taken
  int ties;        // and so many equal to it, from the lowest index
};

template <int THREADS, int ITEMS, typename Key>
struct Row {
  static constexpr int kChunk = THREADS * ITEMS;
  Key key;
  int n;
  Counter<THREADS> counter;
  unsigned keys[ITEMS];

  // All of a thread's values are on their way before the first is looked at.
  __device__ void load(int base) {
    decltype(key.read(0)) raw[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) raw[i] = key.read(min(base + static_cast<int>(threadIdx.x) * ITEMS + i, n - 1));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + threadIdx.x * ITEMS + i;
      keys[i] = j < n ? key.make(j, raw[i]) : 0u;
    }
  }
  __device__ int at_least(unsigned c) {
    int m = 0;
    for (int base = 0; base < n; base += kChunk) {
      if (n > kChunk) load(base);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) m += keys[i] >= c;
    }
    return counter.sum(m);
  }
  // Border of the `want` highest.
  __device__ Border border(int want) {
    if (n == 0) return {0xffffffffu, 0};
    if (n <= kChunk) load(0);
    want = min(want, at_least(1u));
    if (want == 0) return {0xffffffffu, 0};
    unsigned t = 0;
    int over = 0;  // keys above all that begin like t
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned c = t | 1u << bit;
      const int m = at_least(c);
      if (m == want) return {c - 1, 0};
      if (m > want)
        t = c;
      else
        over = m;
    }
    return {t, want - over};
  }
  // put(index, key, rank among the taken) for what is taken, leave(index, rank) for
  // the others that could be; returns the number of the taken.
  template <typename Put, typename Leave>
  __device__ int emit(const Border& e, Put put, Leave leave) {
    int ties = 0, done = 0, gone = 0;
    for (int base = 0; base < n; base += kChunk) {
      if (n > kChunk) load(base);
      int tie = 0, can = 0;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) tie += keys[i] == e.above && keys[i] != 0, can += keys[i] != 0;
      int all_ties, all;
      const int tie0 = ties + counter.before(tie, all_ties);
      int take = 0, seen = tie0;
      bool taken[ITEMS];
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const bool equal = keys[i] == e.above && keys[i] != 0;
        taken[i] = keys[i] > e.above || (equal && seen < e.ties);
        seen += equal;
        take += taken[i];
      }
      int at = done + counter.before(take, all), all_gone;
      int out = gone + counter.before(can - take, all_gone);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int j = base + threadIdx.x * ITEMS + i;
        if (taken[i])
          put(j, at++);
        else if (keys[i] != 0)
          leave(j, out++);
      }
      ties += all_ties;
      done += all;
      gone += all_gone;
    }
    left = gone;
    return done;
  }
  int left = 0;  // of the others
};

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) select_kernel(const __grid_constant__ KvSelect s) {
  __shared__ int scratch[2][32];
  const int b = blockIdx.x / s.kv_heads;
  const int n = (length_of(s.req, s.block, b) + s.block - 1) / s.block;
  const float* score = s.scores + static_cast<long long>(blockIdx.x) * s.req.width;
  const int* table = s.req.table + b * s.req.table_stride;
  int* out = s.out + static_cast<long long>(blockIdx.x) * s.keep;
  wait_for_parent();
  Row<THREADS, ITEMS, ValueKey> row{{score, table, s.pages, n, s.sink, s.recent}, n, {scratch}};
  const Border e = row.border(s.keep);
  const int done = row.emit(e, [&](int j, int at) { out[at] = j; }, [](int, int) {});
  for (int j = done + threadIdx.x; j < s.keep; j += THREADS) out[j] = -1;
}

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) evict_kernel(const __grid_constant__ KvEvict e) {
  __shared__ int scratch[2][32];
  const int b = blockIdx.x, width = e.req.width, len = length_of(e.req, e.block, b);
  const int n = (len + e.block - 1) / e.block;
  const float* mass = e.mass + b * e.mass_stride;
  const int* table = e.req.table + b * e.req.table_stride;
  const long long at0 = static_cast<long long>(b) * width;
  Row<THREADS, ITEMS, ValueKey> row{{mass, table, INT_MAX, n, e.sink, e.recent}, n, {scratch}};
  const Border border = row.border(e.budget);
  int tokens = 0;
  const int kept = row.emit(
      border,
      [&](int j, int at) {
        e.new_table[at0 + at] = table[j];
        e.new_mass[at0 + at] = mass[j];
        tokens += min(e.block, len - j * e.block);
      },
      [&](int j, int at) {
        e.evicted[at0 + at] = table[j];
        e.evicted_at[at0 + at] = j;
      });
  for (int j = kept + threadIdx.x; j < width; j += THREADS) e.new_table[at0 + j] = -1, e.new_mass[at0 + j] = 0.f;
  for (int j = row.left + threadIdx.x; j < width; j += THREADS) e.evicted[at0 + j] = -1, e.evicted_at[at0 + j] = -1;
  tokens = row.counter.sum(tokens);
  if (threadIdx.x == 0) {
    e.new_lens[b] = tokens;
    e.evicted_count[b] = row.left;
  }
}

// By the longest row there can be: fewer threads mean cheaper barriers.
template <typename Launch>
void for_width(int width, Launch launch) {
  using std::integral_constant;
  if (width <= 1024)
    launch(integral_constant<int, 256>(), integral_constant<int, 4>());
  else if (width <= 4096)
    launch(integral_constant<int, 512>(), integral_constant<int, 8>());
  else
    launch(integral_constant<int, 1024>(), integral_constant<int, 16>());
}

}  // namespace

cudaError_t paged_kv_bounds(const PagedKv& kv, const KvRequests& req, int new_tokens, void* bounds,
                            cudaStream_t stream) {
  const int blocks = new_tokens < 0 ? req.width
                                    : static_cast<int>(std::min((long long)req.width, (new_tokens + kv.block - 2ll) / kv.block + 1));
  if (req.requests == 0 || blocks == 0 || new_tokens == 0) return cudaSuccess;
  const dim3 grid(blocks, req.requests);
  const int threads = std::min(256, (kv.kv_heads * kv.dim / 8 + 31) / 32 * 32);
  if (kv.type == kKvBf16)
    bounds_kernel<<<grid, threads, 0, stream>>>(kv, req, new_tokens, static_cast<__nv_bfloat16*>(bounds));
  else
    bounds_kernel<<<grid, threads, 0, stream>>>(kv, req, new_tokens, static_cast<__half*>(bounds));
  return cudaGetLastError();
}

cudaError_t paged_kv_select(const KvSelect& s, cudaStream_t stream) {
  if (s.req.requests == 0) return cudaSuccess;
  if (s.req.width) {
    const dim3 grid((s.req.width + kScoreBlocks - 1) / kScoreBlocks, s.req.requests);
    auto score = s.type == kKvBf16 ? (s.dim <= kReach ? score_kernel<__nv_bfloat16, 1> : score_kernel<__nv_bfloat16, 2>)
                                   : (s.dim <= kReach ? score_kernel<__half, 1> : score_kernel<__half, 2>);
    score<<<grid, kScoreWarps * 32, 0, stream>>>(s);
    const cudaError_t rc = cudaGetLastError();
    if (rc != cudaSuccess) return rc;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(s.req.requests * s.kv_heads);
  config.stream = stream;
  cudaLaunchAttribute attr;  // it waits for the scores itself
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = s.req.width ? 1 : 0;
  cudaError_t rc = cudaSuccess;
  for_width(s.req.width, [&](auto threads, auto items) {
    config.blockDim = dim3(threads());
    rc = cudaLaunchKernelEx(&config, select_kernel<threads(), items()>, s);
  });
  return rc;
}

cudaError_t paged_kv_evict(const KvEvict& e, cudaStream_t stream) {
  if (e.req.requests == 0) return cudaSuccess;
  for_width(e.req.width, [&](auto threads, auto items) {
    evict_kernel<threads(), items()><<<e.req.requests, threads(), 0, stream>>>(e);
  });
  return cudaGetLastError();
}

}  // namespace ppb
