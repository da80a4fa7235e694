// Which blocks of a paged KV cache matter: key bounds of its pages, the choice of
// blocks by those bounds, and eviction by accumulated attention weight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "device_utils.cuh"
#include "kv_device.cuh"
#include "kv_plan.h"
#include "paged_kv.h"

namespace ppb {
namespace {

using namespace dev;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

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

// ---- key bounds -------------------------------------------------------------------
// A CTA for each block in turn, of those that there are: a thread takes 8 channels of
// 16 tokens at a time, 16 loads of 16 bytes in flight, and the next block's page is
// looked up meanwhile.  The keys' bytes bound it: 8 prompts of 181 to 32768 tokens (1024
// channels, 144 MB) take 24 us, 5.95 TB/s; the last blocks of 64 requests 3.6 us.
constexpr int kBoundsRows = 16;

template <typename T>
__global__ void __launch_bounds__(256, 2)
    bounds_kernel(const __grid_constant__ PagedKv kv, const __grid_constant__ KvRequests r, FastDiv by_block, int new_tokens,
                  T* __restrict__ bounds) {
  extern __shared__ uint32_t starts[];  // of the requests' blocks that are due
  __shared__ uint32_t scratch[8];
  auto from = [&](int len) { return new_tokens < 0 ? 0 : static_cast<int>(by_block.quotient(max(0, len - new_tokens))); };
  running_sums(r.requests,
               [&](int b) {
                 const int len = length_of(r, kv.block, b);
                 return by_block.quotient(len + kv.block - 1) - (len > 0 ? from(len) : 0);
               },
               starts, scratch);
  struct Due {
    int page, tokens;
  };
  auto look_up = [&](uint32_t item) {
    if (item >= starts[r.requests]) return Due{-1, 0};
    const int b = request_of(starts, r.requests, item), len = length_of(r, kv.block, b);
    const int j = from(len) + static_cast<int>(item - starts[b]);
    return Due{r.table[b * r.table_stride + j], min(kv.block, len - j * kv.block)};
  };
  const int per = kv.dim / 8;
  Due next = look_up(blockIdx.x);
  for (uint32_t item = blockIdx.x; item < starts[r.requests]; item += gridDim.x) {
    const Due due = next;
    next = look_up(item + gridDim.x);
    if (due.page < 0 || due.page >= kv.pages) continue;
    for (int c = threadIdx.x; c < kv.kv_heads * per; c += blockDim.x) {
      const int g = c / per, d = (c - g * per) * 8;
      const T* k = static_cast<const T*>(kv.base) + due.page * kv.page_stride + g * kv.head_stride + d;
      uint4 lo, hi;
      for (int t0 = 0; t0 < due.tokens; t0 += kBoundsRows) {
        uint4 v[kBoundsRows];
#pragma unroll
        for (int i = 0; i < kBoundsRows; ++i)  // behind the last token its row again
          v[i] = __ldcs(reinterpret_cast<const uint4*>(k + min(t0 + i, due.tokens - 1) * kv.token_stride));
        if (t0 == 0) lo = hi = v[0];
#pragma unroll
        for (int i = 0; i < kBoundsRows; ++i) {
          lo = make_uint4(least2<T>(lo.x, v[i].x), least2<T>(lo.y, v[i].y), least2<T>(lo.z, v[i].z), least2<T>(lo.w, v[i].w));
          hi = make_uint4(most2<T>(hi.x, v[i].x), most2<T>(hi.y, v[i].y), most2<T>(hi.z, v[i].z), most2<T>(hi.w, v[i].w));
        }
      }
      T* o = bounds + (static_cast<long long>(due.page) * kv.kv_heads + g) * 2 * kv.dim + d;
      *reinterpret_cast<uint4*>(o) = lo;
      *reinterpret_cast<uint4*>(o + kv.dim) = hi;
    }
  }
}

// ---- scores -------------------------------------------------------------------------
// score = sum over the group's heads h and the channels d of max(q_hd lo_d, q_hd hi_d)
//       = sum_d A_d hi_d + B_d lo_d,  A = sum_h max(q_h, 0),  B = sum_h min(q_h, 0),
// so a group costs as much as one head.  The sums are taken in 64 bits: products of
// two 8- or 11-bit numbers and their sums are then exact for all but far-flung
// exponents, and the order of blocks does not hang on the order of summation.  A
// warp takes eight blocks of one key head as a unit, whose sums are reduced together,
// with 4 of `kReach` channels of a row to a lane.  It asks for all its units' rows
// before it looks at the first (cp.async, through shared memory, since registers would hold
// too few): 192 KiB an SM on their way, of a call that fits in one wave all there is.
// Eight rows at a time in registers took 15 us for 28 MB of bounds, 15 ragged requests
// of 8 key heads; this takes 10.
//
// The conversion to 64 bits (a sixteenth of the rate of a product) is left out:
// the bits of a bf16 or fp16 value, moved to where a double keeps its exponent and
// mantissa, are that value times a power of two, subnormals and zero included.
// A and B carry half of that power, and the sum gets the other half back.  Infinities
// and values that are not a number do not move so; where a row has one (0 * x tells)
// the eight are summed again with converted values, in the same order, so that a
// block's score does not hang on its neighbours.
constexpr int kScoreWarps = 8, kTogether = 8, kReach = 128;

template <typename T>
struct Moved;
template <>
struct Moved<__nv_bfloat16> {  // exponent of 8 bits, bias 127: 2^(127 - 1023)
  static constexpr int kShift = 3;
  static constexpr uint32_t kMask = 0x8fffe000u;
  static constexpr double kHalf = 0x1p448;
};
template <>
struct Moved<__half> {  // exponent of 5 bits, bias 15: 2^(15 - 1023)
  static constexpr int kShift = 6;
  static constexpr uint32_t kMask = 0x81fffc00u;
  static constexpr double kHalf = 0x1p504;
};
template <typename T>
__device__ __forceinline__ double move(uint32_t pair, int which) {
  const int v = static_cast<int>(which ? pair : pair << 16);
  return __hiloint2double((v >> Moved<T>::kShift) & Moved<T>::kMask, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t zero_unless_special(uint32_t pair, uint32_t so_far) {
  using P = typename Pair<T>::type;
  const P zero = {T(0.f), T(0.f)};
  P r = __hfma2(reinterpret_cast<P&>(pair), zero, reinterpret_cast<P&>(so_far));
  return reinterpret_cast<uint32_t&>(r);
}

// PARTS: dim / kReach, rounded up.  A warp has two units, or one of the longer rows.
template <typename T, int PARTS>
__global__ void __launch_bounds__(kScoreWarps * 32) score_kernel(const __grid_constant__ KvSelect s, FastDiv by_block, FastDiv by_heads) {
  constexpr int kUnits = 2 / PARTS, kRowBytes = PARTS * kReach * 4;
  extern __shared__ __align__(128) uint8_t rows[];
  __shared__ uint32_t scratch[kScoreWarps];
  uint32_t* starts = reinterpret_cast<uint32_t*>(rows + kScoreWarps * kUnits * kTogether * kRowBytes);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, G = s.q.heads / s.kv_heads;
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(rows)) + warp * kUnits * kTogether * kRowBytes;
  const int chunks = s.dim / 4;  // 16-byte pieces of a row, both bounds
  const long long row_bytes = static_cast<long long>(s.kv_heads) * 4 * s.dim;
  launch_dependents();
  // items are 16 units (8 of longer rows) of a request, of all requests in a row
  running_sums(s.req.requests,
               [&](int b) {
                 const int batches = (by_block.quotient(length_of(s.req, s.block, b) + s.block - 1) + kTogether - 1) / kTogether;
                 return (batches * s.kv_heads + kScoreWarps * kUnits - 1) / (kScoreWarps * kUnits);
               },
               starts, scratch);
  for (uint32_t item = blockIdx.x; item < starts[s.req.requests]; item += gridDim.x) {
    const int b = request_of(starts, s.req.requests, item);
    const uint32_t unit0 = (item - starts[b]) * (kScoreWarps * kUnits) + warp;
    const int* table = s.req.table + b * s.req.table_stride;
    const int n = by_block.quotient(length_of(s.req, s.block, b) + s.block - 1);
    int pages[kUnits], heads[kUnits], first[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const uint32_t unit = unit0 + u * kScoreWarps, batch = by_heads.quotient(unit);
      heads[u] = unit - batch * s.kv_heads;
      first[u] = batch * kTogether;
      pages[u] = lane < kTogether && first[u] + lane < n ? table[first[u] + lane] : -1;
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (pages[u] >= s.pages) pages[u] = -1;
      const uint8_t* from = static_cast<const uint8_t*>(s.bounds) + static_cast<long long>(heads[u]) * 4 * s.dim + lane * 16;
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int page = __shfl_sync(0xffffffffu, pages[u], i);
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
          if (page >= 0 && p * 32 + lane < chunks)
            cp_async16(mine + (u * kTogether + i) * kRowBytes + (p * 32 + lane) * 16, from + page * row_bytes + p * 512, true);
      }
      cp_commit();
    }
    double above[PARTS][4], below[PARTS][4];
    uint32_t above_on[PARTS][2], below_on[PARTS][2];  // channels that count: 0 * inf shall be nothing
    int have = -1;
#pragma unroll 1
    for (int u = 0; u < kUnits; ++u) {
      const int g = u ? heads[kUnits - 1] : heads[0], j0 = u ? first[kUnits - 1] : first[0];
      if (j0 >= n) break;
      if (have != g) {
        have = g;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          double up[4] = {}, down[4] = {};
          const int d = p * kReach + lane * 4;
          if (d < s.dim) {
            const T* q = static_cast<const T*>(s.q.base) + b * s.q.stride + g * G * s.q.head_stride + d;
#pragma unroll 4
            for (int h = 0; h < G; ++h, q += s.q.head_stride) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(q), y = *reinterpret_cast<const uint32_t*>(q + 2);
              const float2 f = floats<T>(x), e = floats<T>(y);
              const float v[4] = {f.x, f.y, e.x, e.y};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const double w = v[i];
                if (v[i] < 0.f)
                  down[i] += w;
                else
                  up[i] += w;
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            above_on[p][i] = (up[2 * i] != 0 ? 0xffffu : 0u) | (up[2 * i + 1] != 0 ? 0xffff0000u : 0u);
            below_on[p][i] = (down[2 * i] != 0 ? 0xffffu : 0u) | (down[2 * i + 1] != 0 ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) above[p][i] = up[i] * Moved<T>::kHalf, below[p][i] = down[i] * Moved<T>::kHalf;
        }
      }
      if (u + 1 < kUnits)
        cp_wait<1>();
      else
        cp_wait<0>();
      __syncwarp();
      // this lane's channels of a row's bounds, those that count
      const uint8_t* at = rows + (warp * kUnits + u) * kTogether * kRowBytes + lane * 8;
      auto bounds_of = [&](int i, int p, uint2& top, uint2& low) {
        top = low = make_uint2(0, 0);
        if (p * kReach + lane * 4 < s.dim) {
          const uint2 l = *reinterpret_cast<const uint2*>(at + i * kRowBytes + p * 256);
          const uint2 h = *reinterpret_cast<const uint2*>(at + i * kRowBytes + p * 256 + s.dim * 2);
          top = make_uint2(most2<T>(l.x, h.x) & above_on[p][0], most2<T>(l.y, h.y) & above_on[p][1]);
          low = make_uint2(least2<T>(l.x, h.x) & below_on[p][0], least2<T>(l.y, h.y) & below_on[p][1]);
        }
      };
      double sum[kTogether];
      uint32_t special = 0;
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        sum[i] = 0;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          uint2 top, low;
          bounds_of(i, p, top, low);
          special = zero_unless_special<T>(top.x, zero_unless_special<T>(top.y, special));
          special = zero_unless_special<T>(low.x, zero_unless_special<T>(low.y, special));
          sum[i] += above[p][0] * move<T>(top.x, 0);
          sum[i] += above[p][1] * move<T>(top.x, 1);
          sum[i] += above[p][2] * move<T>(top.y, 0);
          sum[i] += above[p][3] * move<T>(top.y, 1);
          sum[i] += below[p][0] * move<T>(low.x, 0);
          sum[i] += below[p][1] * move<T>(low.x, 1);
          sum[i] += below[p][2] * move<T>(low.y, 0);
          sum[i] += below[p][3] * move<T>(low.y, 1);
        }
      }
      // (rows of blocks that are not there hold what was there before: nobody reads their scores)
      double by = Moved<T>::kHalf;
      if (__any_sync(0xffffffffu, special & 0x7fff7fffu)) {
        by = 1 / Moved<T>::kHalf;
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          sum[i] = 0;
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            uint2 top, low;
            bounds_of(i, p, top, low);
            const float2 a0 = floats<T>(top.x), a1 = floats<T>(top.y), b0 = floats<T>(low.x), b1 = floats<T>(low.y);
            sum[i] += above[p][0] * a0.x;
            sum[i] += above[p][1] * a0.y;
            sum[i] += above[p][2] * a1.x;
            sum[i] += above[p][3] * a1.y;
            sum[i] += below[p][0] * b0.x;
            sum[i] += below[p][1] * b0.y;
            sum[i] += below[p][2] * b1.x;
            sum[i] += below[p][3] * b1.y;
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
        s.scores[(static_cast<long long>(b) * s.kv_heads + g) * s.req.width + j] = static_cast<float>(sum[0] * by);
    }
    __syncwarp();  // the rows have been read
  }
}

// ---- the highest of a row --------------------------------------------------------------
// A CTA for each row.  A thread holds every THREADS-th value as an unsigned key in
// the order of the values.  The border is found by counting: the keys between the
// least and the highest that are still in question fall into 2048 bins of the
// highest bits in which they differ, the bin that holds the border is what is in
// question next, three times at most.  The row is then written in order by the
// counts of every warp's share of it.  Rows longer than THREADS * ITEMS are read
// again in every pass.  Latency bounds it: of the reads, some ten barriers, and the
// atomics of keys that fall together.

// Not a number is the lowest value, both zeros are equal.  0 is left for what cannot
// be taken, all ones for what must be.
__device__ __forceinline__ unsigned key_of(float v) {
  if (v != v) return 1u;
  const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

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
  static constexpr int kChunk = THREADS * ITEMS, kWarps = THREADS / 32, kShares = ITEMS * kWarps;
  static constexpr int kBinBits = 11, kBins = 1 << kBinBits, kOwn = kBins / THREADS;
  static constexpr unsigned kMust = 0xffffffffu;
  struct Shared {
    int bins[kBins];
    int sums[kWarps];
    unsigned least[kWarps], most[kWarps];
    int must[kWarps];
    int found[3];            // the border's bin, the keys above it, the keys in it
    int share[kShares + 1];  // of a chunk, in its order: item by item, warp by warp
  };
  Key key;
  int n;
  Shared& shared;
  unsigned keys[ITEMS];
  int taken = 0, left = 0;

  __device__ Row(const Key& k, int n_, Shared& s) : key(k), n(n_), shared(s) {}

  // All of a thread's values are on their way before the first is looked at.
  __device__ void load(int base) {
    typename Key::Raw raw[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) raw[i] = key.read(min(base + i * THREADS + static_cast<int>(threadIdx.x), n - 1));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + i * THREADS + threadIdx.x;
      keys[i] = j < n ? key.make(j, raw[i]) : 0u;
    }
  }
  // f(key) for every key of the row.
  template <typename F>
  __device__ void each(F f) {
    for (int base = 0; base < n; base += kChunk) {
      if (n > kChunk) load(base);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) f(keys[i]);
    }
  }
  // Border of the `want` highest; those that must be taken are no more than that.
  __device__ Border border(int want) {
    if (n == 0) return {kMust, 0};
    if (n <= kChunk) load(0);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    unsigned least = kMust, most = 0;
    int can = 0, must = 0;
    each([&](unsigned k) {
      must += k == kMust;
      if (k != 0 && k != kMust) {
        ++can;
        least = min(least, k);
        most = max(most, k);
      }
    });
    can = __reduce_add_sync(0xffffffffu, can);
    must = __reduce_add_sync(0xffffffffu, must);
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) shared.sums[warp] = can, shared.must[warp] = must, shared.least[warp] = least, shared.most[warp] = most;
    for (int i = threadIdx.x; i < kBins; i += THREADS) shared.bins[i] = 0;
    __syncthreads();
    can = must = 0;
    for (int w = 0; w < kWarps; ++w) {
      can += shared.sums[w];
      must += shared.must[w];
      least = min(least, shared.least[w]);
      most = max(most, shared.most[w]);
    }
    want -= must;
    if (want >= can) return {0u, 0};
    if (want <= 0) return {kMust - 1, 0};
    while (true) {  // 0 < want < number of the keys in [least, most]
      if (least == most) return {least, want};
      const int shift = max(0, 32 - __clz(least ^ most) - kBinBits);
      const unsigned low = least >> shift;
      each([&](unsigned k) {
        if (k >= least && k <= most && k != kMust) atomicAdd(&shared.bins[(k >> shift) - low], 1);
      });
      __syncthreads();
      // from the highest bin down: thread t owns bins [kBins - (t + 1) kOwn, kBins - t kOwn)
      int own[kOwn], mine = 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        own[i] = shared.bins[kBins - 1 - (threadIdx.x * kOwn + i)];
        mine += own[i];
      }
      int upto = mine;
#pragma unroll
      for (int x = 1; x < 32; x *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += u;
      }
      if (lane == 31) shared.sums[warp] = upto;
      __syncthreads();
      int above = upto - mine;
      for (int w = 0; w < warp; ++w) above += shared.sums[w];
      if (above < want && above + mine >= want) {
        int i = 0;
#pragma unroll
        for (int x = 0; x < kOwn - 1; ++x)
          if (i == x && above + own[x] < want) {
            above += own[x];
            ++i;
          }
        shared.found[0] = kBins - 1 - (threadIdx.x * kOwn + i);
        shared.found[1] = above;
        shared.found[2] = shared.bins[kBins - 1 - (threadIdx.x * kOwn + i)];
      }
      __syncthreads();
      const unsigned bin = low + shared.found[0];
      want -= shared.found[1];
      const unsigned from = max(least, bin << shift), to = min(most, (bin << shift) + ((1u << shift) - 1));
      if (want == shared.found[2]) return {from - 1, 0};  // all of the bin; from > 0
      least = from;
      most = to;
      for (int i = threadIdx.x; i < kBins; i += THREADS) shared.bins[i] = 0;
      __syncthreads();
    }
  }
  // Before this thread's item i in the chunk: where `flag` holds, by the ballots in
  // `votes` and the shares' sums.
  __device__ int rank(unsigned vote, int i) const {
    return shared.share[i * kWarps + threadIdx.x / 32] + __popc(vote & ((1u << threadIdx.x % 32) - 1));
  }
  // Turns the shares' counts into the numbers before them; returns their total.
  __device__ int scan_shares() {
    __syncthreads();
    if (threadIdx.x < 32) {
      constexpr int kEach = (kShares + 31) / 32;
      const int lane = threadIdx.x;
      int v[kEach], mine = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int at = lane * kEach + i;
        v[i] = at < kShares ? shared.share[at] : 0;
        mine += v[i];
      }
      int upto = mine;
#pragma unroll
      for (int x = 1; x < 32; x *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += u;
      }
      int before = upto - mine;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int at = lane * kEach + i;
        if (at < kShares) shared.share[at] = before;
        before += v[i];
      }
      if (lane == 31) shared.share[kShares] = upto;
    }
    __syncthreads();
    return shared.share[kShares];
  }
  // put(index, rank among the taken) for what is taken, leave(index, rank) for the
  // others that could be; sets the numbers of both.
  template <bool LEAVE, typename Put, typename Leave>
  __device__ void emit(const Border& e, Put put, Leave leave) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    int ties = 0;
    taken = left = 0;
    for (int base = 0; base < n; base += kChunk) {
      if (n > kChunk) load(base);
      unsigned take[ITEMS];
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) take[i] = __ballot_sync(0xffffffffu, keys[i] > e.above);
      if (e.ties > 0) {
        unsigned tie[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          tie[i] = __ballot_sync(0xffffffffu, keys[i] == e.above && keys[i] != 0);
          if (lane == 0) shared.share[i * kWarps + warp] = __popc(tie[i]);
        }
        const int all = scan_shares();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          take[i] |= __ballot_sync(0xffffffffu, (tie[i] >> lane & 1) && ties + rank(tie[i], i) < e.ties);
        ties += all;
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (lane == 0) shared.share[i * kWarps + warp] = __popc(take[i]);
      const int all = scan_shares();
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (take[i] >> lane & 1) put(base + i * THREADS + static_cast<int>(threadIdx.x), taken + rank(take[i], i));
      taken += all;
      __syncthreads();
      if (LEAVE) {
        unsigned rest[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          rest[i] = __ballot_sync(0xffffffffu, keys[i] != 0) & ~take[i];
          if (lane == 0) shared.share[i * kWarps + warp] = __popc(rest[i]);
        }
        const int others = scan_shares();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (rest[i] >> lane & 1) leave(base + i * THREADS + static_cast<int>(threadIdx.x), left + rank(rest[i], i));
        left += others;
        __syncthreads();
      }
    }
  }
};

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) select_kernel(const __grid_constant__ KvSelect s) {
  using Keys = Row<THREADS, ITEMS, ValueKey>;
  __shared__ typename Keys::Shared shared;
  const int b = blockIdx.x / s.kv_heads;
  const int n = (length_of(s.req, s.block, b) + s.block - 1) / s.block;
  const float* score = s.scores + static_cast<long long>(blockIdx.x) * s.req.width;
  const int* table = s.req.table + b * s.req.table_stride;
  int* out = s.out + static_cast<long long>(blockIdx.x) * s.keep;
  wait_for_parent();
  Keys row({score, table, s.pages, n, s.sink, s.recent}, n, shared);
  const Border e = row.border(s.keep);
  row.template emit<false>(e, [&](int j, int at) { out[at] = j; }, [](int, int) {});
  // (unsigned: keep may be 2^31 - 1, where a step of an int would wrap around)
  for (unsigned j = row.taken + threadIdx.x; j < static_cast<unsigned>(s.keep); j += THREADS) out[j] = -1;
}

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) evict_kernel(const __grid_constant__ KvEvict e) {
  using Keys = Row<THREADS, ITEMS, ValueKey>;
  __shared__ typename Keys::Shared shared;
  const int b = blockIdx.x, width = e.req.width, len = length_of(e.req, e.block, b);
  const int n = (len + e.block - 1) / e.block;
  const float* mass = e.mass + b * e.mass_stride;
  const int* table = e.req.table + b * e.req.table_stride;
  const long long at0 = static_cast<long long>(b) * width;
  Keys row({mass, table, e.pages, n, e.sink, e.recent}, n, shared);
  const Border border = row.border(e.budget);
  int tokens = 0;
  row.template emit<true>(
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
  for (int j = row.taken + threadIdx.x; j < width; j += THREADS) e.new_table[at0 + j] = -1, e.new_mass[at0 + j] = 0.f;
  for (int j = row.left + threadIdx.x; j < width; j += THREADS) e.evicted[at0 + j] = -1, e.evicted_at[at0 + j] = -1;
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  if (threadIdx.x % 32 == 0) shared.sums[threadIdx.x / 32] = tokens;
  __syncthreads();
  if (threadIdx.x == 0) {
    tokens = 0;
    for (int w = 0; w < THREADS / 32; ++w) tokens += shared.sums[w];
    e.new_lens[b] = tokens;
    e.evicted_count[b] = row.left;
  }
}

// By the longest row there can be: few threads with many values each, since what a
// warp does besides its values costs more than they do, but no more places than values
// (512 x 32 for rows of 8192 makes the selection 3 us longer than 512 x 16).
template <typename Launch>
void for_width(int width, Launch launch) {
  using std::integral_constant;
  if (width <= 1024)
    launch(integral_constant<int, 128>(), integral_constant<int, 8>());
  else if (width <= 4096)
    launch(integral_constant<int, 256>(), integral_constant<int, 16>());
  else if (width <= 8192)
    launch(integral_constant<int, 512>(), integral_constant<int, 16>());
  else
    launch(integral_constant<int, 512>(), integral_constant<int, 32>());
}

}  // namespace

cudaError_t paged_kv_bounds(const PagedKv& kv, const KvRequests& req, int new_tokens, void* bounds,
                            cudaStream_t stream) {
  const int64_t blocks = new_tokens < 0 ? req.width : std::min<int64_t>(req.width, (new_tokens + kv.block - 2ll) / kv.block + 1);
  if (req.requests == 0 || blocks == 0 || new_tokens == 0) return cudaSuccess;
  if (req.requests > kMostRequests) return cudaErrorInvalidValue;
  int sms = 0, device = 0;
  const cudaError_t rc = sm_count(&sms, &device);
  if (rc != cudaSuccess) return rc;
  const int threads = std::min<int64_t>(256, (static_cast<int64_t>(kv.kv_heads) * kv.dim / 8 + 31) / 32 * 32);
  const int64_t ctas = std::min<int64_t>(blocks * req.requests, sms * (512 / threads));
  const int smem = (req.requests + 1) * 4;
  const FastDiv by_block = FastDiv::make(kv.block);
  if (kv.type == kKvBf16)
    bounds_kernel<<<ctas, threads, smem, stream>>>(kv, req, by_block, new_tokens, static_cast<__nv_bfloat16*>(bounds));
  else
    bounds_kernel<<<ctas, threads, smem, stream>>>(kv, req, by_block, new_tokens, static_cast<__half*>(bounds));
  return cudaGetLastError();
}

cudaError_t paged_kv_select(const KvSelect& s, cudaStream_t stream) {
  if (s.req.requests == 0) return cudaSuccess;
  if (s.req.width) {
    const int64_t units = (s.req.width + kTogether - 1ll) / kTogether * s.kv_heads;
    const int64_t items = (units / kScoreWarps + 1) * s.req.requests;
    if (units > INT_MAX || items > INT_MAX || s.req.requests > kMostRequests) return cudaErrorInvalidValue;
    constexpr int kBytes = kScoreWarps * 2 * kTogether * kReach * 4;  // two units, or one of twice the length
    auto score = s.type == kKvBf16 ? (s.dim <= kReach ? score_kernel<__nv_bfloat16, 1> : score_kernel<__nv_bfloat16, 2>)
                                   : (s.dim <= kReach ? score_kernel<__half, 1> : score_kernel<__half, 2>);
    static std::atomic<uint64_t> ready[4];  // devices that know the kernels' shared memory
    const int which = (s.type == kKvBf16) + 2 * (s.dim <= kReach);
    int device = 0, sms = 0;
    cudaError_t rc = sm_count(&sms, &device);
    if (rc != cudaSuccess) return rc;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(ready[which].load(std::memory_order_relaxed) & bit)) {
      rc = cudaFuncSetAttribute(score, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes + (kMostRequests + 1) * 4);
      if (rc != cudaSuccess) return rc;
      ready[which].fetch_or(bit, std::memory_order_relaxed);
    }
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(items, 3 * sms));  // three CTAs to an SM
    score<<<grid, kScoreWarps * 32, kBytes + (s.req.requests + 1) * 4, stream>>>(s, FastDiv::make(s.block), FastDiv::make(s.kv_heads));
    rc = cudaGetLastError();
    if (rc != cudaSuccess) return rc;
  }
  cudaError_t rc = cudaSuccess;
  for_width(s.req.width, [&](auto threads, auto items) {
    rc = launch_after(select_kernel<threads(), items()>, s.req.requests * s.kv_heads, threads(), stream, s);
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
