// Attention of one new token per request over a paged KV cache.
//
//   s_t = scale * <q, K_t>,  out = sum_t exp(s_t - lse) V_t,  lse = log sum_t exp(s_t)
//   mass_j += sum over heads and the tokens t of block j of exp(s_t - lse)
//
// Every key and value is read once and used for the G query heads of its key
// head: 2 G flops a byte, so the cache's bytes bound it, not the arithmetic.  A
// warp works alone: it streams tiles of 16 tokens of one key head through its
// own ring of shared memory (cp.async, 16 bytes a lane, pages looked up 32 blocks
// ahead) and keeps the G x dim result in registers with the running maximum
// and sum of the softmax.  No barrier stands in the loop, and tiles of the next
// request are already on their way while the last one is finished.  Consecutive
// warps take the key heads of the same tokens, so a page's rows, which lie next
// to each other, are fetched together.  kv_plan.h says how the tiles are shared
// out and attention_join_kernel adds up what was cut.
//
// The products run on mma.m16n8k16 with the heads as rows: a token's 16 columns
// cost the same whether 1 or 16 heads use them, and at 16 tokens a step the tensor
// pipe is far from its limit (tcgen05's 128 rows would be 4 or 8 heads and
// padding).  Weights are multiplied as two numbers of the cache's type, high part and
// remainder: 16 of their 24 bits in bf16, 22 in fp16, far below the result's own 8 and
// 11 (of 8 x 32768 tokens in bf16, 1.9 results in a thousand are not the nearest to 64
// bits; with all 24 bits it is 0.6).  Their sum, the log-sums and the mass take them
// whole.  fp16 ends at 2^-24,
// so there the weights, at most 1, are multiplied by 2^15 and the result is divided by it:
// what is lost of a weight beside the leading one is 2^-40 of that, not 2^-25.  Up to eight
// heads, the remainders are the eight rows that the heads leave free and cost nothing.
//
// Measured (bf16, 32 heads on 8 key heads of 128, blocks of 16, both kernels, a graph of
// calls over cold data): 8 x 32768 tokens, 1.07 GB, 163 us, 6.59 TB/s, what a copy
// reaches; 64 requests of 91 to 8192 tokens, 462 MB, 83 us; 64 x 1024, 268 MB, 53 us;
// 1 x 16384, 67 MB, 18 us; 1 x 300, 8 us.  What is above the bytes' time is 4 us until
// the first tiles are asked for (lengths, then pages, each a read from memory), 3 us
// where a request ends within a range, and 4 us from the last range's end to the
// join's.  Over a second of such calls the chip is at its power limit and at
// 1.64 GHz; 8 x 32768 tokens then take 177 to 192 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>

#include "device_utils.cuh"
#include "kv_device.cuh"
#include "kv_plan.h"
#include "paged_kv.h"

namespace ppb {
namespace {

using namespace dev;

constexpr int kTile = 16;      // tokens of a step; the mass is gathered by tiles
constexpr int kRowGroup = 16;  // query heads of one warp at most
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Warps of a CTA and tiles in flight of each, by the padded dim: about 192 KiB
// of shared memory, one CTA to an SM.  (Two tiles of dim 128 in place of three are 13%
// slower at 64 x 1024 tokens.)
template <int DP>
struct Shape {
  static constexpr int kWarps = DP == 256 ? 4 : 8;
  static constexpr int kStages = DP == 64 ? 6 : 3;
  static constexpr int kStageBytes = 2 * kTile * DP * 2;  // K, then V
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  // of a thread: a quarter of the SM's registers is left for a CTA of the join (with 255,
  // the join starts later: 9.1 us in place of 8.1 for one request of 300 tokens)
  static constexpr int kRegisters = DP == 256 ? 255 : 192;
};

struct Work {
  float* part_o;        // [2 ranges, groups, rows, dim]
  float2* part_ml;      // [2 ranges, groups, rows]: maximum (base 2) and sum
  int4* items;          // what there may be to join, by request or by cut: request, ranges, first slot
  uint32_t* first;      // [requests + 1], for the mass
  float* z;             // [requests, max_tiles, heads]: log2 of a tile's sum, or null
  int max_tiles;        // of a request
  int mass_ctas;        // of a request
  int most_ranges;
  int shared;           // query heads of a key head
  int groups_each;      // row groups of a key head
  int groups;           // of all key heads
  bool by_cut;          // more requests than cuts: items go by cut
  FastDiv by_ranges, by_block, by_groups, by_groups_each;
  int rows;             // of a group's partial result: 8 or 16
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
struct Type;

template <>
struct Type<__nv_bfloat16> {
  static constexpr float kLift = 1.f;  // what weights are multiplied by before they are split
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<uint32_t&>(v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

template <>
struct Type<__half> {
  static constexpr float kLift = 0x1p15f;
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return reinterpret_cast<uint32_t&>(v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(reinterpret_cast<__half2&>(v));
  }
};

// High part of two lifted weights and what it leaves, as pairs.
template <typename T>
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  x *= Type<T>::kLift;
  y *= Type<T>::kLift;
  hi = Type<T>::pack(x, y);
  const float2 h = Type<T>::unpack(hi);
  lo = Type<T>::pack(x - h.x, y - h.y);
}

// Tiles of the blocks of a request that are read: all that hold tokens, or the
// listed ones.
__device__ __forceinline__ uint32_t tiles_of(const KvAttention& a, const Work& w, int len) {
  const int n = w.by_block.quotient(len + a.kv.block - 1);
  const uint32_t slots = a.blocks != nullptr && a.blocks_width < n ? a.blocks_width : n;
  return (slots * a.kv.block + kTile - 1) / kTile;
}

// What the kernels behind need to know, and the results of requests without tokens;
// the warps of all CTAs take the requests (or the cuts) in turn.
template <typename T>
__device__ __forceinline__ void note_items(const KvAttention& a, const Work& w, const uint32_t* first, const KvPlan& plan) {
  const int lane = threadIdx.x % 32, n = a.req.requests;
  const int warp = threadIdx.x / 32 * gridDim.x + blockIdx.x, warps = gridDim.x * (blockDim.x / 32);
  for (int b = warp; b < n; b += warps) {
    if (w.z != nullptr && lane == 0) w.first[b] = first[b];
    if (first[b] == first[b + 1]) {
      T* out = static_cast<T*>(a.out) + static_cast<long long>(b) * a.q.heads * a.kv.dim;
      for (int i = 2 * lane; i < a.q.heads * a.kv.dim; i += 64) *reinterpret_cast<uint32_t*>(out + i) = 0u;
      for (int i = lane; i < a.q.heads; i += 32) a.lse[static_cast<long long>(b) * a.q.heads + i] = -INFINITY;
    }
  }
  if (w.z != nullptr && warp == 0 && lane == 0) w.first[n] = first[n];
  const int items = w.by_cut ? w.most_ranges - 1 : n;
  for (int i = warp + lane * warps; i < items; i += warps * 32) {
    int4 v = make_int4(0, 0, 0, 0);  // nothing to join
    v.x = w.by_cut ? i + 1 < plan.ranges ? request_of(first, n, plan.begin(i + 1)) : -1 : i;
    if (v.x >= 0 && first[v.x] < first[v.x + 1]) {
      v.y = plan.of(first[v.x]);
      v.z = plan.of(first[v.x + 1] - 1);
      // the first part may lie in its range's second place, the others lie in the first
      v.w = plan.slot(v.y, first[v.x]);
      if (w.by_cut && v.y != i) v.z = v.y;  // not its request's first cut
    }
    w.items[i] = v;
  }
}

// DP: dim padded to 64, 128 or 256.  PACKED: at most eight heads share a key head,
// rows 8 to 15 carry the weights' remainders.  MASS: the tiles' sums are kept.
template <typename T, int DP, bool PACKED, bool MASS>
__global__ void __maxnreg__(Shape<DP>::kRegisters)
    attention_kernel(const __grid_constant__ KvAttention a, const __grid_constant__ Work w) {
  using S = Shape<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t scratch[S::kWarps];
  __shared__ uint32_t valid_of[S::kWarps][S::kStages];
  uint32_t* first = reinterpret_cast<uint32_t*>(smem + S::kRingBytes);
  int* lens = reinterpret_cast<int*>(first + a.req.requests + 1);
  const uint32_t warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int D = a.kv.dim, bs = a.kv.block, G = w.shared, n = a.req.requests;
  launch_dependents();
  if (D < DP)  // what the copies leave of a row stays zero
    for (int i = threadIdx.x; i < S::kRingBytes / 16; i += blockDim.x)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  running_sums(n, [&](int b) { return tiles_of(a, w, lens[b] = length_of(a.req, bs, b)); }, first, scratch);
  const KvPlan plan = KvPlan::make(first[n], w.by_ranges);
  const uint32_t units = static_cast<uint32_t>(plan.ranges) * w.groups;
  // few units: one to a CTA before two
  const uint32_t per_cta = min(static_cast<uint32_t>(S::kWarps), (units + gridDim.x - 1) / gridDim.x);
  const uint32_t unit0 = blockIdx.x * per_cta + warp;
  if (warp >= per_cta || unit0 >= units) {
    note_items<T>(a, w, first, plan);
    return;
  }
  const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStageBytes;

  for (uint32_t unit = unit0; unit < units; unit += gridDim.x * per_cta) {
    const int r = static_cast<int>(w.by_groups.quotient(unit)), group = static_cast<int>(unit) - r * w.groups;
    const int g = w.by_groups_each.quotient(group), row0 = (group - g * w.groups_each) * kRowGroup;
    const int rows = min(kRowGroup, G - row0);
    const uint32_t lo = plan.begin(r), hi = plan.begin(r + 1);
    const T* cache = static_cast<const T*>(a.kv.base) + g * a.kv.head_stride;

    float o[DP / 8][4], m[2], l[2];
    uint32_t q[DP / 16][4] = {};
    const float to_base2 = a.scale * kLog2e;
    int b = request_of(first, n, lo);
    uint32_t end = 0;  // of request b's tiles

    // A window is 32 neighbouring blocks of a request, a lane each: their pages, and
    // how many tokens of each count.  The next window is looked up while this one is
    // used.
    struct Window {
      int b, slot;   // its request and first block
      uint32_t end;  // of the tiles that lie in it
      int page, tokens;  // of this lane's block
    };
    auto look_up = [&](uint32_t tile, int request) {
      Window v;
      v.b = request;
      v.end = tile;
      v.slot = v.tokens = 0;
      v.page = -1;
      if (tile >= hi) return v;
      while (first[v.b + 1] <= tile) ++v.b;
      const int len = lens[v.b], blocks = w.by_block.quotient(len + bs - 1);
      v.slot = static_cast<int>(w.by_block.quotient((tile - first[v.b]) * kTile));
      int block = v.slot + lane;
      if (a.blocks != nullptr)
        block = block < min(blocks, a.blocks_width)
                    ? a.blocks[(static_cast<long long>(v.b) * a.kv.kv_heads + g) * a.blocks_width + block]
                    : -1;
      if (block >= 0 && block < blocks) {
        v.tokens = min(bs, len - block * bs);
        v.page = a.req.table[v.b * a.req.table_stride + block];
      }
      const long long tiles = (v.slot + 32ll) * bs / kTile;  // whose blocks all lie in the window
      v.end = static_cast<uint32_t>(min(first[v.b] + tiles, static_cast<long long>(min(first[v.b + 1], hi))));
      return v;
    };
    Window next = look_up(lo, b), now = next;
    if (unit == unit0) {  // while the first blocks are looked up
      note_items<T>(a, w, first, plan);
      __syncwarp();
    }
    now.end = lo;

    // Keys and values have rings of kStages tiles each: the keys of a tile are asked
    // for kStages tiles ahead, its values kStages - 1, each as soon as its place has
    // been read, so that 2 kStages - 1 of the 2 kStages places are always on their way.
    // One loop does copies and products, so that no code stands twice: at the
    // start of a kernel instructions come from memory too, and wait in line with the
    // first tiles.
    constexpr int kChunks = DP / 8;  // 16-byte pieces of a row
    long long row_at = 0;  // where lane & 15's row of the tile asked for last begins
    uint32_t rows_ok = 0;
    auto copy = [&](uint32_t to, long long from) {
#pragma unroll
      for (int i = 0; i < kTile * kChunks / 32; ++i) {
        const int row = (i * 32 + lane) / kChunks, chunk = (i * 32 + lane) % kChunks;
        const T* src = cache + from + __shfl_sync(0xffffffffu, row_at, row) + chunk * 8;
        const bool ok = rows_ok >> row & 1;
        if (chunk * 8 < D) cp_async16(to + row * DP * 2 + ((chunk ^ (row & 7)) * 16), ok ? src : a.kv.base, ok);
      }
    };
    int stage = 0, into = 0;  // places of `tile` and `ahead`
    for (uint32_t ahead = lo; ahead < hi + S::kStages; ++ahead) {
      const uint32_t tile = ahead - S::kStages;  // whose products are taken, if ahead >= lo + kStages
      const bool takes = ahead >= lo + S::kStages;
      if (ahead == lo || (takes && tile >= end)) {  // a request's first: its heads' rows
        while (first[b + 1] <= (takes ? tile : lo)) ++b;
        end = first[b + 1];
        const T* qp = static_cast<const T*>(a.q.base) + b * a.q.stride + (g * G + row0) * a.q.head_stride;
        qp += (lane / 4) * a.q.head_stride + (lane & 3) * 2;
#pragma unroll
        for (int x = 0; x < (PACKED ? 1 : 2); ++x) {
          const bool on = lane / 4 + 8 * x < rows;
          const T* at = qp + 8 * x * a.q.head_stride;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            q[k][x] = on && (D == DP || k * 16 < D) ? *reinterpret_cast<const uint32_t*>(at + k * 16) : 0u;
            q[k][x + 2] = on && (D == DP || k * 16 + 8 < D) ? *reinterpret_cast<const uint32_t*>(at + k * 16 + 8) : 0u;
          }
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
      }
      if (takes) {
        cp_wait<2 * S::kStages - 2>();  // the tile's keys
        __syncwarp();
      }
      // the values of the tile whose keys were asked for in the last step, into the
      // place that the last step's products emptied
      if (ahead > lo && ahead <= hi) copy(ring + (into == 0 ? S::kStages - 1 : into - 1) * S::kStageBytes + kTile * DP * 2, a.kv.lane_stride);
      cp_commit();
      float s[2][4] = {};
      constexpr int kHalves = PACKED ? 1 : 2;  // row lane / 4, and the one eight below
      uint32_t p[4], rest[4];
      if (takes) {
        const uint32_t ok = valid_of[warp][stage];
        const uint32_t ks = ring + stage * S::kStageBytes;
        {
          const int row = (lane & 7) + ((lane >> 4) << 3);
          const uint32_t base = ks + row * DP * 2;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            uint32_t f[4];
            ldsm4(f, base + (((2 * k + ((lane >> 3) & 1)) ^ (row & 7)) * 16));
            Type<T>::mma(s[0], q[k], f[0], f[1]);
            Type<T>::mma(s[1], q[k], f[2], f[3]);
          }
        }
        bool grew = false;
        float ratio[2];
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int col = (lane & 3) * 2 + (i & 1) + (i >> 1) * 8;
            float& v = s[i >> 1][2 * x + (i & 1)];
            v = ok >> col & 1 ? v * to_base2 : -INFINITY;
            top = fmaxf(top, v);
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[x], top), at = now == -INFINITY ? 0.f : now;
          ratio[x] = ex2(m[x] - at);
          grew |= now > m[x];
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& v = s[i >> 1][2 * x + (i & 1)];
            v = ex2(v - at);
            sum += v;
          }
          m[x] = now;
          l[x] = l[x] * ratio[x] + sum;  // of this lane's columns
          if (MASS) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = lane / 4 + 8 * x;
            if ((lane & 3) == 0 && row < rows)
              w.z[(static_cast<long long>(b) * w.max_tiles + (tile - first[b])) * a.q.heads + g * G + row0 + row] = at + lg2(sum);
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][0] *= ratio[0];
            o[i][1] *= ratio[0];
            o[i][2] *= ratio[kHalves - 1];
            o[i][3] *= ratio[kHalves - 1];
          }
        }
        if constexpr (PACKED) {
          split<T>(s[0][0], s[0][1], p[0], p[1]);
          split<T>(s[1][0], s[1][1], p[2], p[3]);
        } else {
          split<T>(s[0][0], s[0][1], p[0], rest[0]);
          split<T>(s[0][2], s[0][3], p[1], rest[1]);
          split<T>(s[1][0], s[1][1], p[2], rest[2]);
          split<T>(s[1][2], s[1][3], p[3], rest[3]);
        }
        cp_wait<2 * S::kStages - 2>();  // its values
        __syncwarp();
      }
      if (ahead < hi) {  // the keys of the tile kStages ahead, into the place of this one's
        const bool entered = ahead >= now.end;  // the next window
        if (entered) now = next;
        const uint32_t t = (ahead - first[now.b]) * kTile + (lane & 15);
        const int slot = static_cast<int>(w.by_block.quotient(t)), off = static_cast<int>(t) - slot * bs;
        const int page = __shfl_sync(0xffffffffu, now.page, slot - now.slot);
        const bool ok = off < __shfl_sync(0xffffffffu, now.tokens, slot - now.slot) && page >= 0 && page < a.kv.pages;
        row_at = ok ? page * a.kv.page_stride + off * a.kv.token_stride : 0;
        rows_ok = __ballot_sync(0xffffffffu, ok) & 0xffffu;
        if (lane == 0) valid_of[warp][into] = rows_ok;
        copy(ring + into * S::kStageBytes, 0);
        if (entered) {
          const int d = lane * 64;  // of its heads' rows, 128 bytes a lane
          if (d < rows * D)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const T*>(a.q.base) + now.b * a.q.stride +
                                                          (g * G + row0 + d / D) * a.q.head_stride + d % D));
          next = look_up(now.end, now.b);
        }
      }
      cp_commit();
      into = into + 1 == S::kStages ? 0 : into + 1;
      if (!takes) continue;
      const uint32_t vs = ring + stage * S::kStageBytes + kTile * DP * 2;
      {
        const int row = lane & 15;
        const uint32_t base = vs + row * DP * 2;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t f[4];
          ldsm4_t(f, base + (((2 * k + (lane >> 4)) ^ (row & 7)) * 16));
          Type<T>::mma(o[2 * k], p, f[0], f[1]);
          Type<T>::mma(o[2 * k + 1], p, f[2], f[3]);
          if constexpr (!PACKED) {
            Type<T>::mma(o[2 * k], rest, f[0], f[1]);
            Type<T>::mma(o[2 * k + 1], rest, f[2], f[3]);
          }
        }
      }
      stage = stage + 1 == S::kStages ? 0 : stage + 1;

      if (tile + 1 == end || tile + 1 == hi) {  // the request's or the range's last
        const bool whole = first[b] >= lo && end <= hi;
        const int slot = plan.slot(r, first[b]);
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          const int row = lane / 4 + 8 * x;
          float sum = l[x];
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (row >= rows) continue;
          const int h = g * G + row0 + row;
          const long long at = static_cast<long long>(slot) * w.groups * w.rows + static_cast<long long>(group) * w.rows + row;
          if ((lane & 3) == 0) {
            if (whole)
              a.lse[static_cast<long long>(b) * a.q.heads + h] = sum == 0.f ? -INFINITY : (m[x] + lg2(sum)) * kLn2;
            else
              w.part_ml[at] = make_float2(m[x], sum);
          }
          // (a loop for each: the branch within one loop made a request's end 1 us longer)
          if (whole) {
            const float by = sum == 0.f ? 0.f : 1.f / Type<T>::kLift / sum;
            T* to = static_cast<T*>(a.out) + (static_cast<long long>(b) * a.q.heads + h) * D + (lane & 3) * 2;
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) {
              const float u = PACKED ? o[i][0] + o[i][2] : o[i][2 * x], v = PACKED ? o[i][1] + o[i][3] : o[i][2 * x + 1];
              if (D == DP || i * 8 < D) *reinterpret_cast<uint32_t*>(to + i * 8) = Type<T>::pack(sum == 0.f ? 0.f : u * by, sum == 0.f ? 0.f : v * by);
            }
          } else {
            float* to = w.part_o + at * D + (lane & 3) * 2;
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) {
              const float u = PACKED ? o[i][0] + o[i][2] : o[i][2 * x], v = PACKED ? o[i][1] + o[i][3] : o[i][2 * x + 1];
              if (D == DP || i * 8 < D)
                *reinterpret_cast<float2*>(to + i * 8) = make_float2(u * (1.f / Type<T>::kLift), v * (1.f / Type<T>::kLift));
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();
  }
}

constexpr int kJoinWarps = 8, kJoinParts = 5;

struct Join {
  uint32_t ctas;       // that join; the others add the mass
  uint32_t ctas_each;  // of a request, or of a cut
  int units_each;
};

// The mass of kMassBlocks blocks of a request, a warp for each: the sums of its
// tiles for every head (they lie together) over the heads' totals.  The totals of
// a request that was cut are taken from its parts, eight lanes for a head, since
// the join beside it only writes them now; the tiles' sums and the old mass are on
// their way meanwhile.  It adds 2 to 3 us to a call (64 x 1024 tokens: 53 and 55 us).
// A tile's sum waits as its logarithm (base 2, fp32), since the heads' totals are known
// only at the end: half a step of that is what a weight is off by, as it is by half a step
// of its score.  CTAs go by the table's width: 256 x 100 tokens take 34 us with 7 columns, 61
// with 1024, 239 with 8192, where most find nothing to do.
constexpr int kMassBlocks = kJoinWarps, kMassHeads = 1024, kMassAhead = 8;

__device__ __forceinline__ void add_mass(const KvAttention& a, const Work& w, uint32_t cta) {
  __shared__ float total[kMassHeads];
  const int b = cta / w.mass_ctas, j = (cta - b * w.mass_ctas) * kMassBlocks + threadIdx.x / 32;
  const int lane = threadIdx.x % 32, H = a.q.heads, per = a.kv.block / kTile;
  const int G = w.shared, per_head = w.groups_each;
  wait_for_parent();
  const uint32_t f0 = w.first[b], f1 = w.first[b + 1];  // a request's tiles are all its blocks'
  const int t0 = j * per, blocks = (f1 - f0 + per - 1) / per;
  if (j - static_cast<int>(threadIdx.x / 32) >= blocks) return;
  const int count = j < blocks ? min(per, static_cast<int>(f1 - f0) - t0) * H : 0;
  const float* z = w.z + (static_cast<long long>(b) * w.max_tiles + t0) * H;
  float* mass = a.mass + b * a.mass_stride + j;
  float ahead[kMassAhead], old = 0.f;
#pragma unroll
  for (int i = 0; i < kMassAhead; ++i) ahead[i] = i * 32 + lane < count ? z[i * 32 + lane] : -INFINITY;
  if (j < blocks) old = *mass;
  const KvPlan plan = KvPlan::make(w.first[a.req.requests], w.by_ranges);
  const int r0 = plan.of(f0), r1 = plan.of(f1 - 1), slot0 = plan.slot(r0, f0);
  for (int h = threadIdx.x / 8; h < (H + 3) / 4 * 4; h += kJoinWarps * 4) {  // whole warps: they shuffle
    float m = -INFINITY, l = 0.f;
    if (r0 == r1) {
      if (h < H) m = a.lse[static_cast<long long>(b) * H + h] * kLog2e, l = 1.f;
    } else {
      const long long base = static_cast<long long>(h / G * per_head + h % G / kRowGroup) * w.rows + h % G % kRowGroup;
      const long long step = static_cast<long long>(w.groups) * w.rows;
#pragma unroll 4
      for (int r = r0 + (lane & 7); r <= r1; r += 8) {
        const float2 ml = h < H ? w.part_ml[base + step * (r == r0 ? slot0 : 2 * r)] : make_float2(-INFINITY, 0.f);
        const float now = fmaxf(m, ml.x), ref = now == -INFINITY ? 0.f : now;
        l = l * ex2(m - ref) + ml.y * ex2(ml.x - ref);
        m = now;
      }
#pragma unroll
      for (int x = 4; x > 0; x /= 2) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, x), now = fmaxf(m, m2), ref = now == -INFINITY ? 0.f : now;
        l = l * ex2(m - ref) + __shfl_xor_sync(0xffffffffu, l, x) * ex2(m2 - ref);
        m = now;
      }
    }
    if ((lane & 7) == 0 && h < H) total[h] = l == 0.f ? -INFINITY : m + lg2(l);
  }
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMassAhead; ++i)
    if (ahead[i] != -INFINITY) sum += ex2(ahead[i] - total[(i * 32 + lane) % H]);
  for (int i = kMassAhead * 32 + lane; i < count; i += 32) {
    const float v = z[i];
    if (v != -INFINITY) sum += ex2(v - total[i % H]);
  }
  sum = warp_sum(sum);
  if (j < blocks && lane == 0) *mass = old + sum;
}

// Adds up what the ranges left of a request that was cut.  There are no more cuts
// than ranges: with few requests a CTA goes by a request, with many by a range's
// begin, and is the one to work if that is the first cut of its request.  Its warps
// share `units_each` units, 4 * LANES columns of a query head; LANES lanes take a part
// and a warp 32 / LANES * kJoinParts parts at a time.  With LANES = 8 that is 160 for a
// CTA: all parts of a request that lies over all SMs are in flight at once.  With a CTA
// for each request and head, 1024 requests of 16 tokens took 96 us, this way 35 (26 now).
template <typename T, int LANES, bool MASS>
__global__ void __launch_bounds__(kJoinWarps * 32, 4)
    attention_join_kernel(const __grid_constant__ KvAttention a, const __grid_constant__ Work w, const __grid_constant__ Join j) {
  if (MASS && blockIdx.x >= j.ctas) {
    add_mass(a, w, blockIdx.x - j.ctas);
    return;
  }
  const int units_each = j.units_each, item = blockIdx.x / j.ctas_each;
  constexpr int kColumns = 4 * LANES, kAtOnce = 32 / LANES;
  __shared__ __align__(16) float sum_o[kJoinWarps][kColumns];
  __shared__ float sum_m[kJoinWarps], sum_l[kJoinWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps_each = kJoinWarps / units_each, mine = warp % warps_each;
  const int D = a.kv.dim, G = w.shared, per_head = w.groups_each;
  const int chunks = (D + kColumns - 1) / kColumns, unit = (blockIdx.x - item * j.ctas_each) * units_each + warp / warps_each;
  const int h = unit / chunks, d = unit % chunks * kColumns + lane % LANES * 4;
  const bool on = h < a.q.heads && d < D;
  // the place of head h's row in a part, and the parts' distance
  const long long base = static_cast<long long>(h / G * per_head + h % G / kRowGroup) * w.rows + h % G % kRowGroup;
  const long long step = static_cast<long long>(w.groups) * w.rows;
  wait_for_parent();
  const int4 found = w.items[item];
  const int b = found.x, r0 = found.y, r1 = found.z, slot0 = found.w;
  if (r0 == r1) return;  // finished where it was computed
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  int r = r0 + mine * kAtOnce * kJoinParts + lane / LANES;
  do {
    float2 ml[kJoinParts];
    float4 v[kJoinParts];
#pragma unroll
    for (int k = 0; k < kJoinParts; ++k) {
      const int x = r + kAtOnce * k;
      const long long at = base + step * (x == r0 ? slot0 : 2 * x);
      ml[k] = make_float2(-INFINITY, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (x <= r1 && on) {
        ml[k] = w.part_ml[at];
        v[k] = *reinterpret_cast<const float4*>(w.part_o + at * D + d);
      }
    }
    float now = m;
#pragma unroll
    for (int k = 0; k < kJoinParts; ++k) now = fmaxf(now, ml[k].x);
    const float ref = now == -INFINITY ? 0.f : now, c = ex2(m - ref);
    m = now;
    l *= c;
    o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
#pragma unroll
    for (int k = 0; k < kJoinParts; ++k) {
      const float p = ex2(ml[k].x - ref);
      l += ml[k].y * p;
      o = make_float4(o.x + v[k].x * p, o.y + v[k].y * p, o.z + v[k].z * p, o.w + v[k].w * p);
    }
    r += warps_each * kAtOnce * kJoinParts;
  } while (r - lane / LANES <= r1);
  // the groups of lanes, then the warps
#pragma unroll
  for (int x = LANES; x < 32; x *= 2) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, x), now = fmaxf(m, m2), ref = now == -INFINITY ? 0.f : now;
    const float p = ex2(m - ref), p2 = ex2(m2 - ref);
    m = now;
    l = l * p + __shfl_xor_sync(0xffffffffu, l, x) * p2;
    o.x = o.x * p + __shfl_xor_sync(0xffffffffu, o.x, x) * p2;
    o.y = o.y * p + __shfl_xor_sync(0xffffffffu, o.y, x) * p2;
    o.z = o.z * p + __shfl_xor_sync(0xffffffffu, o.z, x) * p2;
    o.w = o.w * p + __shfl_xor_sync(0xffffffffu, o.w, x) * p2;
  }
  if (warps_each > 1) {
    if (lane == 0) sum_m[warp] = m, sum_l[warp] = l;
    if (lane < LANES) *reinterpret_cast<float4*>(&sum_o[warp][lane * 4]) = o;
    __syncthreads();
    const int w0 = warp - mine;
    float top = -INFINITY;
    for (int i = 0; i < warps_each; ++i) top = fmaxf(top, sum_m[w0 + i]);
    const float ref = top == -INFINITY ? 0.f : top;
    m = top;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < warps_each; ++i) {
      const float p = ex2(sum_m[w0 + i] - ref);
      const float4 v = *reinterpret_cast<const float4*>(&sum_o[w0 + i][lane % LANES * 4]);
      l += p * sum_l[w0 + i];
      o = make_float4(o.x + v.x * p, o.y + v.y * p, o.z + v.z * p, o.w + v.w * p);
    }
  }
  if (mine != 0 || lane >= LANES || !on) return;
  const long long row = static_cast<long long>(b) * a.q.heads + h;
  const uint32_t lo = l == 0.f ? 0u : Type<T>::pack(o.x / l, o.y / l), hi = l == 0.f ? 0u : Type<T>::pack(o.z / l, o.w / l);
  T* out = static_cast<T*>(a.out) + row * D + d;
  *reinterpret_cast<uint32_t*>(out) = lo;
  *reinterpret_cast<uint32_t*>(out + 2) = hi;
  if (d == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + lg2(l)) * kLn2;
}

int padded(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// The workspace's parts behind a.work; returns its size.
uint64_t lay_out(const KvAttention& a, int sms, Work& w) {
  const int dim = a.kv.dim, heads = a.q.heads, requests = a.req.requests, G = heads / a.kv.kv_heads;
  const int warps = sms * (padded(dim) == 256 ? Shape<256>::kWarps : Shape<128>::kWarps);
  w.shared = G;
  w.groups_each = (G + kRowGroup - 1) / kRowGroup;
  w.groups = a.kv.kv_heads * w.groups_each;
  w.rows = G <= 8 ? 8 : 16;
  w.most_ranges = warps / w.groups > 0 ? warps / w.groups : 1;
  w.by_ranges = FastDiv::make(w.most_ranges);
  w.by_block = FastDiv::make(a.kv.block);
  w.by_groups = FastDiv::make(w.groups);
  w.by_groups_each = FastDiv::make(w.groups_each);
  w.max_tiles = static_cast<int>((static_cast<int64_t>(a.req.width) * a.kv.block + kTile - 1) / kTile);
  w.mass_ctas = a.mass ? (a.req.width + kMassBlocks - 1) / kMassBlocks : 0;
  w.by_cut = requests >= w.most_ranges;
  const uint64_t parts = 2ull * w.most_ranges * w.groups * w.rows;
  uint8_t* p = static_cast<uint8_t*>(a.work);
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    uint8_t* here = p + at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  w.part_o = reinterpret_cast<float*>(take(parts * dim * 4));
  w.part_ml = reinterpret_cast<float2*>(take(parts * 8));
  w.first = reinterpret_cast<uint32_t*>(take((requests + 1ull) * 4));
  w.items = reinterpret_cast<int4*>(take((w.by_cut ? w.most_ranges : requests) * 16ull));
  w.z = a.mass ? reinterpret_cast<float*>(take(uint64_t(requests) * w.max_tiles * heads * 4)) : nullptr;
  return at;
}

template <typename T, int DP>
cudaError_t launch(const KvAttention& a, const Work& w, int sms, int device, cudaStream_t stream) {
  const int smem = Shape<DP>::kRingBytes + (2 * a.req.requests + 1) * 4, threads = Shape<DP>::kWarps * 32;
  auto kernel = w.rows == 8 ? (w.z ? attention_kernel<T, DP, true, true> : attention_kernel<T, DP, true, false>)
                            : (w.z ? attention_kernel<T, DP, false, true> : attention_kernel<T, DP, false, false>);
  const int which = (w.rows == 8) + 2 * (w.z != nullptr);
  static_assert(Shape<DP>::kRingBytes + (2 * kMostRequests + 1) * 4 <= 226 * 1024, "more shared memory than an SM has");
  static std::atomic<uint64_t> ready[4];  // devices that know the kernels' shared memory
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  cudaError_t rc = cudaSuccess;
  if (!(ready[which].load(std::memory_order_relaxed) & bit)) {
    rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Shape<DP>::kRingBytes + (2 * kMostRequests + 1) * 4);
    if (rc != cudaSuccess) return rc;
    ready[which].fetch_or(bit, std::memory_order_relaxed);
  }
  kernel<<<sms, threads, smem, stream>>>(a, w);
  rc = cudaGetLastError();
  if (rc != cudaSuccess) return rc;
  Join j;
  const uint32_t items = w.by_cut ? w.most_ranges - 1 : a.req.requests;
  // narrow units while the CTAs fit beside the attention's, else whole rows, and
  // as many warps for a unit as leave two CTAs to an SM (1 x 16384 tokens: 20.6 us with
  // narrow units, 24.2 with rows; 8 x 300: 20.3 with 1024 narrow CTAs, 12.6 this way; 18.1 and 10.2 now)
  auto join = w.z ? attention_join_kernel<T, 8, true> : attention_join_kernel<T, 8, false>;
  auto share_out = [&](int columns, int64_t most) {
    const int units = a.q.heads * ((a.kv.dim + columns - 1) / columns);
    for (j.units_each = 1;; j.units_each *= 2) {
      j.ctas_each = (units + j.units_each - 1) / j.units_each;
      if (j.units_each == kJoinWarps || static_cast<int64_t>(items) * j.ctas_each <= most) break;
    }
    j.ctas = items * j.ctas_each;
    return static_cast<int64_t>(items) * j.ctas_each <= most;
  };
  if (!share_out(32, sms)) {
    join = w.z ? attention_join_kernel<T, 32, true> : attention_join_kernel<T, 32, false>;
    share_out(128, 2 * sms);
  }
  const uint32_t ctas = j.ctas + static_cast<uint32_t>(a.req.requests) * w.mass_ctas;
  if (ctas == 0) return cudaSuccess;
  return launch_after(join, ctas, kJoinWarps * 32, stream, a, w, j);
}

template <typename T>
cudaError_t launch(const KvAttention& a, const Work& w, int sms, int device, cudaStream_t stream) {
  switch (padded(a.kv.dim)) {
    case 64: return launch<T, 64>(a, w, sms, device, stream);
    case 128: return launch<T, 128>(a, w, sms, device, stream);
    default: return launch<T, 256>(a, w, sms, device, stream);
  }
}

}  // namespace

uint64_t paged_kv_attention_work(const KvAttention& a) {
  int sms = 0, device = 0;
  Work w;
  return sm_count(&sms, &device) == cudaSuccess ? lay_out(a, sms, w) : 0;
}

cudaError_t paged_kv_attention(const KvAttention& a, cudaStream_t stream) {
  if (a.req.requests == 0) return cudaSuccess;
  if (a.req.requests > kMostRequests) return cudaErrorInvalidValue;
  int sms = 0, device = 0;
  cudaError_t rc = sm_count(&sms, &device);
  if (rc != cudaSuccess) return rc;
  Work w;
  lay_out(a, sms, w);
  rc = a.kv.type == kKvBf16 ? launch<__nv_bfloat16>(a, w, sms, device, stream)
                             : launch<__half>(a, w, sms, device, stream);
  return rc;
}

}  // namespace ppb
