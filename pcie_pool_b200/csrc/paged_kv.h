// Operators on a paged KV cache in HBM: attention of one new token per request,
// the key bounds of the cache's pages, the choice of pages for sparse attention,
// and eviction by accumulated attention weight.  Raw addresses and a stream, as
// in native_ops.h; strides are in elements.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace ppb {

constexpr int kMostRequests = 4096;

enum KvType : int { kKvBf16 = 0, kKvFp16 = 1 };

// One layer's cache [2, pages, block, kv_heads, dim]: K, and V `lane_stride`
// behind it.  The last dimension is contiguous; the base and every stride are
// multiples of 16 bytes.
struct PagedKv {
  const void* base = nullptr;
  int64_t lane_stride = 0, page_stride = 0, token_stride = 0, head_stride = 0;
  int pages = 0, block = 0, kv_heads = 0, dim = 0;
  int type = kKvBf16;
};

// At most kMostRequests requests: their block table (int32, `width` entries a row) and lengths.
// An entry outside [0, pages) is a block that is not resident: its tokens are
// left out.  Lengths are cut to the table's width * block.
struct KvRequests {
  const int* table = nullptr;
  int64_t table_stride = 0;
  const int* lens = nullptr;
  int requests = 0, width = 0;
};

// The new tokens' queries [requests, heads, dim]; the last dimension is contiguous,
// pairs of values lie on 4-byte boundaries.
struct KvQuery {
  const void* base = nullptr;
  int64_t stride = 0, head_stride = 0;
  int heads = 0;
};

struct KvAttention {
  PagedKv kv;
  KvRequests req;
  KvQuery q;
  float scale = 0.f;
  const int* blocks = nullptr;  // [requests, kv_heads, blocks_width] or null: every block
  int blocks_width = 0;
  float* mass = nullptr;  // [requests, width] or null
  int64_t mass_stride = 0;
  void* out = nullptr;     // [requests, heads, dim]
  float* lse = nullptr;    // [requests, heads]
  void* work = nullptr;    // paged_kv_attention_work() bytes
};

// Workspace bytes of a call on the current device (nothing that `a` points to is read).
uint64_t paged_kv_attention_work(const KvAttention& a);
cudaError_t paged_kv_attention(const KvAttention& a, cudaStream_t stream);

// Bounds [pages, kv_heads, 2, dim] (smallest, then largest key of each channel) of
// every page that holds one of the last `new_tokens` tokens of its request (all
// pages for new_tokens < 0).
cudaError_t paged_kv_bounds(const PagedKv& kv, const KvRequests& req, int new_tokens, void* bounds,
                            cudaStream_t stream);

struct KvSelect {
  KvRequests req;
  KvQuery q;
  const void* bounds = nullptr;  // [pages, kv_heads, 2, dim] contiguous
  int pages = 0, block = 0, kv_heads = 0, dim = 0, type = kKvBf16;
  int keep = 0, sink = 0, recent = 0;
  float* scores = nullptr;  // workspace [requests, kv_heads, width]
  int* out = nullptr;       // [requests, kv_heads, keep]
};
cudaError_t paged_kv_select(const KvSelect& s, cudaStream_t stream);

struct KvEvict {
  KvRequests req;
  const float* mass = nullptr;
  int64_t mass_stride = 0;
  int pages = 0;  // table entries outside [0, pages) are dropped
  int block = 0, budget = 0, sink = 0, recent = 0;
  int* new_table = nullptr;    // [requests, width]
  int* new_lens = nullptr;     // [requests]
  float* new_mass = nullptr;   // [requests, width]
  int* evicted = nullptr;      // [requests, width] pages
  int* evicted_at = nullptr;   // [requests, width] their places in the old table
  int* evicted_count = nullptr;  // [requests]
};
cudaError_t paged_kv_evict(const KvEvict& e, cudaStream_t stream);

}  // namespace ppb
