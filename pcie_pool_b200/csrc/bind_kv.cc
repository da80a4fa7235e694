// Bindings of the paged-KV operators.  Addresses are integers as in bind_ops.cc;
// the calls run on `device`, whatever device is current.  The arguments stand in
// groups, each in the order of its record in paged_kv.h: the cache (10), the
// requests (5), the queries (4).
#include <pybind11/pybind11.h>

#include "paged_kv.h"
#include "ppb_common.h"

namespace py = pybind11;
using namespace ppb;

namespace {

template <typename T>
T* at(uint64_t p) {
  return reinterpret_cast<T*>(p);
}

}  // namespace

void bind_kv(py::module_& m) {
  m.def("paged_kv_attention_work", [](int requests, int width, int block, int heads, int kv_heads, int dim, bool mass,
                                      int device) {
    DeviceGuard guard(device);
    return paged_kv_attention_work(requests, width, block, heads, kv_heads, dim, mass);
  });
  m.def("paged_kv_attention",
        [](uint64_t base, int64_t lane, int64_t page, int64_t token, int64_t head, int pages, int block, int kv_heads,
           int dim, int type, uint64_t table, int64_t table_stride, uint64_t lens, int requests, int width, uint64_t q,
           int64_t q_stride, int64_t q_head_stride, int heads, float scale, uint64_t blocks, int blocks_width,
           uint64_t mass, int64_t mass_stride, uint64_t out, uint64_t lse, uint64_t work, int device, uint64_t stream) {
          DeviceGuard guard(device);
          KvAttention a;
          a.kv = PagedKv{at<void>(base), lane, page, token, head, pages, block, kv_heads, dim, type};
          a.req = KvRequests{at<int>(table), table_stride, at<int>(lens), requests, width};
          a.q = KvQuery{at<void>(q), q_stride, q_head_stride, heads};
          a.scale = scale;
          a.blocks = at<int>(blocks);
          a.blocks_width = blocks_width;
          a.mass = at<float>(mass);
          a.mass_stride = mass_stride;
          a.out = at<void>(out);
          a.lse = at<float>(lse);
          a.work = at<void>(work);
          check_cuda(paged_kv_attention(a, at<CUstream_st>(stream)), "paged_kv_attention");
        });
  m.def("paged_kv_bounds",
        [](uint64_t base, int64_t lane, int64_t page, int64_t token, int64_t head, int pages, int block, int kv_heads,
           int dim, int type, uint64_t table, int64_t table_stride, uint64_t lens, int requests, int width,
           int new_tokens, uint64_t bounds, int device, uint64_t stream) {
          DeviceGuard guard(device);
          check_cuda(paged_kv_bounds(PagedKv{at<void>(base), lane, page, token, head, pages, block, kv_heads, dim, type},
                                     KvRequests{at<int>(table), table_stride, at<int>(lens), requests, width},
                                     new_tokens, at<void>(bounds), at<CUstream_st>(stream)),
                     "paged_kv_bounds");
        });
  m.def("paged_kv_select",
        [](uint64_t table, int64_t table_stride, uint64_t lens, int requests, int width, uint64_t q, int64_t q_stride,
           int64_t q_head_stride, int heads, uint64_t bounds, int pages, int block, int kv_heads, int dim, int type,
           int keep, int sink, int recent, uint64_t scores, uint64_t out, int device, uint64_t stream) {
          DeviceGuard guard(device);
          const KvSelect s{KvRequests{at<int>(table), table_stride, at<int>(lens), requests, width},
                           KvQuery{at<void>(q), q_stride, q_head_stride, heads},
                           at<void>(bounds), pages, block, kv_heads, dim, type, keep, sink, recent,
                           at<float>(scores), at<int>(out)};
          check_cuda(paged_kv_select(s, at<CUstream_st>(stream)), "paged_kv_select");
        });
  m.def("paged_kv_evict",
        [](uint64_t table, int64_t table_stride, uint64_t lens, int requests, int width, uint64_t mass,
           int64_t mass_stride, int block, int budget, int sink, int recent, uint64_t new_table, uint64_t new_lens,
           uint64_t new_mass, uint64_t evicted, uint64_t evicted_at, uint64_t evicted_count, int device,
           uint64_t stream) {
          DeviceGuard guard(device);
          const KvEvict e{KvRequests{at<int>(table), table_stride, at<int>(lens), requests, width},
                          at<float>(mass), mass_stride, block, budget, sink, recent,
                          at<int>(new_table), at<int>(new_lens), at<float>(new_mass),
                          at<int>(evicted), at<int>(evicted_at), at<int>(evicted_count)};
          check_cuda(paged_kv_evict(e, at<CUstream_st>(stream)), "paged_kv_evict");
        });
}
