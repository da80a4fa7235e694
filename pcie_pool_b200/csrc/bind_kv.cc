// Bindings of the paged-KV operators.  Addresses are integers as in bind_ops.cc;
// the calls run on `device`, whatever device is current.
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
  m.attr("KV_BF16") = static_cast<int>(kKvBf16);
  m.attr("KV_FP16") = static_cast<int>(kKvFp16);
  py::class_<PagedKv>(m, "PagedKv")
      .def(py::init([](uint64_t base, int64_t lane, int64_t page, int64_t token, int64_t head, int pages, int block,
                       int kv_heads, int dim, int type) {
        return PagedKv{at<void>(base), lane, page, token, head, pages, block, kv_heads, dim, type};
      }));
  py::class_<KvRequests>(m, "KvRequests")
      .def(py::init([](uint64_t table, int64_t stride, uint64_t lens, int requests, int width) {
        return KvRequests{at<int>(table), stride, at<int>(lens), requests, width};
      }));
  py::class_<KvAttention>(m, "KvAttention")
      .def(py::init([](const PagedKv& kv, const KvRequests& req, uint64_t q, int64_t q_stride, int64_t q_head_stride,
                       int heads, float scale, uint64_t blocks, int blocks_width, uint64_t mass, int64_t mass_stride) {
        KvAttention a;
        a.kv = kv;
        a.req = req;
        a.q = at<void>(q);
        a.q_stride = q_stride;
        a.q_head_stride = q_head_stride;
        a.heads = heads;
        a.scale = scale;
        a.blocks = at<int>(blocks);
        a.blocks_width = blocks_width;
        a.mass = at<float>(mass);
        a.mass_stride = mass_stride;
        return a;
      }))
      .def("work_bytes",
           [](const KvAttention& a, int device) {
             DeviceGuard guard(device);
             return paged_kv_attention_work(a);
           })
      .def("run", [](KvAttention a, uint64_t out, uint64_t lse, uint64_t work, int device, uint64_t stream) {
        DeviceGuard guard(device);
        a.out = at<void>(out);
        a.lse = at<float>(lse);
        a.work = at<void>(work);
        check_cuda(paged_kv_attention(a, at<CUstream_st>(stream)), "paged_kv_attention");
      });
  m.def("paged_kv_bounds",
        [](const PagedKv& kv, const KvRequests& req, int new_tokens, uint64_t bounds, int device, uint64_t stream) {
          DeviceGuard guard(device);
          check_cuda(paged_kv_bounds(kv, req, new_tokens, at<void>(bounds), at<CUstream_st>(stream)),
                     "paged_kv_bounds");
        });
  m.def("paged_kv_select",
        [](const KvRequests& req, uint64_t q, int64_t q_stride, int64_t q_head_stride, int heads, uint64_t bounds,
           int pages, int block, int kv_heads, int dim, int type, int keep, int sink, int recent, uint64_t scores,
           uint64_t out, int device, uint64_t stream) {
          DeviceGuard guard(device);
          KvSelect s;
          s.req = req;
          s.q = at<void>(q);
          s.q_stride = q_stride;
          s.q_head_stride = q_head_stride;
          s.heads = heads;
          s.bounds = at<void>(bounds);
          s.pages = pages;
          s.block = block;
          s.kv_heads = kv_heads;
          s.dim = dim;
          s.type = type;
          s.keep = keep;
          s.sink = sink;
          s.recent = recent;
          s.scores = at<float>(scores);
          s.out = at<int>(out);
          check_cuda(paged_kv_select(s, at<CUstream_st>(stream)), "paged_kv_select");
        });
  m.def("paged_kv_evict",
        [](const KvRequests& req, uint64_t mass, int64_t mass_stride, int block, int budget, int sink, int recent,
           uint64_t new_table, uint64_t new_lens, uint64_t new_mass, uint64_t evicted, uint64_t evicted_at,
           uint64_t evicted_count, int device, uint64_t stream) {
          DeviceGuard guard(device);
          KvEvict e;
          e.req = req;
          e.mass = at<float>(mass);
          e.mass_stride = mass_stride;
          e.block = block;
          e.budget = budget;
          e.sink = sink;
          e.recent = recent;
          e.new_table = at<int>(new_table);
          e.new_lens = at<int>(new_lens);
          e.new_mass = at<float>(new_mass);
          e.evicted = at<int>(evicted);
          e.evicted_at = at<int>(evicted_at);
          e.evicted_count = at<int>(evicted_count);
          check_cuda(paged_kv_evict(e, at<CUstream_st>(stream)), "paged_kv_evict");
        });
}
