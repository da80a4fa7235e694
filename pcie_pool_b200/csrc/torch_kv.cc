// The paged-KV operators' entry points on torch tensors (module pcie_pool_b200._kv):
// checks of arguments, outputs and workspaces, the launch on the tensors' current
// stream.  They are here and not in Python because a call for one request is over in
// 8 us on the device: with checks and allocations in Python it took 17 us of the host's
// time, here it takes 7.7 (eviction 8.9 for 17.7, bounds 3.6 for 7.4).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <limits>
#include <optional>
#include <string>
#include <tuple>

#include "paged_kv.h"
#include "ppb_common.h"

namespace py = pybind11;
using namespace ppb;
using at::Tensor;

namespace {

constexpr int64_t kMaxDim = 256, kMaxBlock = 65536, kMaxMassHeads = 1024, kInt = int64_t(1) << 31;

void need(bool ok, const char* why) {
  if (!ok) throw py::value_error(why);
}

// An integer of Python (truth values are none) from `least` on, below 2^31.
int whole(const py::object& v, int64_t least, const char* why) {
  need(PyLong_Check(v.ptr()) && !PyBool_Check(v.ptr()), why);
  int overflow = 0;
  const long long x = PyLong_AsLongLongAndOverflow(v.ptr(), &overflow);
  need(overflow == 0 && x >= least && x < kInt, why);
  return static_cast<int>(x);
}

KvType type_of(at::ScalarType t) {
  need(t == at::kBFloat16 || t == at::kHalf, "the cache must be bf16 or fp16");
  return t == at::kBFloat16 ? kKvBf16 : kKvFp16;
}

uintptr_t address(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

// The last check of every call: the stream that it runs on.
cudaStream_t stream_of(std::initializer_list<const Tensor*> tensors) {
  const Tensor& t = **tensors.begin();
  if (c10::GradMode::is_enabled())
    for (const Tensor* x : tensors)
      need(!x->requires_grad(), "the paged-KV operators have no gradient: call them under torch.no_grad()");
  need(t.is_cuda(), "the tensors must be on a CUDA device");
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// at::empty without its way through the dispatcher, which is half of its time.
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

KvRequests requests_of(const Tensor& table, const Tensor& lens, const at::Device& device, int64_t block) {
  need(table.scalar_type() == at::kInt && table.dim() == 2, "block_table must be int32 [requests, blocks]");
  const int64_t n = table.size(0), width = table.size(1);
  need(n <= kMostRequests, "at most 4096 requests");
  need(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == n, "context_lens must be int32 [requests]");
  need(table.device() == device && lens.device() == device, "all tensors must be on one CUDA device");
  need(block <= kMaxBlock, "at most 65536 tokens a block");
  need(width <= (kInt - 2 * kMaxBlock) / block, "block_table is too wide: a request has at most 2**31 tokens");
  need(n * width < kInt && n * width * block < int64_t(1) << 34,
       "block_table is too large: at most 2**31 blocks and 2**34 tokens in all");
  need(width <= 1 || table.stride(1) == 1, "block_table's rows must be contiguous");
  need(n <= 1 || lens.stride(0) == 1, "context_lens must be contiguous");
  return {table.data_ptr<int>(), table.stride(0), lens.data_ptr<int>(), static_cast<int>(n), static_cast<int>(width)};
}

PagedKv cache_of(const Tensor& kv) {
  need(kv.dim() == 5 && kv.size(0) == 2, "kv must be [2, pages, block, kv_heads, dim]");
  const KvType type = type_of(kv.scalar_type());
  const int64_t dim = kv.size(4);
  need(dim % 8 == 0 && dim >= 8 && dim <= kMaxDim && kv.size(3) >= 1 && kv.size(2) >= 1,
       "kv's dim must be a multiple of 8 from 8 to 256, and it must have heads and tokens");
  need(kv.size(1) < kInt && kv.size(2) < kInt && kv.size(3) < kInt / kMaxDim, "too many pages, tokens of a page or heads");
  need(kv.stride(4) == 1, "kv's last dimension must be contiguous");
  int64_t strides = 0;  // of a dimension of one nothing is multiplied
  for (int i = 0; i < 4; ++i) strides |= kv.size(i) > 1 ? kv.stride(i) : 0;
  need(address(kv) % 16 == 0 && strides % 8 == 0, "kv's address and strides must be multiples of 16 bytes");
  return {kv.data_ptr(), kv.stride(0), kv.stride(1), kv.stride(2), kv.stride(3), static_cast<int>(kv.size(1)),
          static_cast<int>(kv.size(2)), static_cast<int>(kv.size(3)), static_cast<int>(dim), type};
}

// Pairs of a query are loaded at once: a view that splits them is copied.
Tensor whole_pairs(const Tensor& q) {
  if (q.stride(2) == 1 && address(q) % 4 == 0 && (q.stride(0) | q.stride(1)) % 2 == 0) return q;
  return q.clone(at::MemoryFormat::Contiguous);
}

Tensor query_of(const Tensor& given, const at::Device& device, at::ScalarType type, int64_t dim, int64_t kv_heads,
                int64_t requests, KvQuery& out) {
  need(given.dim() == 3 && given.scalar_type() == type && given.device() == device,
       "q must be [requests, heads, dim] in the cache's type and on its device");
  need(given.size(0) == requests, "q and block_table must have as many requests");
  need(given.size(2) == dim && given.size(1) >= 1 && given.size(1) % kv_heads == 0 && given.size(1) < kInt / kMaxDim,
       "q's dim must be the cache's, and its heads a multiple of the cache's");
  Tensor q = whole_pairs(given);
  out = {q.data_ptr(), q.stride(0), q.stride(1), static_cast<int>(q.size(1))};
  return q;
}

// Tells autograd that a tensor of the caller's is written: a graph that saved it then says so in its backward pass.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Bytes that a tensor spans in its dimensions from `dim` on.
uintptr_t span_of(const Tensor& t, int64_t dim) {
  int64_t last = 0;
  for (int64_t i = dim; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return (last + 1) * t.element_size();
}

// Whether what two tensors span has memory in common.  Requests' parts of one buffer that
// stand next to each other (equal strides of the first dimension) do not.
bool overlaps(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  if (address(a) >= address(b) + span_of(b, 0) || address(b) >= address(a) + span_of(a, 0)) return false;
  if (a.size(0) < 2 || b.size(0) < 2) return true;
  const uintptr_t pitch = a.stride(0) * a.element_size(), row_a = span_of(a, 1), row_b = span_of(b, 1);
  if (pitch != b.stride(0) * b.element_size() || row_a > pitch || row_b > pitch) return true;
  const uintptr_t apart = address(b) >= address(a) ? (address(b) - address(a)) % pitch : (pitch - (address(a) - address(b)) % pitch) % pitch;
  return apart < row_a || apart + row_b > pitch;
}

py::object kv_attention(const Tensor& given, const Tensor& kv, const Tensor& table, const Tensor& lens,
                     std::optional<double> scale, const std::optional<Tensor>& blocks, const std::optional<Tensor>& mass,
                     std::optional<Tensor> out, bool return_lse) {
  KvAttention a;
  a.kv = cache_of(kv);
  const at::Device device = kv.device();
  a.req = requests_of(table, lens, device, a.kv.block);
  const int64_t n = a.req.requests, width = a.req.width;
  const Tensor q = query_of(given, device, kv.scalar_type(), a.kv.dim, a.kv.kv_heads, n, a.q);
  a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(a.kv.dim)));
  if (blocks) {
    need(blocks->scalar_type() == at::kInt && blocks->device() == device && blocks->dim() == 3 && blocks->is_contiguous() &&
             blocks->size(0) == n && blocks->size(1) == a.kv.kv_heads && blocks->size(2) < kInt,
         "blocks must be contiguous int32 [requests, kv_heads, n]");
    a.blocks = blocks->data_ptr<int>();
    a.blocks_width = static_cast<int>(blocks->size(2));
  }
  if (mass) {
    need(!blocks, "mass is gathered over all blocks: it takes no blocks=");
    need(a.q.heads <= kMaxMassHeads, "mass takes at most 1024 heads");
    need(a.kv.block % 16 == 0, "mass needs a block size that is a multiple of 16");
    need(mass->scalar_type() == at::kFloat && mass->device() == device && mass->sizes() == table.sizes(),
         "mass must be fp32 in block_table's shape");
    need((width <= 1 || mass->stride(1) == 1) && (n <= 1 || mass->stride(0) >= width),
         "mass must have contiguous rows of their own");
    need(!overlaps(*mass, q) && !overlaps(*mass, kv) && !overlaps(*mass, table) && !overlaps(*mass, lens),
         "mass must not overlap q, kv, block_table or context_lens");
    a.mass = mass->data_ptr<float>();
    a.mass_stride = mass->stride(0);
  }
  if (out) {
    need(out->scalar_type() == q.scalar_type() && out->device() == device && out->sizes() == q.sizes() &&
             out->is_contiguous() && address(*out) % 4 == 0,
         "out must be contiguous, like q, on a 4-byte boundary");
    need(!overlaps(*out, q) && !overlaps(*out, kv) && !overlaps(*out, table) && !overlaps(*out, lens) &&
             !(blocks && overlaps(*out, *blocks)) && !(mass && overlaps(*out, *mass)),
         "out must not overlap q, kv or another argument");
  }
  const cudaStream_t stream = stream_of({&kv, &q, mass ? &*mass : &kv, out ? &*out : &kv});
  if (out) written(*out);
  if (mass) written(*mass);
  if (!out) out = empty(q.sizes(), q.scalar_type(), device);
  const Tensor lse = empty({n, a.q.heads}, at::kFloat, device);
  if (blocks && a.blocks_width == 0) {
    out->zero_();
    lse.fill_(-INFINITY);
  } else {
    DeviceGuard guard(device.index());
    const int64_t bytes = paged_kv_attention_work(a);
    const Tensor work = empty({bytes}, at::kByte, device);
    a.out = out->data_ptr();
    a.lse = lse.data_ptr<float>();
    a.work = work.data_ptr();
    check_cuda(paged_kv_attention(a, stream), "paged_kv_attention");
  }
  return return_lse ? py::cast(std::make_tuple(*out, lse)) : py::cast(*out);
}

void kv_bounds(const Tensor& kv, const Tensor& table, const Tensor& lens, const Tensor& bounds, const py::object& new_tokens) {
  const PagedKv cache = cache_of(kv);
  const KvRequests req = requests_of(table, lens, kv.device(), cache.block);
  need(bounds.scalar_type() == kv.scalar_type() && bounds.device() == kv.device() && bounds.dim() == 4 &&
           bounds.size(0) == cache.pages && bounds.size(1) == cache.kv_heads && bounds.size(2) == 2 &&
           bounds.size(3) == cache.dim && bounds.is_contiguous() && address(bounds) % 16 == 0,
       "bounds must be contiguous [pages, kv_heads, 2, dim] in the cache's type, on a 16-byte boundary");
  need(!overlaps(bounds, kv) && !overlaps(bounds, table) && !overlaps(bounds, lens),
       "bounds must not overlap kv, block_table or context_lens");
  const int since = !new_tokens.is_none() ? whole(new_tokens, 0, "new_tokens must be an integer >= 0") : -1;
  const cudaStream_t stream = stream_of({&kv, &bounds});
  written(bounds);
  DeviceGuard guard(kv.get_device());
  check_cuda(paged_kv_bounds(cache, req, since, bounds.data_ptr(), stream), "paged_kv_bounds");
}

Tensor kv_select(const Tensor& given, const Tensor& bounds, const Tensor& table, const Tensor& lens, const py::object& keep,
                 const py::object& block, const py::object& sink, const py::object& recent) {
  need(bounds.dim() == 4 && bounds.size(2) == 2 && bounds.is_contiguous() && address(bounds) % 16 == 0,
       "bounds must be contiguous [pages, kv_heads, 2, dim] on a 16-byte boundary");
  KvSelect s;
  const int64_t dim = bounds.size(3);
  s.type = type_of(bounds.scalar_type());
  need(bounds.size(1) >= 1 && bounds.size(1) < kInt / kMaxDim && dim % 8 == 0 && dim >= 8 && dim <= kMaxDim && bounds.size(0) < kInt,
       "bounds' dim must be a multiple of 8 from 8 to 256");
  s.bounds = bounds.data_ptr();
  s.pages = static_cast<int>(bounds.size(0));
  s.kv_heads = static_cast<int>(bounds.size(1));
  s.dim = static_cast<int>(dim);
  s.block = whole(block, 1, "block_size must be an integer >= 1");
  s.req = requests_of(table, lens, bounds.device(), s.block);
  const Tensor q = query_of(given, bounds.device(), bounds.scalar_type(), dim, s.kv_heads, s.req.requests, s.q);
  // a CTA of the selection has a request's key head, a unit of the scores 8 blocks of one
  const int64_t rows = int64_t(s.req.requests) * s.kv_heads, units = (int64_t(s.req.width) + 7) / 8 * s.kv_heads;
  need(rows < kInt && units < kInt - kMaxDim && (units / 8 + 1) * s.req.requests < kInt,
       "too many key heads: at most 2**31 rows of requests and key heads, and 2**34 scores");
  s.keep = whole(keep, 1, "keep must be an integer >= 1");
  s.sink = whole(sink, 0, "sink must be an integer >= 0");
  s.recent = whole(recent, 0, "recent must be an integer >= 0");
  need(int64_t(s.sink) + s.recent <= s.keep, "keep must be at least sink + recent");
  const cudaStream_t stream = stream_of({&bounds, &q});
  const Tensor out = empty({s.req.requests, s.kv_heads, s.keep}, at::kInt, bounds.device());
  const Tensor scores = empty({int64_t(s.req.requests) * s.kv_heads * s.req.width}, at::kFloat, bounds.device());
  s.out = out.data_ptr<int>();
  s.scores = scores.data_ptr<float>();
  DeviceGuard guard(bounds.get_device());
  check_cuda(paged_kv_select(s, stream), "paged_kv_select");
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> kv_evict(const Tensor& mass, const Tensor& table,
                                                                    const Tensor& lens, const py::object& budget,
                                                                    const py::object& block, const py::object& sink,
                                                                    const py::object& recent, const py::object& pages) {
  need(mass.scalar_type() == at::kFloat && mass.sizes() == table.sizes(), "mass must be fp32 in block_table's shape");
  KvEvict e;
  e.block = whole(block, 1, "block_size must be an integer >= 1");
  e.req = requests_of(table, lens, mass.device(), e.block);
  need(e.req.width <= 1 || mass.stride(1) == 1, "mass' rows must be contiguous");
  e.mass = mass.data_ptr<float>();
  e.mass_stride = mass.stride(0);
  e.budget = whole(budget, 1, "budget must be an integer >= 1");
  e.sink = whole(sink, 0, "sink must be an integer >= 0");
  e.recent = whole(recent, 1, "recent must be an integer >= 1");
  need(int64_t(e.sink) + e.recent <= e.budget, "budget must be at least sink + recent");
  e.pages = !pages.is_none() ? whole(pages, 0, "pages must be an integer >= 0") : std::numeric_limits<int>::max();
  const cudaStream_t stream = stream_of({&mass});
  const at::IntArrayRef rows = table.sizes();
  const at::Device device = mass.device();
  const Tensor kept = empty(rows, at::kInt, device), gone = empty(rows, at::kInt, device), places = empty(rows, at::kInt, device);
  const Tensor new_mass = empty(rows, at::kFloat, device);
  const Tensor new_lens = empty(lens.sizes(), at::kInt, device), count = empty(lens.sizes(), at::kInt, device);
  e.new_table = kept.data_ptr<int>();
  e.new_lens = new_lens.data_ptr<int>();
  e.new_mass = new_mass.data_ptr<float>();
  e.evicted = gone.data_ptr<int>();
  e.evicted_at = places.data_ptr<int>();
  e.evicted_count = count.data_ptr<int>();
  DeviceGuard guard(mass.get_device());
  check_cuda(paged_kv_evict(e, stream), "paged_kv_evict");
  return {kept, new_lens, new_mass, gone, places, count};
}

}  // namespace

PYBIND11_MODULE(_kv, m) {
  // torch's C++ classes are laid out by version: a module of another one must not run
  // (the installed package's version, which the build took too; torch.__version__ may say more than it)
  const auto version = py::str(py::module_::import("importlib.metadata").attr("version")("torch")).cast<std::string>();
  if (version != PPB_TORCH)
    throw py::import_error("pcie_pool_b200._kv was built for torch " PPB_TORCH ", this is torch " + version +
                           ": run `python -m pcie_pool_b200._build` and start anew");
  m.doc() = "paged-KV operators on torch tensors (sm_100a kernels)";
  m.def("attention", &kv_attention);
  m.def("bounds", &kv_bounds);
  m.def("select", &kv_select);
  m.def("evict", &kv_evict);
  m.def("whole_pairs", &whole_pairs);
}
