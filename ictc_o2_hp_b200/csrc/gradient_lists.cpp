// Lists of tensors to the C ABI's gradient norm and clipping: argument checks, copies of what
// the kernels cannot address, allocation.  In C++ because a call takes hundreds of tensors,
// whose addresses and sizes Python would read one attribute at a time.
#include <ATen/MemoryOverlap.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "ictc_o2_b200.h"

namespace {

using at::Tensor;

struct Api {
  decltype(&ictc_o2_last_error) last_error;
  decltype(&ictc_o2_grad_norm_workspace) workspace;
  decltype(&ictc_o2_grad_norm) norm;
  decltype(&ictc_o2_clip_grads) clip;
};

Api api{};

void check(int32_t status, const char* what) {
  if (status == ICTC_OK) return;
  const std::string message = std::string(what) + ": " + api.last_error();
  TORCH_CHECK_VALUE(status != ICTC_ERR_INVALID, message);
  TORCH_CHECK_NOT_IMPLEMENTED(status != ICTC_ERR_UNSUPPORTED, message);
  TORCH_CHECK(false, message);
}

// A Python sequence of tensors (or one tensor), read where it lies.
class Sequence {
 public:
  Sequence(const char* what, py::handle given) : what_(what) {
    if (THPVariable_Check(given.ptr())) {
      items_ = py::make_tuple(given);
    } else {
      items_ = py::reinterpret_steal<py::object>(PySequence_Fast(given.ptr(), "expected tensors"));
      if (!items_) throw py::error_already_set();
    }
    size_ = static_cast<size_t>(PySequence_Fast_GET_SIZE(items_.ptr()));
  }
  size_t size() const { return size_; }
  const Tensor& operator[](size_t i) const {
    PyObject* item = PySequence_Fast_GET_ITEM(items_.ptr(), static_cast<Py_ssize_t>(i));
    TORCH_CHECK_TYPE(THPVariable_Check(item), what_, " takes tensors, got ", Py_TYPE(item)->tp_name);
    return THPVariable_Unpack(item);
  }
  const py::object& items() const { return items_; }

 private:
  const char* what_;
  py::object items_;
  size_t size_;
};

// Which calls the dispatcher has to see (a trace, fake tensors).  Asked of each tensor just
// before it is read, in the one pass over a list: a list of thousands does not stay in the
// CPU's caches for a second.
class Watch {
 public:
  Watch() {
    const auto local = c10::impl::tls_local_dispatch_key_set();
    watchers_ = c10::DispatchKeySet({K::Python, K::Tracer, K::Functionalize,
                                     K::FuncTorchDynamicLayerFrontMode, K::FuncTorchBatched,
                                     K::FuncTorchGradWrapper}) - local.excluded_;
    everything_ = !(local.included_ & watchers_).empty();
  }
  bool sees(const Tensor& t) const {
    return everything_ || !(t.key_set() & watchers_).empty();
  }

 private:
  using K = c10::DispatchKey;
  c10::DispatchKeySet watchers_;
  bool everything_;
};

// A dual tensor's tangent would be left out, or left as it was beside a scaled value.
class Tangents {
 public:
  Tangents() : some_(torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr) {}
  void refuse(const char* what, const Tensor& t) const {
    TORCH_CHECK_NOT_IMPLEMENTED(!some_ || !t._fw_grad(0).defined(), what,
                                " has no forward-mode derivative");
  }

 private:
  bool some_;  // no tensor has one outside of a level
};

void check_input(const char* what, const Tensor& t, c10::Device device) {
  const auto type = t.scalar_type();
  TORCH_CHECK_TYPE(t.layout() == at::kStrided && t.is_cuda() &&
                       (type == at::kFloat || type == at::kBFloat16 || type == at::kHalf),
                   what, " takes dense CUDA float32, bfloat16 or float16 tensors; got ", type,
                   " (", t.layout(), ") on ", t.device());
  TORCH_CHECK_VALUE(t.device() == device, what, ": tensors are on ", device, " and ", t.device());
}

// Whether the tensor's elements fill its memory, in whatever order of dimensions.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense() && !t.is_neg(); }

struct Lists {
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int64_t> counts;
  std::vector<int32_t> dtypes;
  std::vector<Tensor> kept;  // copies that the call reads

  explicit Lists(size_t size) {
    in.reserve(size);
    out.reserve(size);
    counts.reserve(size);
    dtypes.reserve(size);
  }
  void add(const Tensor& t) {
    const auto type = t.scalar_type();
    in.push_back(t.numel() ? t.const_data_ptr() : nullptr);
    counts.push_back(t.numel());
    dtypes.push_back(type == at::kFloat ? ICTC_DTYPE_F32
                     : type == at::kBFloat16 ? ICTC_DTYPE_BF16 : ICTC_DTYPE_F16);
  }
  void add_copy(const Tensor& t) {
    kept.push_back(t.resolve_neg().contiguous());
    add(kept.back());
  }
  int64_t size() const { return static_cast<int64_t>(in.size()); }
};

// The norm, and workspace that goes back to the current stream's pool with this.
struct Space {
  Tensor norm;
  c10::DataPtr workspace;
  size_t bytes = 0;

  Space(int64_t tensors, c10::Device device) {
    check(api.workspace(tensors, device.index(), &bytes), "grad_norm_workspace");
    norm = at::empty({}, at::TensorOptions().device(device).dtype(at::kFloat));
    workspace = c10::GetAllocator(c10::kCUDA)->allocate(bytes);
  }
};

std::optional<c10::Device> cuda_or_none(c10::Device device) {
  return device.is_cuda() ? std::optional<c10::Device>(device) : std::nullopt;
}

void* stream_of(c10::Device device) {
  return c10::cuda::getCurrentCUDAStream(device.index()).stream();
}

// None where the dispatcher has to see the call.
py::object grad_norm(py::handle given, bool largest) {
  const Sequence tensors("grad_norm", given);
  TORCH_CHECK_VALUE(tensors.size() > 0, "grad_norm: no tensors");
  const Watch watch;
  if (watch.sees(tensors[0])) return py::none();  // before its device is made current
  const auto device = tensors[0].device();
  const at::NoGradGuard no_grad;
  const c10::cuda::OptionalCUDAGuard guard(cuda_or_none(device));
  const Tangents tangents;
  Lists lists(tensors.size());
  for (size_t i = 0; i < tensors.size(); ++i) {
    const Tensor& t = tensors[i];
    if (watch.sees(t)) return py::none();
    check_input("grad_norm", t, device);
    tangents.refuse("grad_norm", t);
    if (dense(t)) lists.add(t);
    else lists.add_copy(t);
  }
  const Space s(lists.size(), device);
  check(api.norm(lists.in.data(), lists.counts.data(), lists.dtypes.data(), lists.size(),
                 largest ? ICTC_GRAD_NORM_MAX : ICTC_GRAD_NORM_2, s.norm.data_ptr<float>(),
                 s.workspace.get(), s.bytes, stream_of(device)),
        "grad_norm");
  return py::cast(s.norm);
}

struct Range {
  uintptr_t begin, end;
};

// From the first to the last element.
Range extent(const Tensor& t) {
  const auto begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {begin, begin + static_cast<uintptr_t>((last + 1) * static_cast<int64_t>(t.element_size()))};
}

// Stride and size of the dimensions, the smallest stride first; expanded ones left out.
std::vector<std::pair<int64_t, int64_t>> by_stride(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) != 0) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  return dims;
}

// Whether every stride steps over all that smaller ones reach, as in slices of a dense tensor;
// then no two elements are one.
bool is_nested(const Tensor& t) {
  int64_t reach = 0;
  for (const auto& [stride, size] : by_stride(t)) {
    if (stride <= reach) return false;
    reach += stride * (size - 1);
  }
  return true;
}

// Every run of elements that follow one another in memory.
void add_runs(const Tensor& t, std::vector<Range>& runs) {
  const auto dims = by_stride(t);
  int64_t run = 1;
  size_t outer = 0;
  for (; outer < dims.size() && dims[outer].first == run; ++outer) run *= dims[outer].second;
  const auto size = static_cast<int64_t>(t.element_size());
  const auto start = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  std::vector<int64_t> at(dims.size(), 0);
  int64_t offset = 0;
  for (;;) {
    const uintptr_t begin = start + static_cast<uintptr_t>(offset * size);
    runs.push_back({begin, begin + static_cast<uintptr_t>(run * size)});
    size_t d = outer;
    for (; d < dims.size(); ++d) {
      offset += dims[d].first;
      if (++at[d] < dims[d].second) break;
      offset -= dims[d].first * dims[d].second;
      at[d] = 0;
    }
    if (d == dims.size()) return;
  }
}

// Whether no output shares memory with another or with a gradient.  (A gradient may share
// memory with another gradient.)  Outputs and gradients come apart, each in the order of their
// memory as a rule.
bool are_apart(std::vector<Range>& outs, std::vector<Range>& grads) {
  const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  for (auto* r : {&outs, &grads})
    if (!std::is_sorted(r->begin(), r->end(), before)) std::sort(r->begin(), r->end(), before);
  uintptr_t out_end = 0, any_end = 0;
  for (auto o = outs.begin(), g = grads.begin(); o != outs.end() || g != grads.end();) {
    const bool is_out = g == grads.end() || (o != outs.end() && o->begin <= g->begin);
    const Range r = is_out ? *o++ : *g++;
    if (r.begin < (is_out ? any_end : out_end)) return false;
    if (is_out) out_end = std::max(out_end, r.end);
    any_end = std::max(any_end, r.end);
  }
  return true;
}

// Refuses outputs that share memory with one another or with another gradient: their elements
// would be scaled twice, be read by some CTAs after others wrote them, or be overwritten by a
// later copy.  `copied`: the entries whose gradient the kernels read a copy of, whose memory may
// have gaps; that of the others is the list's.
void check_apart(const Lists& lists, const Sequence& given, const Sequence& to,
                 const std::vector<size_t>& copied) {
  std::vector<Range> outs, grads;
  outs.reserve(lists.in.size());
  grads.reserve(lists.in.size());
  auto next = copied.begin();
  bool nested = true;
  const auto same_view = [](const Tensor& a, const Tensor& b) {
    if (a.is_same(b)) return true;
    bool same = a.const_data_ptr() == b.const_data_ptr();
    for (int64_t d = 0; same && d < a.dim(); ++d) same = a.size(d) == 1 || a.stride(d) == b.stride(d);
    return same;
  };
  for (size_t i = 0; i < lists.in.size(); ++i) {
    const uintptr_t bytes = static_cast<uintptr_t>(lists.counts[i]) *
                            (lists.dtypes[i] == ICTC_DTYPE_F32 ? 4 : 2);
    const bool apart = next != copied.end() && *next == i;
    if (apart) ++next;
    if (!bytes) continue;
    if (apart) {
      outs.push_back(extent(to[i]));
      nested = nested && is_nested(to[i]);
      if (!same_view(given[i], to[i])) grads.push_back(extent(given[i]));
      continue;
    }
    const auto out = reinterpret_cast<uintptr_t>(lists.out[i]);
    const auto in = reinterpret_cast<uintptr_t>(lists.in[i]);
    outs.push_back({out, out + bytes});
    if (in != out) grads.push_back({in, in + bytes});
  }
  bool fine = are_apart(outs, grads) && nested;
  if (!fine && !copied.empty()) {  // extents cross; slices of one tensor may do so without sharing
    std::vector<Range> runs[2];
    for (size_t i = 0; i < lists.in.size(); ++i) {
      if (!lists.counts[i]) continue;
      add_runs(to[i], runs[0]);
      if (!same_view(given[i], to[i])) add_runs(given[i], runs[1]);
    }
    fine = are_apart(runs[0], runs[1]);
  }
  TORCH_CHECK_VALUE(fine, "clip_grads: gradients or outputs share memory; list each tensor once");
}

Tensor launch(const Lists& lists, c10::Device device, double max_norm, bool largest) {
  const Space s(lists.size(), device);
  check(api.clip(lists.in.data(), lists.out.data(), lists.counts.data(), lists.dtypes.data(),
                 lists.size(), largest ? ICTC_GRAD_NORM_MAX : ICTC_GRAD_NORM_2, max_norm,
                 s.norm.data_ptr<float>(), s.workspace.get(), s.bytes, stream_of(device)),
        "clip_grads");
  return s.norm;
}

// Into the tensors of `out`; nothing where the dispatcher has to see the call.
std::optional<Tensor> clip_into(const Sequence& grads, const Sequence& out, double max_norm,
                                bool largest) {
  TORCH_CHECK_VALUE(out.size() == grads.size(), "clip_grads: ", grads.size(), " gradients and ",
                    out.size(), " outputs");
  const auto device = grads[0].device();
  const Watch watch;
  const Tangents tangents;
  Lists lists(grads.size());
  std::vector<std::pair<size_t, Tensor>> apart;  // results that the kernels leave elsewhere
  std::vector<size_t> copied;                    // gradients that they read a copy of
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = out[i];
    if (watch.sees(g) || watch.sees(o)) return std::nullopt;
    check_input("clip_grads", g, device);
    tangents.refuse("clip_grads", g);
    const bool one = g.is_same(o);
    if (!one) {
      tangents.refuse("clip_grads", o);
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && o.scalar_type() == g.scalar_type() &&
                            o.device() == g.device() && o.layout() == at::kStrided,
                        "clip_grads: output ", i, " must have its gradient's shape, type and "
                        "device");
    }
    if (dense(g) && (one || (dense(o) && g.strides() == o.strides()))) {
      lists.add(g);
      lists.out.push_back(g.numel() ? o.data_ptr() : nullptr);
      continue;
    }
    TORCH_CHECK_VALUE(at::has_internal_overlap(o) != at::MemOverlap::Yes, "clip_grads: output ", i,
                      " has elements that share memory");
    lists.add_copy(g);
    copied.push_back(i);
    if (!dense(o) || !o.is_contiguous())
      apart.emplace_back(i, at::empty(g.sizes(), g.options()));
    const Tensor& to = !apart.empty() && apart.back().first == i ? apart.back().second : o;
    lists.out.push_back(g.numel() ? to.data_ptr() : nullptr);
  }
  check_apart(lists, grads, out, copied);
  const Tensor norm = launch(lists, device, max_norm, largest);
  size_t next = 0;
  for (size_t i = 0; i < out.size(); ++i) {
    if (next < apart.size() && apart[next].first == i) out[i].copy_(apart[next++].second);
    else if (!out[i].is_inference()) out[i].unsafeGetTensorImpl()->bump_version();
  }
  return norm;
}

// New outputs are parts of one allocation, each at a multiple of 64 bytes: an allocation for
// each took 1.3 us a tensor, most of a call.
constexpr int64_t kApart = 64;

int64_t bytes_of(const Tensor& t) {
  return (t.numel() * static_cast<int64_t>(t.element_size()) + kApart - 1) / kApart * kApart;
}

c10::Storage one_buffer(const Sequence& like) {
  int64_t bytes = 0;
  for (size_t i = 0; i < like.size(); ++i) bytes += bytes_of(like[i]);
  return at::empty({bytes}, at::TensorOptions().device(like[0].device()).dtype(at::kByte)).storage();
}

// A tensor like `t` (its order of dimensions where that is dense) at byte `at`, which moves on.
Tensor part_of(const c10::Storage& memory, int64_t& at, const Tensor& t) {
  Tensor part = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(memory), c10::DispatchKeySet(c10::DispatchKey::CUDA), t.dtype());
  auto* impl = part.unsafeGetTensorImpl();
  impl->set_storage_offset(at / static_cast<int64_t>(t.element_size()));
  if (dense(t)) impl->set_sizes_and_strides(t.sizes(), t.strides());
  else impl->set_sizes_contiguous(t.sizes());
  at += bytes_of(t);
  return part;
}

// (outputs, norm); None where the dispatcher has to see the call.
py::object clip_grads(py::handle given, double max_norm, bool largest, py::handle out) {
  const Sequence grads("clip_grads", given);
  TORCH_CHECK_VALUE(max_norm >= 0, "clip_grads: max_norm must be >= 0, got ", max_norm);
  TORCH_CHECK_VALUE(grads.size() > 0, "clip_grads: no tensors");
  const Watch watch;
  if (watch.sees(grads[0])) return py::none();  // before its device is made current
  const auto device = grads[0].device();
  const at::NoGradGuard no_grad;
  const c10::cuda::OptionalCUDAGuard guard(cuda_or_none(device));
  if (!out.is_none()) {
    const Sequence to("clip_grads", out);
    const auto norm = clip_into(grads, to, max_norm, largest);
    return norm ? py::object(py::make_tuple(py::list(to.items()), *norm)) : py::none();
  }
  const Tangents tangents;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (watch.sees(grads[i])) return py::none();
    check_input("clip_grads", grads[i], device);
    tangents.refuse("clip_grads", grads[i]);
  }
  Lists lists(grads.size());
  py::list made(grads.size());
  const auto memory = one_buffer(grads);
  int64_t at = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& g = grads[i];
    const Tensor o = part_of(memory, at, g);
    made[i] = py::cast(o);
    if (dense(g)) lists.add(g);
    else lists.add_copy(g);
    lists.out.push_back(o.numel() ? o.data_ptr() : nullptr);
  }
  const Tensor norm = launch(lists, device, max_norm, largest);
  return py::make_tuple(made, norm);
}

// Entry points of the loaded kernel library, by address.
void bind(uintptr_t last_error, uintptr_t workspace, uintptr_t norm, uintptr_t clip_entry) {
  const auto set = [](auto& fn, uintptr_t at) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at); };
  set(api.last_error, last_error);
  set(api.workspace, workspace);
  set(api.norm, norm);
  set(api.clip, clip_entry);
}

}  // namespace

PYBIND11_MODULE(_gradient_lists, m) {
  m.def("bind", &bind);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
