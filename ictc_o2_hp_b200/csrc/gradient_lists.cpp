// Lists of tensors to the C ABI's gradient norm and clipping: argument checks, copies of what
// the kernels cannot address, allocation.  In C++ because a call takes hundreds of tensors,
// whose addresses and sizes Python would read one attribute at a time.
#include <ATen/MemoryOverlap.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "ictc_o2_b200.h"

namespace {

using at::Tensor;
using Tensors = std::vector<Tensor>;

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

// Whether a call on these tensors has to be seen by the dispatcher (a trace, fake tensors).
bool watched(const Tensors& tensors) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet kWatchers(
      {K::Python, K::Tracer, K::Functionalize, K::FuncTorchDynamicLayerFrontMode,
       K::FuncTorchBatched, K::FuncTorchGradWrapper});
  const auto local = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = local.included_;
  for (const Tensor& t : tensors) keys = keys | t.key_set();
  return !((keys - local.excluded_) & kWatchers).empty();
}

void check_inputs(const char* what, const Tensors& tensors) {
  for (const Tensor& t : tensors) {
    const auto type = t.scalar_type();
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && t.is_cuda() &&
                         (type == at::kFloat || type == at::kBFloat16 || type == at::kHalf),
                     what, " takes dense CUDA float32, bfloat16 or float16 tensors; got ", type,
                     " (", t.layout(), ") on ", t.device());
    TORCH_CHECK_VALUE(t.device() == tensors[0].device(), what, ": tensors are on ",
                      tensors[0].device(), " and ", t.device());
  }
}

// Whether the tensor's elements fill its memory, in whatever order of dimensions.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense() && !t.is_neg(); }

struct Lists {
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int64_t> counts;
  std::vector<int32_t> dtypes;
  Tensors kept;  // copies that the call reads

  void add(const Tensor& t) {
    const auto type = t.scalar_type();
    in.push_back(t.numel() ? t.data_ptr() : nullptr);
    counts.push_back(t.numel());
    dtypes.push_back(type == at::kFloat ? ICTC_DTYPE_F32
                     : type == at::kBFloat16 ? ICTC_DTYPE_BF16 : ICTC_DTYPE_F16);
  }
};

Tensor plain_copy(const Tensor& t) { return t.resolve_neg().contiguous(); }

struct Space {
  Tensor norm, workspace;
  size_t bytes = 0;
};

Space space_for(const Tensors& tensors) {
  Space s;
  const auto options = at::TensorOptions().device(tensors[0].device());
  check(api.workspace(static_cast<int64_t>(tensors.size()), tensors[0].device().index(), &s.bytes),
        "grad_norm_workspace");
  s.norm = at::empty({}, options.dtype(at::kFloat));
  s.workspace = at::empty({static_cast<int64_t>(s.bytes)}, options.dtype(at::kByte));
  return s;
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

Tensor grad_norm(const Tensors& tensors, bool largest) {
  check_inputs("grad_norm", tensors);
  TORCH_CHECK_VALUE(!tensors.empty(), "grad_norm: no tensors");
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(tensors[0].device());
  Lists lists;
  for (const Tensor& t : tensors) {
    lists.kept.push_back(dense(t) ? t : plain_copy(t));
    lists.add(lists.kept.back());
  }
  const Space s = space_for(tensors);
  check(api.norm(lists.in.data(), lists.counts.data(), lists.dtypes.data(),
                 static_cast<int64_t>(lists.in.size()),
                 largest ? ICTC_GRAD_NORM_MAX : ICTC_GRAD_NORM_2, s.norm.data_ptr<float>(),
                 s.workspace.data_ptr(), s.bytes, stream_of(tensors[0])),
        "grad_norm");
  return s.norm;
}

// Refuses outputs that share memory with one another or with another gradient: their
// elements would be scaled twice, or be read by some CTAs after others wrote them.
void check_apart(const Lists& lists) {
  struct Range {
    uintptr_t begin, end;
  };
  std::vector<Range> ranges;
  ranges.reserve(2 * lists.in.size());
  for (size_t i = 0; i < lists.in.size(); ++i) {
    const uintptr_t bytes = static_cast<uintptr_t>(lists.counts[i]) *
                            (lists.dtypes[i] == ICTC_DTYPE_F32 ? 4 : 2);
    if (!bytes) continue;
    const auto out = reinterpret_cast<uintptr_t>(lists.out[i]);
    const auto in = reinterpret_cast<uintptr_t>(lists.in[i]);
    ranges.push_back({out, out + bytes});
    if (in != out) ranges.push_back({in, in + bytes});
  }
  const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(ranges.begin(), ranges.end(), before))
    std::sort(ranges.begin(), ranges.end(), before);
  for (size_t i = 1; i < ranges.size(); ++i)
    TORCH_CHECK_VALUE(ranges[i - 1].end <= ranges[i].begin,
                      "clip_grads: gradients or outputs share memory; list each tensor once");
}

// out = grads scaled to at most max_norm; `fresh`: the outputs were made for this call.
Tensor clip(const Tensors& grads, const Tensors& out, double max_norm, bool largest, bool fresh) {
  check_inputs("clip_grads", grads);
  TORCH_CHECK_VALUE(!grads.empty(), "clip_grads: no tensors");
  TORCH_CHECK_VALUE(max_norm >= 0, "clip_grads: max_norm must be >= 0, got ", max_norm);
  TORCH_CHECK_VALUE(out.size() == grads.size(), "clip_grads: ", grads.size(), " gradients and ",
                    out.size(), " outputs");
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(grads[0].device());
  for (size_t i = 0; !fresh && i < out.size(); ++i) {
    TORCH_CHECK_VALUE(out[i].sizes() == grads[i].sizes() &&
                          out[i].scalar_type() == grads[i].scalar_type() &&
                          out[i].device() == grads[i].device() && out[i].layout() == at::kStrided,
                      "clip_grads: output ", i, " must have its gradient's shape, type and "
                      "device");
    TORCH_CHECK_VALUE(at::has_internal_overlap(out[i]) != at::MemOverlap::Yes,
                      "clip_grads: output ", i, " has elements that share memory");
  }
  Lists lists;
  Tensors targets;  // what the kernels write, where it is not the output itself
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = out[i];
    const bool same = dense(g) && dense(o) && g.strides() == o.strides();
    const bool plain = !same && dense(o) && o.is_contiguous();
    lists.kept.push_back(same ? g : plain_copy(g));
    lists.add(lists.kept.back());
    targets.push_back(same || plain ? o : at::empty(g.sizes(), g.options()));
    lists.out.push_back(g.numel() ? targets.back().data_ptr() : nullptr);
  }
  if (!fresh) check_apart(lists);
  const Space s = space_for(grads);
  check(api.clip(lists.in.data(), lists.out.data(), lists.counts.data(), lists.dtypes.data(),
                 static_cast<int64_t>(lists.in.size()),
                 largest ? ICTC_GRAD_NORM_MAX : ICTC_GRAD_NORM_2, max_norm,
                 s.norm.data_ptr<float>(), s.workspace.data_ptr(), s.bytes, stream_of(grads[0])),
        "clip_grads");
  for (size_t i = 0; !fresh && i < out.size(); ++i) {
    if (!targets[i].is_same(out[i])) out[i].copy_(targets[i]);
    else if (!out[i].is_inference()) out[i].unsafeGetTensorImpl()->bump_version();
  }
  return s.norm;
}

std::tuple<Tensors, Tensor> clip_grads(const Tensors& grads, double max_norm, bool largest,
                                       const std::optional<Tensors>& out) {
  if (out.has_value()) return {*out, clip(grads, *out, max_norm, largest, false)};
  check_inputs("clip_grads", grads);
  const at::NoGradGuard no_grad;
  Tensors made;
  made.reserve(grads.size());
  for (const Tensor& g : grads) made.push_back(at::empty_like(g));
  const Tensor norm = clip(grads, made, max_norm, largest, true);
  return {made, norm};
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
  m.def("watched", &watched);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
