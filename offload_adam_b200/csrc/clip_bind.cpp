// Python bindings of the global gradient norm and clipping.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <tuple>

#include "clip_ops.h"

namespace py = pybind11;
using at::Tensor;

namespace {

void ok(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

// The gradients as ranges of memory; a tensor that does not fill a range of its own is copied,
// and written back by the caller, so whatever such tensors share is scaled once.  A gradient that
// stands in the list twice, whatever tensor it is a view by, counts once.
struct Gradients {
  std::vector<oab::ClipEntry> entries;
  std::vector<Tensor> copies;                       // keeps them alive
  std::vector<std::pair<Tensor, Tensor>> scattered;  // gradient, its copy

  static bool same(const oab::ClipEntry& a, const oab::ClipEntry& b) { return a.p == b.p && a.n == b.n && a.dtype == b.dtype; }
  static bool before(const oab::ClipEntry* a, const oab::ClipEntry* b) {
    return std::tie(a->p, a->n, a->dtype) < std::tie(b->p, b->n, b->dtype);
  }

  Gradients(const std::vector<Tensor>& grads, bool write) {
    entries.reserve(grads.size());
    for (const Tensor& g : grads) {
      TORCH_CHECK(g.is_cuda() && g.device() == grads[0].device(), "gradients must be on one CUDA device");
      const auto t = g.scalar_type();
      TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "gradients must be bf16, fp16 or fp32");
      if (g.numel() == 0) continue;
      const uint32_t dtype = t == at::kBFloat16 ? oab::kClipBF16 : t == at::kHalf ? oab::kClipF16 : oab::kClipF32;
      Tensor x = g;
      if (!g.is_non_overlapping_and_dense()) {
        bool seen = false;
        for (const auto& [a, b] : scattered)
          seen = seen || (a.data_ptr() == g.data_ptr() && a.scalar_type() == t && a.sizes() == g.sizes() && a.strides() == g.strides());
        if (seen) continue;
        if (write) {
          const auto z = g.strides();
          for (int64_t i = 0; i < g.dim(); ++i)
            TORCH_CHECK_VALUE(z[i] != 0 || g.size(i) <= 1, "a gradient whose elements share memory cannot be clipped in place");
        }
        x = g.clone(at::MemoryFormat::Contiguous);
        scattered.emplace_back(g, x);
        copies.push_back(x);
      }
      entries.push_back({x.data_ptr(), x.numel(), dtype, 0});
    }
    std::vector<const oab::ClipEntry*> order;
    order.reserve(entries.size());
    bool sorted = true;
    for (const auto& e : entries) {
      sorted = sorted && (order.empty() || before(order.back(), &e));
      order.push_back(&e);
    }
    if (!sorted) std::sort(order.begin(), order.end(), before);
    bool twice = false;
    for (size_t i = 1; i < order.size(); ++i) {
      const auto &a = *order[i - 1], &b = *order[i];
      if (same(a, b)) twice = true;
      else  // a norm may read both; scaled in place, what they share would be multiplied twice
        TORCH_CHECK_VALUE(!write || static_cast<char*>(a.p) + a.n * (a.dtype == oab::kClipF32 ? 4 : 2) <= b.p,
                          "two gradients share a part of their memory");
    }
    if (twice) {
      std::vector<oab::ClipEntry> once;
      for (size_t i = 0; i < order.size(); ++i)
        if (i == 0 || !same(*order[i], *order[i - 1])) once.push_back(*order[i]);
      entries.swap(once);
    }
  }
};

void written(const std::vector<Tensor>& grads, const Gradients& g) {
  for (const auto& [to, from] : g.scattered) to.copy_(from);
  for (const Tensor& t : grads)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// {coefficient, norm} as one fp32 tensor; with `scale`, the gradients are multiplied by the first.
Tensor grad_norm(const std::vector<Tensor>& grads, int64_t norm, double max_norm, bool scale) {
  TORCH_CHECK(!grads.empty(), "grad_norm: no gradient");
  c10::cuda::CUDAGuard guard(grads[0].device());
  Gradients g(grads, scale);
  const auto opts = grads[0].options().dtype(at::kFloat).layout(at::kStrided);
  if (g.entries.empty()) {
    Tensor out = at::zeros({2}, opts);
    out[0].fill_(1.0);
    return out;
  }
  Tensor out = at::empty({2}, opts);
  const int64_t count = (int64_t)g.entries.size();
  const Tensor partials = at::empty({oab::clip_partials(count)}, opts.dtype(at::kDouble));
  ok(oab::launch_grad_norm(g.entries.data(), count, (int)norm, (float)max_norm, scale, partials.data_ptr<double>(),
                           out.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()), "grad_norm");
  if (scale) written(grads, g);
  return out;
}

// The same for the gradients of `params`, the norm alone unless `both`; None (and nothing done) when
// one of them is not a plain gradient of one CUDA device that the kernels take, or when there is none.
py::object param_grad_norm(const py::list& params, int64_t norm, double max_norm, bool scale, bool both) {
  at::NoGradGuard no_grad;
  std::vector<Tensor> grads;
  grads.reserve(params.size());
  for (const py::handle& h : params) {
    TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), "parameters must be tensors");
    const Tensor& g = THPVariable_Unpack(h.ptr()).grad();
    if (!g.defined()) continue;
    const auto t = g.scalar_type();
    if (!g.is_cuda() || g.layout() != at::kStrided || g.key_set().has(c10::DispatchKey::Python) ||
        (t != at::kBFloat16 && t != at::kHalf && t != at::kFloat) || (!grads.empty() && g.get_device() != grads[0].get_device()))
      return py::none();
    grads.push_back(g);
  }
  if (grads.empty()) return py::none();
  const Tensor out = grad_norm(grads, norm, max_norm, scale);
  return py::cast(both ? out : out.select(0, 1));
}

// The gradients times `coef`, one fp32 value on their device.
void grad_scale(const std::vector<Tensor>& grads, const Tensor& coef) {
  if (grads.empty()) return;
  TORCH_CHECK(coef.device() == grads[0].device() && coef.scalar_type() == at::kFloat && coef.numel() >= 1, "grad_scale: fp32 coefficient");
  c10::cuda::CUDAGuard guard(grads[0].device());
  Gradients g(grads, true);
  ok(oab::launch_grad_scale(g.entries.data(), (int64_t)g.entries.size(), coef.data_ptr<float>(),
                            at::cuda::getCurrentCUDAStream().stream()), "grad_scale");
  written(grads, g);
}

}  // namespace

void bind_clip(py::module_& m) {
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("norm"), py::arg("max_norm"), py::arg("scale"));
  m.def("param_grad_norm", &param_grad_norm, py::arg("params"), py::arg("norm"), py::arg("max_norm"), py::arg("scale"),
        py::arg("both") = true);
  m.def("grad_scale", &grad_scale, py::arg("grads"), py::arg("coef"));
}
