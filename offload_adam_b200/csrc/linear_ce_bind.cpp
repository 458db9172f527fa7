// Autograd function of the cross entropy that keeps no logits, and its Python binding.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>

#include "linear_ce.h"
#include "loss_ops.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream().stream(); }
void ok(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

// Rows that the kernels can read in place: 16-byte aligned, none overlapping.
Tensor rows_layout(const Tensor& t) {
  const bool fits = t.stride(1) == 1 && (t.size(0) == 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&
                    (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t row_stride(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

// What backward needs of forward, in one tensor of bytes: the packed rows of h (backward needs them in
// any case, so keeping them instead of h leaves its peak), then index, label, top, rest and miss of each,
// their number with the ticket, 1 / number, and whether a wait was given up.
int64_t packed_bytes(int64_t rows, int64_t hidden) { return 2 * oab::lce_padded(rows) * oab::lce_row_pitch(hidden); }
int64_t kept_bytes(int64_t rows, int64_t hidden) { return packed_bytes(rows, hidden) + 4 * (5 * rows + 4); }
oab::LceArgs make_args(const Tensor& w, const Tensor& labels, void* kept, int64_t ignore) {
  oab::LceArgs a;
  a.w = w.data_ptr();
  a.w_stride = row_stride(w);
  a.labels = labels.data_ptr<int64_t>();
  a.rows = labels.size(0);
  a.hidden = w.size(1);
  a.vocab = w.size(0);
  a.ignore = ignore;
  a.packed = kept;
  int* k = reinterpret_cast<int*>(static_cast<char*>(kept) + packed_bytes(a.rows, a.hidden));
  a.index = k;
  a.label = k + a.rows;
  a.top = reinterpret_cast<float*>(k + 2 * a.rows);
  a.rest = reinterpret_cast<float*>(k + 3 * a.rows);
  a.miss = reinterpret_cast<float*>(k + 4 * a.rows);
  a.count = k + 5 * a.rows;
  a.inv = reinterpret_cast<float*>(k + 5 * a.rows + 2);
  a.lost = k + 5 * a.rows + 3;
  a.report = oab::loss_report();
  return a;
}
// Fresh memory for the values of one call, cut into parts that start on 256 bytes.
struct Scratch {
  int64_t bytes = 0;
  Tensor memory;
  int64_t add(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
  void take(const Tensor& like) { memory = at::empty({bytes}, like.options().dtype(at::kByte)); }
  template <class T>
  T* at_byte(int64_t at) const { return reinterpret_cast<T*>(static_cast<char*>(memory.data_ptr()) + at); }
};

// The loss, and what backward needs of it if `keep`.
Tensor run_forward(const Tensor& h, const Tensor& w, const Tensor& labels, int64_t reduction, int64_t ignore, Tensor* keep) {
  c10::cuda::CUDAGuard guard(h.device());
  oab::raise_loss_report();
  const Tensor hc = rows_layout(h), wc = rows_layout(w);
  const int64_t rows = h.size(0);
  const auto f32 = h.options().dtype(at::kFloat);
  Tensor loss = reduction == oab::kLceNone ? at::empty({rows}, f32) : at::empty({}, f32);
  Scratch x;
  const int64_t kept = x.add(keep != nullptr ? 0 : kept_bytes(rows, h.size(1)));
  const int64_t part = x.add(4 * oab::lce_part_floats(rows, w.size(0))), picked = x.add(4 * rows), sums = x.add(8 * oab::lce_sum_doubles(rows));
  x.take(h);
  if (keep != nullptr) *keep = at::empty({kept_bytes(rows, h.size(1))}, h.options().dtype(at::kByte));
  auto a = make_args(wc, labels, keep != nullptr ? keep->data_ptr() : x.at_byte<void>(kept), ignore);
  a.h = hc.data_ptr();
  a.h_stride = row_stride(hc);
  ok(oab::launch_lce_forward(a, (int)reduction, x.at_byte<float>(part), x.at_byte<float>(picked), x.at_byte<double>(sums),
                             loss.data_ptr<float>(), cur()),
     "linear_cross_entropy");
  return loss;
}

struct LinearCE : torch::autograd::Function<LinearCE> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& labels, int64_t reduction,
                        int64_t ignore, int64_t piece) {
    Tensor kept;
    Tensor loss = run_forward(h, w, labels, reduction, ignore, &kept);
    ctx->save_for_backward({w, labels, kept});
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["piece"] = piece;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& g = grads[0];
    const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    if (!g.defined() || !(want_h || want_w)) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    // the gradients can be had with create_graph, but not differentiated again
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    const Tensor &w = saved[0], &labels = saved[1];
    const int64_t reduction = ctx->saved_data["reduction"].toInt(), ignore = ctx->saved_data["ignore"].toInt();
    c10::cuda::CUDAGuard guard(w.device());
    oab::raise_loss_report();
    // hooks on saved tensors may have returned copies of another layout
    const bool whole = saved[2].is_contiguous() && (reinterpret_cast<uintptr_t>(saved[2].data_ptr()) & 15u) == 0;
    const Tensor kept = whole ? saved[2] : saved[2].clone(at::MemoryFormat::Contiguous), wc = rows_layout(w), lc = labels.contiguous();
    const Tensor gc = g.to(at::kFloat).contiguous();
    const int64_t rows = labels.size(0), hidden = w.size(1), vocab = w.size(0);
    int64_t piece = ctx->saved_data["piece"].toInt();
    piece = std::min({piece, vocab, oab::kLceMaxPiece});
    piece = piece > 0 ? (piece + oab::kLceTile - 1) / oab::kLceTile * oab::kLceTile : oab::lce_default_piece(rows, vocab);
    oab::LceGrad x;
    x.reduction = (int)reduction;
    x.g = gc.data_ptr<float>();
    x.piece = piece;
    x.splits = want_h ? oab::lce_splits(rows, hidden, vocab, piece) : 1;
    Tensor gh, gw;
    Scratch t;
    const int64_t d = t.add(2 * oab::lce_padded(rows) * oab::lce_piece_pitch(vocab, piece));
    const int64_t acc = t.add(want_h && !oab::lce_direct(vocab, piece, x.splits) ? 4 * x.splits * oab::lce_padded(rows) * oab::lce_row_pitch(hidden) : 0);
    const int64_t scaled = t.add(want_w ? packed_bytes(rows, hidden) : 0);
    const int64_t wacc = t.add(want_w && oab::lce_row_groups(rows) > 1 ? 4 * std::min(piece, vocab) * oab::lce_row_pitch(hidden) : 0);
    t.take(w);
    x.d = t.at_byte<void>(d);
    if (want_h) {
      gh = at::empty({rows, hidden}, w.options());
      x.gh = gh.data_ptr();
      x.acc = t.at_byte<float>(acc);
    }
    if (want_w) {
      gw = at::empty({vocab, hidden}, w.options());
      x.gw = gw.data_ptr();
      x.scaled = t.at_byte<void>(scaled);
      x.wacc = t.at_byte<float>(wacc);
    }
    ok(oab::launch_lce_backward(make_args(wc, lc, kept.data_ptr(), ignore), x, cur()), "linear_cross_entropy backward");
    if (graph) {
      const auto last = std::make_shared<torch::autograd::DelayedError>("linear_cross_entropy has no second derivative", 2);
      for (Tensor* t : {&gh, &gw})
        if (t->defined()) t->set_requires_grad(true);
      at::AutoGradMode with_grad(true);
      auto out = (*last)({gh, gw});
      gh = out[0];
      gw = out[1];
    }
    return {gh, gw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// Whether the kernels take these; the rest is the caller's, its refusals too.
bool takes(const Tensor& h, const Tensor& w, const Tensor& labels) {
  for (const Tensor* t : {&h, &w, &labels})
    if (!t->defined() || !t->is_cuda() || t->layout() != at::kStrided || t->key_set().has(c10::DispatchKey::Python)) return false;
  if (h.scalar_type() != at::kBFloat16 || w.scalar_type() != at::kBFloat16 || labels.scalar_type() != at::kLong || h.dim() < 1 || w.dim() != 2 ||
      h.size(-1) != w.size(1) || labels.sizes() != h.sizes().slice(0, h.dim() - 1) || h.device() != w.device() || h.device() != labels.device())
    return false;
  const int64_t rows = labels.numel(), hidden = w.size(1), vocab = w.size(0);
  return rows > 0 && rows <= oab::kLceMaxRows && hidden % 8 == 0 && hidden > 0 && hidden <= oab::kLceMaxHidden && vocab > 0 &&
         vocab <= oab::kLceMaxVocab;
}

// Unless `required`, None for what the kernels do not take.
py::object linear_ce(const Tensor& h, const Tensor& w, const Tensor& labels, int64_t reduction, int64_t ignore, int64_t piece, bool required) {
  TORCH_CHECK(reduction >= 0 && reduction <= 2 && piece >= 0, "linear_cross_entropy: reduction or piece");
  if (!takes(h, w, labels)) {
    TORCH_CHECK(!required, "linear_cross_entropy: the kernels take bf16 CUDA tensors of one device, rows of a multiple of 8, an int64 label each");
    return py::none();
  }
  const Tensor rows = h.dim() == 2 ? h : h.reshape({-1, h.size(-1)});
  const Tensor each = labels.dim() == 1 && labels.is_contiguous() ? labels : labels.reshape(-1).contiguous();
  const bool graph = at::GradMode::is_enabled() && (rows.requires_grad() || w.requires_grad());
  Tensor loss = graph ? LinearCE::apply(rows, w, each, reduction, ignore, piece) : run_forward(rows, w, each, reduction, ignore, nullptr);
  if (reduction == oab::kLceNone && labels.dim() != 1) loss = loss.view(labels.sizes());
  return py::cast(loss);
}

}  // namespace

void bind_linear_ce(py::module_& m) {
  m.def("linear_ce", &linear_ce, py::arg("h"), py::arg("w"), py::arg("labels"), py::arg("reduction"), py::arg("ignore"), py::arg("piece"),
        py::arg("required") = true);
  m.def("linear_ce_wait_limit", &oab::lce_wait_limit, py::arg("nanoseconds"));
}
