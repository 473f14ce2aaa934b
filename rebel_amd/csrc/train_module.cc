// rebel_amd/csrc/train_module.cc -- the training operators of the C ABI (include/rebel_hip.h) on torch tensors, with their
// gradients.  rebel_amd/training.py is the public face.
//
// Work is enqueued on torch's current stream of the tensors' device; outputs, statistics and workspaces come from torch's
// allocator on that stream, so a captured graph keeps its own and nothing is shared between two calls.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <mutex>
#include <numeric>
#include <optional>
#include <stdexcept>
#include <utility>
#include <vector>

#include "../../include/rebel_hip.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

void check(int status) {
  if (status != 0) throw std::runtime_error(rbl_last_error());
}
// A refused argument is a ValueError
template <class... Words>
void require(bool ok, const Words&... words) {
  if (!ok) throw std::invalid_argument(c10::str(words...));
}

// -1: not one of the operators' types
int element_type(at::ScalarType t) {
  return t == at::kFloat ? RBL_F32 : t == at::kHalf ? RBL_F16 : t == at::kBFloat16 ? RBL_BF16 : -1;
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// Whether a dense tensor's elements lie in memory that it has.  Its storage may have been given back (resized to nothing, as sharded
// trainers do between uses), or a subclass that wraps other tensors may have none: the address is then null, which the C entries
// take for a parameter that is not given.
bool in_memory(const Tensor& t) {
  if (t.numel() == 0) return true;
  if (!t.has_storage()) return false;
  const c10::StorageImpl& memory = *t.storage().unsafeGetStorageImpl();
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t reach = t.storage_offset() + 1;
  for (size_t i = 0; i < sizes.size(); ++i) reach += (sizes[i] - 1) * strides[i];
  return reach * (int64_t)t.element_size() <= (int64_t)memory.nbytes() && memory.data();
}

// The elements from one row of the last dimension to the next, where all rows lie at one distance; -1 where they do not, or
// where a row's elements do not lie side by side.
int64_t row_stride(const Tensor& t) {
  const auto sizes = t.sizes();
  const auto strides = t.strides();
  const int d = (int)sizes.size() - 1;
  if (t.numel() == 0) return sizes[d];
  if (sizes[d] > 1 && strides[d] != 1) return -1;
  int64_t step = -1, rows = 1;  // of the dimensions behind i that have more than one entry
  for (int i = d - 1; i >= 0; --i) {
    if (sizes[i] == 1) continue;
    if (step >= 0 && strides[i] != step * rows) return -1;
    if (step < 0) step = strides[i];
    rows *= sizes[i];
  }
  return step < 0 ? sizes[d] : step;
}

// What the kernels can read: values as they lie in memory (a view may be marked as negated), rows at one distance.
Tensor with_rows(const Tensor& t) {
  const Tensor v = t.is_neg() ? t.resolve_neg() : t;
  return row_stride(v) < 0 ? v.contiguous() : v;
}
Tensor dense(const Tensor& t) { return !t.defined() ? t : t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

Tensor workspace(const Tensor& like, int64_t bytes) {
  check(bytes < 0);
  return bytes == 0 ? Tensor() : at::empty({bytes}, like.options().dtype(at::kByte));
}
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

rbl_layer_norm_shape shape_of(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t activation) {
  rbl_layer_norm_shape s{};
  s.cols = x.size(-1);
  s.rows = s.cols ? x.numel() / s.cols : 0;
  s.x_stride = s.dy_stride = s.cols;
  s.dtype = element_type(x.scalar_type());
  s.param_dtype = w.defined() ? element_type(w.scalar_type()) : b.defined() ? element_type(b.scalar_type()) : RBL_F32;
  s.activation = (int32_t)activation;
  s.eps = (float)eps;
  return s;
}

void check_arguments(const Tensor& x, const Tensor& w, const Tensor& b) {
  require(x.defined() && x.dim() >= 1, "layer_norm: x needs at least one dimension");
  require(element_type(x.scalar_type()) >= 0, "layer_norm: x must be float32, float16 or bfloat16, not ", x.scalar_type());
  require(x.size(-1) >= 1, "layer_norm: the last dimension of x is empty");
  for (const Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    require(p->dim() == 1 && p->size(0) == x.size(-1), "layer_norm: weight and bias must have shape [", x.size(-1),
                "], the last dimension of x, not ", p->sizes());
    require(p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type(),
                "layer_norm: weight and bias must be float32 or of x's type, not ", p->scalar_type());
    require(p->device() == x.device(), "layer_norm: weight and bias must be on x's device ", x.device(), ", not ",
                p->device());
  }
  require(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
              "layer_norm: weight and bias must have one type");
  require(x.layout() == at::kStrided, "layer_norm: x must be a dense tensor");
  for (const Tensor* t : {&x, &w, &b}) {
    require(!t->defined() || t->layout() == at::kStrided, "layer_norm: weight and bias must be dense tensors");
    require(!t->defined() || in_memory(*t), "layer_norm: x, weight or bias has no memory of its own, or too little");
    require(!t->defined() || !t->_fw_grad(0).defined(), "layer_norm: forward-mode derivatives are not supported");
  }
  require(x.is_cuda(), "layer_norm: x must be on the GPU: there is no CPU path");
}

// y, and the rows' statistics if `stats` is not null
Tensor forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t activation, Tensor* stats) {
  c10::DeviceGuard guard(x.device());
  rbl_layer_norm_shape s = shape_of(x, w, b, eps, activation);
  s.x_stride = row_stride(x);
  Tensor y = at::empty(x.sizes(), x.options());
  if (stats) *stats = at::empty({s.rows, 2}, x.options().dtype(at::kFloat));
  Tensor space = workspace(x, rbl_layer_norm_workspace(&s, 0));
  check(rbl_layer_norm_forward(x.get_device(), &s, data(x), data(w), data(b), data(y), stats ? stats->data_ptr<float>() : nullptr,
                               data(space), space.defined() ? space.numel() : 0, stream_of(x)));
  return y;
}

// A leaf's gradient is added up on the stream on which its accumulator was made.  If an earlier, eager graph of the same leaf
// is still alive, a backward pass that is being captured would run into that other stream, and the process would end.
void refuse_foreign_accumulator(const Tensor& t) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto s = node->stream();
  require(s && *s == c10::hip::getCurrentHIPStream(t.get_device()).unwrap(),
              "layer_norm: a graph that was made outside this capture still holds a leaf of this call; delete its outputs before "
              "capturing (or make it on the capturing stream)");
}

// What a saved tensor came back as.  A hook of the saved tensors may return anything, and torch compares it with nothing.
Tensor unpacked(const torch::autograd::SavedVariable& saved, c10::IntArrayRef sizes, at::ScalarType type, at::Device device,
                const char* what) {
  Tensor t = saved.unpack();
  if (!t.defined()) return t;
  if (t.layout() != at::kStrided || t.sizes() != sizes || t.scalar_type() != type || t.device() != device || !in_memory(t))
    throw std::runtime_error(c10::str("layer_norm: a hook of the saved tensors has returned ", what, " as ", t.scalar_type(), " ", t.sizes(),
                                      " on ", t.device(), ", not as the dense ", type, " ", sizes, " on ", device, " that was saved"));
  return t;
}

// The backward pass of one layer_norm call.  Edges: x, weight, bias (empty where one was not given).
class LayerNormBackward : public torch::autograd::Node {
 public:
  LayerNormBackward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& stats, double eps, int64_t activation,
                    at::ScalarType param_type)
      : x_(x, false),
        stats_(stats),
        sizes_(x.sizes().vec()),
        type_(x.scalar_type()),
        device_(x.device()),
        eps_(eps),
        activation_(activation),
        param_type_(param_type) {
    if (w.defined()) w_ = torch::autograd::SavedVariable(w, false);
    // the bias comes back only where the activation's slope depends on it
    if (b.defined() && activation != RBL_ACT_NONE) b_ = torch::autograd::SavedVariable(b, false);
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("layer_norm: its gradient has no gradient of its own (create_graph)");
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(3);
    // torch's engine hands over what fits y; a call of the node itself may hand over anything
    if (!grads[0].defined()) return out;
    if (grads[0].layout() != at::kStrided || grads[0].sizes() != sizes_ || grads[0].scalar_type() != type_ ||
        grads[0].device() != device_ || !in_memory(grads[0]))
      throw std::runtime_error(c10::str("layer_norm: the gradient of the result must be a dense ", type_, " ", c10::IntArrayRef(sizes_), " on ",
                                        device_, ", not ", grads[0].scalar_type(), " ", grads[0].sizes(), " on ", grads[0].device()));
    // a hook of the saved tensors may run operations with gradients here (recomputation), so not below autograd
    const Tensor x_back = unpacked(x_, sizes_, type_, device_, "x");
    const Tensor w_back = unpacked(w_, sizes_.back(), param_type_, device_, "weight");
    const Tensor b_back = unpacked(b_, sizes_.back(), param_type_, device_, "bias");
    at::AutoDispatchBelowADInplaceOrView plain;
    c10::DeviceGuard guard(device_);
    // laid out as forward: a copy that a hook has kept need not have the strides of what it copied
    const Tensor x = with_rows(x_back), w = dense(w_back), b = dense(b_back);
    const Tensor dy = with_rows(grads[0]);
    rbl_layer_norm_shape s = shape_of(x, w, b, eps_, activation_);
    s.param_dtype = element_type(param_type_);
    s.x_stride = row_stride(x);
    s.dy_stride = row_stride(dy);
    if (task_should_compute_output(0)) out[0] = at::empty(x.sizes(), x.options());
    for (int i = 1; i < 3; ++i)
      if (task_should_compute_output(i)) out[i] = at::empty({s.cols}, x.options().dtype(param_type_));
    const Tensor space = workspace(x, rbl_layer_norm_workspace(&s, 1));
    check(rbl_layer_norm_backward(x.get_device(), &s, data(dy), data(x), data(w), data(b), stats_.data_ptr<float>(), data(out[0]),
                                  data(out[1]), data(out[2]), data(space), space.defined() ? space.numel() : 0, stream_of(x)));
    return out;
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data();
    w_.reset_data();
    b_.reset_data();
    stats_.reset();
  }
  std::string name() const override { return "LayerNormBackward"; }

 private:
  torch::autograd::SavedVariable x_, w_, b_;
  Tensor stats_;
  std::vector<int64_t> sizes_;  // of x
  at::ScalarType type_;
  at::Device device_;
  double eps_;
  int64_t activation_;
  at::ScalarType param_type_;
};

Tensor layer_norm(const Tensor& x_in, const OptTensor& weight, const OptTensor& bias, double eps, int64_t activation) {
  const Tensor w_in = weight.value_or(Tensor()), b_in = bias.value_or(Tensor());
  check_arguments(x_in, w_in, b_in);
  // what is copied for its layout is copied where its gradient does not see it: the edges lead to the arguments themselves
  std::optional<at::AutoDispatchBelowADInplaceOrView> plain(std::in_place);
  const Tensor x = with_rows(x_in), w = dense(w_in), b = dense(b_in);
  const bool grad = at::GradMode::is_enabled() && (x_in.requires_grad() || (w_in.defined() && w_in.requires_grad()) ||
                                                   (b_in.defined() && b_in.requires_grad()));
  if (!grad) return forward(x, w, b, eps, activation, nullptr);
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    for (const Tensor* t : {&x_in, &w_in, &b_in}) refuse_foreign_accumulator(*t);
  Tensor stats;
  Tensor y = forward(x, w, b, eps, activation, &stats);
  const auto param_type = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
  plain.reset();  // before the tensors are saved: their hooks may run operations with gradients
  auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(x, w, b, stats, eps, activation, param_type),
                                                 torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x_in, w_in, b_in));
  torch::autograd::set_history(y, node);
  return y;
}

// ------------------------------------------------------------------------------------------------ gradient norm
struct Gradients {
  std::vector<rbl_grad> list;
  std::vector<std::pair<Tensor, Tensor>> copies;  // tensors with gaps: (the tensor, its values side by side)
  std::vector<const Tensor*> in_place;            // the others, where they are scaled
  Tensor any;
};

// The memory of a tensor that is scaled
struct Span {
  uintptr_t begin, end;
  const Tensor* tensor;
};

// The bytes of a tensor from its first one: its elements' size and the dimensions of more than one entry, strides in bytes
struct Lattice {
  struct Dim {
    int64_t size, stride;
  };
  std::vector<Dim> dims;
  int64_t element;

  explicit Lattice(const Tensor& t) : element((int64_t)t.element_size()) {
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1) dims.push_back({t.size(i), t.stride(i) * element});
  }
  int64_t length() const {
    int64_t n = element;
    for (const Dim& d : dims) n += (d.size - 1) * d.stride;
    return n;
  }
  Lattice modulo(int64_t step) const {
    Lattice rest = *this;
    rest.dims.erase(std::remove_if(rest.dims.begin(), rest.dims.end(), [&](const Dim& d) { return d.stride % step == 0; }), rest.dims.end());
    return rest;
  }
};

// Whether two tensors share no byte, b beginning `ahead` bytes behind a (or before it): blocks and steps of one buffer can be told
// apart.  Modulo a distance S the dimensions whose stride S divides drop out.  Where neither of the rests is longer than S, a byte
// of both would lie in both rests, at the distance `ahead` modulo S or S less: two smaller questions of the same kind.  S is
// tried at the strides and their common divisors: of two blocks of a grid that differ in some dimension, the stride of the next
// outer one that either has kept separates them.  `tries` bounds the search; false: not shown.
bool apart(const Lattice& a, const Lattice& b, int64_t ahead, int& tries) {
  if (ahead >= a.length() || ahead + b.length() <= 0) return true;
  std::vector<int64_t> steps;
  for (const Lattice* l : {&a, &b})
    for (const auto& d : l->dims) steps.push_back(d.stride);
  for (size_t i = 0, own = steps.size(); i < own; ++i)
    for (size_t j = 0; j < i; ++j) steps.push_back(std::gcd(steps[i], steps[j]));
  std::sort(steps.begin(), steps.end(), std::greater<>());
  steps.erase(std::unique(steps.begin(), steps.end()), steps.end());
  for (const int64_t step : steps) {
    if (--tries < 0) return false;
    const Lattice p = a.modulo(step), q = b.modulo(step);
    if (p.length() > step || q.length() > step) continue;
    const int64_t d = (ahead % step + step) % step;
    if (apart(p, q, d, tries) && apart(p, q, d - step, tries)) return true;
  }
  return false;
}

Gradients gather(const std::vector<const Tensor*>& tensors, bool scaled) {
  Gradients g;
  g.list.reserve(tensors.size());
  std::vector<Span> spans;
  if (scaled) {
    spans.reserve(tensors.size());
    g.in_place.reserve(tensors.size());
  }
  for (const Tensor* each : tensors) {
    const Tensor& t = *each;
    require(t.defined(), "gradients: a tensor is undefined");
    require(t.layout() == at::kStrided, "gradients: sparse gradients are not supported");
    const int type = element_type(t.scalar_type());
    require(type >= 0, "gradients: must be float32, float16 or bfloat16, not ", t.scalar_type());
    if (!g.any.defined()) g.any = t;
    require(t.device() == g.any.device(), "gradients: all must be on one device, not on ", g.any.device(), " and ", t.device());
    require(in_memory(t), "gradients: a tensor has no memory of its own, or too little");
    if (t.numel() == 0) continue;
    void* at_data = t.data_ptr();
    if (!t.is_non_overlapping_and_dense()) {
      const Tensor dense = t.contiguous();  // alive until the launch
      at_data = dense.data_ptr();
      g.copies.emplace_back(t, dense);
      if (scaled) {
        // to the furthest element; no two may share their memory
        int64_t reach = 1;
        for (int64_t i = 0; i < t.dim(); ++i) {
          require(t.size(i) == 1 || t.stride(i) != 0, "gradients: a tensor that repeats its memory cannot be scaled in place");
          reach += (t.size(i) - 1) * t.stride(i);
        }
        const auto at = (uintptr_t)t.data_ptr();
        spans.push_back({at, at + reach * t.element_size(), each});
      }
    } else if (scaled) {
      const auto at = (uintptr_t)at_data;
      spans.push_back({at, at + t.numel() * t.element_size(), each});
      g.in_place.push_back(each);
    }
    g.list.push_back({at_data, t.numel(), type});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t reach = 0;
  const bool apart_all = std::all_of(spans.begin(), spans.end(), [&](const Span& s) { return s.begin >= std::exchange(reach, s.end); });
  if (apart_all) spans.clear();  // as nearly always
  struct Open {
    uintptr_t begin, end;
    Lattice lattice;
    int64_t outer, rest;  // the largest stride, and what is left modulo it
  };
  std::vector<Open> open;  // those that reach past the begin of the next
  for (const Span& s : spans) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Open& o) { return o.end <= s.begin; }), open.end());
    Open mine{s.begin, s.end, Lattice(*s.tensor), 1, 0};
    for (const auto& d : mine.lattice.dims) mine.outer = std::max(mine.outer, d.stride);
    mine.rest = mine.lattice.modulo(mine.outer).length();
    for (const Open& o : open) {
      const int64_t ahead = (int64_t)(s.begin - o.begin), d = ahead % o.outer;
      if (mine.outer == o.outer && d >= o.rest && d + mine.rest <= o.outer) continue;  // columns of one matrix: told apart at once
      int tries = 2000;
      require(apart(o.lattice, mine.lattice, ahead, tries),
              "gradients: two of them share memory (the same tensor twice?), or are mixed in it in no regular way");
    }
    open.push_back(std::move(mine));
  }
  if (g.any.defined()) require(g.any.is_cuda(), "gradients: must be on the GPU: there is no CPU path");
  return g;
}

int norm_kind(double p) {
  const int kind = p == 1.0 ? RBL_NORM_1 : p == 2.0 ? RBL_NORM_2 : p == INFINITY ? RBL_NORM_INF : 0;
  require(kind, "gradients: norm_type must be 1, 2 or inf, not ", p);
  return kind;
}

Tensor norm_of(const Gradients& g, int kind) {
  c10::DeviceGuard guard(g.any.device());
  Tensor norm = at::empty({}, g.any.options().dtype(at::kFloat).layout(at::kStrided));
  const int n = (int)g.list.size();
  Tensor space = workspace(g.any, rbl_grad_workspace(g.list.data(), n));
  check(rbl_grad_norm(g.any.get_device(), g.list.data(), n, kind, norm.data_ptr<float>(), data(space),
                      space.defined() ? space.numel() : 0, stream_of(g.any)));
  return norm;
}

// The tensors of a Python list, by reference: the list holds them, and the interpreter stays locked.
std::vector<const Tensor*> tensors_of(const py::list& list) {
  std::vector<const Tensor*> out;
  out.reserve(list.size());
  for (const py::handle h : list) {
    if (!THPVariable_Check(h.ptr()))
      throw py::type_error("gradients: expected tensors, not " + std::string(Py_TYPE(h.ptr())->tp_name));
    out.push_back(&THPVariable_Unpack(h.ptr()));
  }
  return out;
}

Tensor grad_norm(const py::list& tensors, double norm_type) {
  const auto list = tensors_of(tensors);
  if (at::GradMode::is_enabled())
    for (const Tensor* t : list)
      require(!t->requires_grad(), "gradients: grad_norm has no gradient of its own; detach the tensors, or call it under no_grad");
  at::NoGradGuard no_grad;
  const int kind = norm_kind(norm_type);
  const Gradients g = gather(list, false);
  return g.any.defined() ? norm_of(g, kind) : at::zeros({});
}

Tensor clip_grad_norm(const py::list& parameters, double max_norm, double norm_type, bool error_if_nonfinite) {
  at::NoGradGuard no_grad;
  const int kind = norm_kind(norm_type);
  require(max_norm >= 0, "gradients: max_norm must be a number >= 0, not ", max_norm);
  std::vector<const Tensor*> grads;
  grads.reserve(parameters.size());
  for (const Tensor* p : tensors_of(parameters)) {
    const Tensor& grad = p->grad();
    if (grad.defined()) grads.push_back(&grad);
  }
  std::vector<Tensor> held;  // while other threads may run and give the parameters other gradients
  if (error_if_nonfinite) {
    held.reserve(grads.size());
    for (const Tensor*& t : grads) {
      held.push_back(*t);
      t = &held.back();
    }
  }
  const Gradients g = gather(grads, true);
  if (!g.any.defined()) return at::zeros({});
  c10::DeviceGuard guard(g.any.device());
  const int n = (int)g.list.size();
  Tensor norm;
  if (error_if_nonfinite) {
    require(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "gradients: error_if_nonfinite looks at the norm on the host, which a capture cannot do");
    norm = norm_of(g, kind);
    float value;
    {
      py::gil_scoped_release unlocked;
      value = norm.item<float>();
    }
    if (!std::isfinite(value))
      throw std::runtime_error(c10::str("gradients: the total norm of order ", norm_type, " is ", value,
                                        ", so they were not clipped (error_if_nonfinite)"));
    check(rbl_grad_scale(g.any.get_device(), g.list.data(), n, max_norm, norm.data_ptr<float>(), stream_of(g.any)));
  } else {
    norm = at::empty({}, g.any.options().dtype(at::kFloat));
    Tensor space = workspace(g.any, rbl_grad_workspace(g.list.data(), n));
    check(rbl_grad_clip(g.any.get_device(), g.list.data(), n, kind, max_norm, norm.data_ptr<float>(), data(space),
                        space.defined() ? space.numel() : 0, stream_of(g.any)));
  }
  for (const auto& c : g.copies) c.first.copy_(c.second);
  // as every operation in place: who has saved a gradient for another one finds out.  Not where the call was refused above.
  for (const Tensor* t : g.in_place)
    if (!t->is_inference()) torch::autograd::impl::bump_version(*t);
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"), py::arg("activation"),
        py::call_guard<py::gil_scoped_release>());
  m.def("grad_norm", &grad_norm, py::arg("tensors"), py::arg("norm_type"));
  m.def("clip_grad_norm", &clip_grad_norm, py::arg("parameters"), py::arg("max_norm"), py::arg("norm_type"),
        py::arg("error_if_nonfinite"));
}
