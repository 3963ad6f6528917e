// The pointwise operators (group norm, gated feed-forward, AdamW) as torch's C++ tensors and autograd
// see them: a call that has everything as the kernels want it goes from the Python function to the
// library without any more Python, and a backward pass runs in the engine's thread without the
// interpreter.  At small sizes the host is what such calls wait for: 2100 rows of 32 floats, group
// norm forward, 14 us a call through Python's binding.
//
// Each function says "not usual" (None, False) to arguments that need a look (strides, other types
// and devices, errors): the Python functions check those, raise or lay them out anew, and call again.
#include <Python.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include "ssc.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
namespace py = pybind11;

// Status codes as the exceptions that the library's other Python functions raise.
void check(int rc) {
  if (rc == SSC_OK) return;
  if (rc == SSC_EINVAL) throw py::value_error(ssc_last_error());
  TORCH_CHECK(false, ssc_last_error());
}

void *pointer(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
ssc_stream_t stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor bytes(size_t n, const Tensor &like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}
Tensor made(const Tensor &like, bool wanted) { return wanted ? at::empty(like.sizes(), like.options()) : Tensor(); }

// Element type of a float, half or bfloat16 tensor, or -1.
int elem(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SSC_F32;
    case at::kHalf: return SSC_F16;
    case at::kBFloat16: return SSC_BF16;
    default: return -1;
  }
}
bool plain(const Tensor &t) { return t.layout() == at::kStrided && t.is_cuda() && t.is_contiguous(); }
bool at16(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// A tensor (or None, an undefined one) from Python; false: something else.
bool take(const py::handle &h, Tensor &t) {
  if (h.is_none()) return true;
  if (!THPVariable_Check(h.ptr())) return false;
  t = THPVariable_Unpack(h.ptr());
  return true;
}

bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
void no_forward_mode(std::initializer_list<Tensor> inputs) {
  for (const Tensor &t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                                "the pointwise operators have no forward-mode derivative");
}

// A node of the autograd graph that can be differentiated once: where its gradients are to be
// differentiated again, what does so raises an error.
struct Once : torch::autograd::Node {
  virtual variable_list gradients(const Tensor &dy) = 0;
  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(num_outputs());
    const bool again = at::GradMode::is_enabled();
    variable_list out;
    {
      at::NoGradGuard no_grad;
      const c10::DeviceGuard device(grads[0].device());
      out = gradients(grads[0].contiguous());
    }
    if (!again) return out;
    for (Tensor &t : out)
      if (t.defined()) t.requires_grad_(true);
    return torch::autograd::DelayedError("trying to differentiate twice: " + name() + " can be differentiated once",
                                         (int64_t)out.size())(std::move(out));
  }
};

// A node whose gradients go to `inputs`.
template <typename N> std::shared_ptr<N> new_node(std::initializer_list<Tensor> inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  edges.reserve(inputs.size());
  for (const Tensor &t : inputs)
    edges.emplace_back(wants(t) ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
  node->set_next_edges(std::move(edges));
  return node;
}

// ---- group norm -----------------------------------------------------------------------------
struct NormArgs {
  int32_t n, c, clouds, groups, elem, wtype, act;
  size_t workspace() const { return ssc_groupnorm_workspace_bytes(n, c, clouds, groups); }
};

Tensor norm_forward(const NormArgs &a, const Tensor &x, const Tensor &offsets, const Tensor &w, const Tensor &b,
                    double eps, Tensor &stats) {
  Tensor y = at::empty(x.sizes(), x.options());
  stats = at::empty({2, a.clouds, a.groups}, x.options().dtype(at::kFloat));
  const Tensor ws = bytes(a.workspace(), x);
  float *mean = stats.data_ptr<float>();
  check(ssc_groupnorm_fwd(a.elem, pointer(x), a.n, a.c, offsets.data_ptr<int32_t>(), a.clouds, a.groups, a.wtype,
                          pointer(w), pointer(b), (float)eps, a.act, pointer(y), mean,
                          mean + (int64_t)a.clouds * a.groups, ws.data_ptr(), ws.numel(), stream_of(x)));
  return y;
}

struct SscGroupNormBackward : Once {
  NormArgs a;
  SavedVariable x_, w_, b_, offsets_, stats_;
  std::string name() const override { return "SscGroupNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable *v : {&x_, &w_, &b_, &offsets_, &stats_}) v->reset_data();
  }
  variable_list gradients(const Tensor &dy) override {
    const Tensor x = x_.unpack(), w = w_.unpack(), b = b_.unpack(), offsets = offsets_.unpack();
    const Tensor stats = stats_.unpack();
    Tensor dx = made(x, task_should_compute_output(0));
    Tensor dw = w.defined() ? made(w, task_should_compute_output(1)) : Tensor();
    Tensor db = b.defined() ? made(b, task_should_compute_output(2)) : Tensor();
    if (a.n == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
      return {dx, dw, db};
    }
    const Tensor ws = bytes(a.workspace(), x);
    float *mean = stats.data_ptr<float>();
    check(ssc_groupnorm_bwd(a.elem, x.data_ptr(), dy.data_ptr(), a.n, a.c, offsets.data_ptr<int32_t>(), a.clouds,
                            a.groups, a.wtype, pointer(w), pointer(b), a.act, mean,
                            mean + (int64_t)a.clouds * a.groups, pointer(dx), pointer(dw), pointer(db),
                            ws.data_ptr(), ws.numel(), stream_of(x)));
    return {dx, dw, db};
  }
};

// Contiguous rows x [n, c], int32 offsets, parameters of one type; else None.
py::object group_norm(py::handle hx, py::handle ho, int64_t groups, py::handle hw, py::handle hb, double eps,
                      int act) {
  Tensor x, offsets, w, b;
  if (!take(hx, x) || !take(ho, offsets) || !take(hw, w) || !take(hb, b) || !x.defined() || !offsets.defined())
    return py::none();
  if (!plain(x) || x.dim() != 2 || elem(x) < 0 || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX) return py::none();
  NormArgs a;
  a.n = (int32_t)x.size(0);
  a.c = (int32_t)x.size(1);
  a.elem = a.wtype = elem(x);
  a.act = act;
  if (groups < 1 || a.c < 1 || a.c % groups != 0 || !(eps >= 0)) return py::none();
  a.groups = (int32_t)groups;
  if (!plain(offsets) || offsets.dim() != 1 || offsets.scalar_type() != at::kInt ||
      offsets.get_device() != x.get_device() || offsets.numel() < (a.n > 0 ? 2 : 1) || offsets.numel() > INT32_MAX)
    return py::none();
  a.clouds = (int32_t)offsets.numel() - 1;
  for (const Tensor *t : {&w, &b})
    if (t->defined()) {
      if (!plain(*t) || t->dim() != 1 || t->size(0) != a.c || t->get_device() != x.get_device() ||
          (elem(*t) != a.elem && elem(*t) != SSC_F32) ||
          (t == &b && w.defined() && w.scalar_type() != b.scalar_type()))
        return py::none();
      a.wtype = elem(*t);
    }
  no_forward_mode({x, w, b});
  const c10::DeviceGuard device(x.device());
  Tensor stats;
  if (!at::GradMode::is_enabled() || !(wants(x) || wants(w) || wants(b))) {
    at::NoGradGuard no_grad;
    return py::cast(norm_forward(a, x, offsets, w, b, eps, stats));
  }
  auto node = new_node<SscGroupNormBackward>({x, w, b});
  Tensor y;
  {
    at::NoGradGuard no_grad;
    y = norm_forward(a, x, offsets, w, b, eps, stats);
  }
  node->a = a;
  node->x_ = SavedVariable(x, false);
  node->w_ = SavedVariable(w, false);
  node->b_ = SavedVariable(b, false);
  node->offsets_ = SavedVariable(offsets, false);
  node->stats_ = SavedVariable(stats, false);
  torch::autograd::set_history(y, node);
  return py::cast(y);
}

// ---- gated feed-forward ---------------------------------------------------------------------
struct GatedArgs {
  int64_t m, k, h;
  int32_t elem, act;
};

Tensor gated_forward(const GatedArgs &a, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &bg,
                     const Tensor &bu, bool keep, Tensor &kept) {
  Tensor y = at::empty({a.m, a.h}, x.options());
  if (keep) kept = bytes(ssc_gated_kept_bytes(a.elem, a.m, a.h), x);
  const Tensor ws = bytes(ssc_gated_fwd_workspace_bytes(a.elem, a.m, a.k, a.h), x);
  check(ssc_gated_fwd(a.elem, pointer(x), a.m, a.k, wg.data_ptr(), wu.data_ptr(), a.h, pointer(bg), pointer(bu),
                      a.act, pointer(y), pointer(kept), ws.data_ptr(), ws.numel(), stream_of(x)));
  return y;
}

struct SscGatedLinearBackward : Once {
  GatedArgs a;
  SavedVariable x_, wg_, wu_, kept_;
  std::string name() const override { return "SscGatedLinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable *v : {&x_, &wg_, &wu_, &kept_}) v->reset_data();
  }
  variable_list gradients(const Tensor &dy) override {
    const Tensor x = x_.unpack(), wg = wg_.unpack(), wu = wu_.unpack(), kept = kept_.unpack();
    const bool gate = task_should_compute_output(1), up = task_should_compute_output(2);
    Tensor dx = made(x, task_should_compute_output(0));
    Tensor dwg = made(wg, gate || up), dwu = made(wu, gate || up);  // (one product gives both)
    Tensor db[2];
    for (int i = 0; i < 2; ++i)
      if (task_should_compute_output(3 + i)) db[i] = at::empty({a.h}, x.options());
    if (a.m == 0) {
      for (Tensor *t : {&dwg, &dwu, &db[0], &db[1]})
        if (t->defined()) t->zero_();
    } else {
      const Tensor ws = bytes(ssc_gated_bwd_workspace_bytes(a.elem, a.m, a.k, a.h), x);
      check(ssc_gated_bwd(a.elem, x.data_ptr(), a.m, a.k, wg.data_ptr(), wu.data_ptr(), a.h, a.act,
                          kept.data_ptr(), dy.data_ptr(), pointer(dx), pointer(dwg), pointer(dwu), pointer(db[0]),
                          pointer(db[1]), ws.data_ptr(), ws.numel(), stream_of(x)));
    }
    return {dx, gate ? dwg : Tensor(), up ? dwu : Tensor(), db[0], db[1]};
  }
};

// Contiguous rows x [m, k], weights [h, k] and biases [h] of one type, x and weights at 16 bytes;
// else None.
py::object gated_linear(py::handle hx, py::handle hg, py::handle hu, py::handle hbg, py::handle hbu, int act) {
  Tensor x, wg, wu, bg, bu;
  if (!take(hx, x) || !take(hg, wg) || !take(hu, wu) || !take(hbg, bg) || !take(hbu, bu) || !x.defined() ||
      !wg.defined() || !wu.defined())
    return py::none();
  if (!plain(x) || x.dim() != 2 || elem(x) < 0 || !at16(x)) return py::none();
  const GatedArgs a = {x.size(0), x.size(1), wg.dim() == 2 ? wg.size(0) : 0, elem(x), act};
  if (a.h < 1 || a.k < 1) return py::none();
  for (const Tensor *t : {&wg, &wu})
    if (t->scalar_type() != x.scalar_type() || !plain(*t) || t->dim() != 2 || t->size(0) != a.h ||
        t->size(1) != a.k || t->get_device() != x.get_device() || !at16(*t))
      return py::none();
  for (const Tensor *t : {&bg, &bu})
    if (t->defined() && (t->scalar_type() != x.scalar_type() || !plain(*t) || t->dim() != 1 ||
                         t->size(0) != a.h || t->get_device() != x.get_device()))
      return py::none();
  no_forward_mode({x, wg, wu, bg, bu});
  const c10::DeviceGuard device(x.device());
  Tensor kept;
  if (!at::GradMode::is_enabled() || !(wants(x) || wants(wg) || wants(wu) || wants(bg) || wants(bu))) {
    at::NoGradGuard no_grad;
    return py::cast(gated_forward(a, x, wg, wu, bg, bu, false, kept));
  }
  auto node = new_node<SscGatedLinearBackward>({x, wg, wu, bg, bu});
  Tensor y;
  {
    at::NoGradGuard no_grad;
    y = gated_forward(a, x, wg, wu, bg, bu, true, kept);
  }
  node->a = a;
  node->x_ = SavedVariable(x, false);
  node->wg_ = SavedVariable(wg, false);
  node->wu_ = SavedVariable(wu, false);
  node->kept_ = SavedVariable(kept, false);
  torch::autograd::set_history(y, node);
  return py::cast(y);
}

// ---- AdamW ----------------------------------------------------------------------------------
// A list or tuple of tensors.
struct Tensors {
  py::object held;
  Py_ssize_t count = -1;
  PyObject **items = nullptr;
  explicit Tensors(const py::handle &h) {
    if (h.is_none() || !(PyList_Check(h.ptr()) || PyTuple_Check(h.ptr()))) return;
    held = py::reinterpret_borrow<py::object>(h);
    count = PySequence_Fast_GET_SIZE(h.ptr());
    items = PySequence_Fast_ITEMS(h.ptr());
  }
  // The i-th one if it is contiguous and on the given GPU (device < 0: any).
  const Tensor *get(Py_ssize_t i, int device) const {
    if (!THPVariable_Check(items[i])) return nullptr;
    const Tensor &t = THPVariable_Unpack(items[i]);
    return plain(t) && (device < 0 || t.get_device() == device) ? &t : nullptr;
  }
};

// Fills the moments' part of a table's entry: codes and scales (8 bits) or floats.
bool put_moments(ssc_adamw_tensor &e, const Tensors *moments, Py_ssize_t i, bool eight, int device) {
  const at::ScalarType codes[2] = {eight ? at::kChar : at::kFloat, eight ? at::kByte : at::kFloat};
  void *p[4] = {nullptr, nullptr, nullptr, nullptr};
  for (int k = 0; k < (eight ? 4 : 2); ++k) {
    const Tensor *t = moments[k].get(i, device);
    if (!t || t->scalar_type() != (k < 2 ? codes[k] : at::kFloat) ||
        t->numel() != (k < 2 ? e.numel : (e.numel + SSC_ADAMW_BLOCK - 1) / SSC_ADAMW_BLOCK))
      return false;
    p[k] = t->data_ptr();
  }
  e.exp_avg = p[0];
  e.exp_avg_sq = p[1];
  e.exp_avg_scale = static_cast<float *>(p[2]);
  e.exp_avg_sq_scale = static_cast<float *>(p[3]);
  return true;
}

// Contiguous tensors on one GPU that fit one another; else False, and nothing is done.
bool adamw(py::handle params, py::handle grads, py::handle m, py::handle v, py::handle mq, py::handle vq,
           int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay) {
  const Tensors p(params), g(grads), moments[4] = {Tensors(m), Tensors(v), Tensors(mq), Tensors(vq)};
  const bool eight = !mq.is_none();
  if (p.count < 1 || g.count != p.count || p.count > INT32_MAX || eight == vq.is_none()) return false;
  for (int k = 0; k < (eight ? 4 : 2); ++k)
    if (moments[k].count != p.count) return false;
  std::vector<ssc_adamw_tensor> table(p.count);
  int device = -1;
  for (Py_ssize_t i = 0; i < p.count; ++i) {
    const Tensor *t = p.get(i, device);
    if (!t || elem(*t) < 0) return false;
    device = t->get_device();
    const Tensor *d = g.get(i, device);
    if (!d || d->scalar_type() != t->scalar_type() || d->sizes() != t->sizes()) return false;
    ssc_adamw_tensor &e = table[i];
    e.param = t->data_ptr();
    e.grad = d->data_ptr();
    e.numel = t->numel();
    e.dtype = elem(*t);
    if (!put_moments(e, moments, i, eight, device)) return false;
  }
  const Tensor &first = THPVariable_Unpack(p.items[0]);
  const c10::DeviceGuard guard(first.device());
  check(ssc_adamw_step(table.data(), (int32_t)p.count, eight ? 8 : 32, lr, beta1, beta2, eps, weight_decay, step,
                       stream_of(first)));
  for (Py_ssize_t i = 0; i < p.count; ++i) {
    const Tensor &t = THPVariable_Unpack(p.items[i]);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  return true;
}

// The values of 8-bit moments, written to the float tensors out_m and out_v; else False.
bool adamw_values(py::handle out_m, py::handle out_v, py::handle m, py::handle v, py::handle mq, py::handle vq) {
  const Tensors o[2] = {Tensors(out_m), Tensors(out_v)};
  const Tensors moments[4] = {Tensors(m), Tensors(v), Tensors(mq), Tensors(vq)};
  const Py_ssize_t count = moments[0].count;
  if (count < 1 || count > INT32_MAX || o[0].count != count || o[1].count != count) return false;
  for (int k = 1; k < 4; ++k)
    if (moments[k].count != count) return false;
  std::vector<ssc_adamw_tensor> table(count);
  int device = -1;
  for (Py_ssize_t i = 0; i < count; ++i) {
    ssc_adamw_tensor &e = table[i];
    const Tensor *t[2] = {o[0].get(i, device), nullptr};
    if (!t[0]) return false;
    device = t[0]->get_device();
    t[1] = o[1].get(i, device);
    if (!t[1] || t[0]->scalar_type() != at::kFloat || t[1]->scalar_type() != at::kFloat ||
        t[1]->numel() != t[0]->numel())
      return false;
    e.param = t[0]->data_ptr();
    e.grad = t[1]->data_ptr();
    e.numel = t[0]->numel();
    e.dtype = SSC_F32;
    if (!put_moments(e, moments, i, true, device)) return false;
  }
  const Tensor &first = THPVariable_Unpack(moments[0].items[0]);
  const c10::DeviceGuard guard(first.device());
  check(ssc_adamw_values(table.data(), (int32_t)count, stream_of(first)));
  return true;
}

}  // namespace

PYBIND11_MODULE(_pointwise, m) {
  m.doc() = "The pointwise operators for tensors that are as the kernels want them.";
  m.def("group_norm", &group_norm);
  m.def("gated_linear", &gated_linear);
  m.def("adamw", &adamw);
  m.def("adamw_values", &adamw_values);
}
