// Calls of a training step on PyTorch's tensors: layer norm with its gradients, AdamW over a list of parameters (module orca_b200._rows).
//
// A step over a model's parameters takes the GPU some ten microseconds: what the host does for each of them (its gradient, its moments, checks)
// is done here.  orca_b200/norm.py and orca_b200/optim.py are the only callers.
#include <algorithm>
#include <functional>

#include "torch_calls.h"

namespace orca_torch {
namespace {

bool is_real(const Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// Rows of the last dimension at one distance from each other.
struct Rows {
  Tensor t;             // as it is, or a contiguous copy
  int64_t n, width, stride;
  explicit Rows(const Tensor &given) : t(given.is_neg() ? given.resolve_neg() : given) {
    width = t.size(-1);
    n = t.numel() / width;
    if (!even()) t = t.contiguous(), stride = width;
    else if (width <= 8192 && (n > 16 || width > 512) && !borders()) t = t.clone(at::MemoryFormat::Contiguous), stride = width;
  }
  // Whether rows lie as new contiguous ones do: on borders of eight bytes, or where four values are four of those.  A copy of others takes less than reading them by
  // values, but for few narrow rows, and for wide ones, which are gone through by blocks from L2 either way.  One value off, us forward / gradients by values, and with
  // copies of rows and gradients: fp32 1 row of 172 2.9 / 5.9, 3.3 / 5.8; 16 of 172 3.0 / 7.9, 3.7 / 6.3; 64 of 172 3.3 / 14.0, 3.7 / 6.7; 1 of 688 3.8 / 7.0, 3.4 / 6.5;
  // 64 of 2051 14.7 / 31.0, 4.3 / 8.9; bf16 66 001 of 172 176 / 285, 57 / 132; 4096 of 8188 99 / 207, 77 / 141, of 8200 98 / 204, 132 / 267.
  bool borders() const {
    const int64_t size = t.element_size(), at = (int64_t)(uintptr_t)t.data_ptr(), row = width * size, step = stride * size;
    return ((at | row | step) % 8 == 0) || (at % (4 * size) == 0 && (step - row) % (4 * size) == 0);
  }
  bool even() {
    stride = width;
    if (t.is_contiguous()) return true;
    if (width > 1 && t.stride(-1) != 1) return false;
    int64_t next = -1;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
      if (t.size(d) == 1) continue;
      if (next < 0) stride = t.stride(d);
      else if (t.stride(d) != next) return false;
      next = t.stride(d) * t.size(d);
    }
    return true;
  }
};

// ---------------------------------------------------------------------------------------------- layer norm
void expect_rows(const Tensor &x) {
  TORCH_CHECK_TYPE(is_real(x) && x.is_cuda() && x.layout() == at::kStrided, "layer_norm takes fp32, bf16 or fp16 on a CUDA device, not ", x.scalar_type(), " on ",
                   x.device());
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0 && x.size(-1) <= 1 << 24, "rows of 1 to 2^24 values, not a tensor of sizes ", x.sizes());
}
void expect_affine(const Tensor &w, const Tensor &x, const char *name) {
  if (!w.defined()) return;
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1) && w.device() == x.device() && w.layout() == at::kStrided, name, " is a tensor [", x.size(-1),
                    "] on ", x.device(), "; not ", w.sizes(), " on ", w.device());
  TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, name, " is of the rows' type or fp32, not ", w.scalar_type());
}
void expect_no_tangent(const Tensor &t, const char *what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward derivative");
}
Tensor plain(const Tensor &w) { return !w.defined() ? w : w.is_neg() ? w.resolve_neg().contiguous() : w.contiguous(); }
void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor normed(const Tensor &given, const Tensor &weight, const Tensor &bias, double eps) {
  const c10::cuda::CUDAGuard guard(given.device());
  const Rows x(given);
  const Tensor w = plain(weight), b = plain(bias);
  Tensor out = at::empty(given.sizes(), x.t.options());
  check(orca_layer_norm(data(x.t), x.stride, x.n, (int32_t)x.width, type_of(x.t), data(w), data(b), w.defined() ? type_of(w) : b.defined() ? type_of(b) : type_of(x.t),
                        (float)eps, data(out), stream_of(out)));
  return out;
}

struct Wanted { bool x, weight, bias; };
struct Grads { Tensor x, weight, bias; };
Grads gradients(const Tensor &grad_out, const Tensor &given, const Tensor &weight, at::ScalarType affine, double eps, const Wanted &want) {
  const c10::cuda::CUDAGuard guard(given.device());
  const Rows x(given), g(grad_out);
  const Tensor w = plain(weight);
  Grads d;
  if (want.x) d.x = at::empty(given.sizes(), x.t.options());
  if (want.weight) d.weight = at::empty({x.width}, x.t.options().dtype(affine));
  if (want.bias) d.bias = at::empty({x.width}, x.t.options().dtype(affine));
  const int64_t need = want.weight || want.bias ? orca_layer_norm_grad_workspace_bytes(x.n, (int32_t)x.width) : 0;
  TORCH_CHECK(need >= 0, "layer_norm: ", x.n, " rows");
  Tensor ws;
  if (need > 0) ws = at::empty({need}, x.t.options().dtype(at::kByte));
  check(orca_layer_norm_grad(data(g.t), g.stride, data(x.t), x.stride, x.n, (int32_t)x.width, type_of(x.t), data(w),
                             affine == at::kFloat ? ORCA_F32 : type_of(x.t), (float)eps, data(d.x), data(d.weight), data(d.bias), data(ws), need,
                             stream_of(x.t)));
  return d;
}
// The same as results that have no derivative: a tangent is refused, and so is, by whoever asks for it, a backward pass.
Grads final_gradients(const Tensor &grad_out, const Tensor &x, const Tensor &weight, at::ScalarType affine, double eps, const Wanted &want) {
  for (const Tensor *t : {&grad_out, &x, &weight}) expect_no_tangent(*t, "the gradient of layer_norm");
  Grads d;
  {
    const at::NoGradGuard no_grad;
    d = gradients(grad_out, x, weight, affine, eps, want);
  }
  if (at::GradMode::is_enabled() && (grad_out.requires_grad() || x.requires_grad() || (weight.defined() && weight.requires_grad())))
    for (Tensor *t : {&d.x, &d.weight, &d.bias})
      if (t->defined())
        ag::set_history(*t, std::make_shared<ag::Error>("the gradient of layer_norm has no derivative", ag::collect_next_edges(grad_out, x, weight)));
  return d;
}

struct NormBackward : public ag::Node {
  ag::SavedVariable x, weight;
  bool has_weight = false, released = false;
  at::ScalarType affine;
  double eps;

  ag::variable_list apply(ag::variable_list &&grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, ag::ERR_BACKWARD_TWICE);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    refuse_capture(*this, grads[0], "layer_norm: this backward pass is captured in a graph while an older graph of its inputs lives; release that, or call layer_norm_grad");
    const Wanted want = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
    Grads d = final_gradients(grads[0], x.unpack(), has_weight ? weight.unpack() : Tensor(), affine, eps, want);
    return {d.x, d.weight, d.bias};
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    released = true;
  }
  std::string name() const override { return "LayerNormBackward"; }
};

Tensor maybe(PyObject *o, const char *name) { return o == Py_None ? Tensor() : tensor(o, name); }

}  // namespace

// (x, weight or None, bias or None, eps)
PyObject *norm(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 4, "norm(x, weight, bias, eps)");
  const Tensor &x = tensor(args[0], "x");
  const Tensor weight = maybe(args[1], "weight"), bias = maybe(args[2], "bias");
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  expect_rows(x), expect_affine(weight, x, "weight"), expect_affine(bias, x, "bias");
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight and bias are of one type");
  Tensor out;
  try {
    const pybind11::gil_scoped_release no_gil;
    for (const Tensor *t : {&x, &weight, &bias}) expect_no_tangent(*t, "layer_norm");
    {
      const at::NoGradGuard no_grad;
      out = normed(x, weight, bias, eps);
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()))) {
      auto node = std::make_shared<NormBackward>();
      node->x = ag::SavedVariable(x, false);
      node->has_weight = weight.defined();
      if (weight.defined()) node->weight = ag::SavedVariable(weight, false);
      node->affine = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
      node->eps = eps;
      node->set_next_edges(ag::collect_next_edges(x, weight, bias));
      ag::set_history(out, node);
    }
  } catch (const Failed &e) {
    return raise(e.rc);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (grad_out, x, weight or None, eps)
PyObject *norm_grad(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 4, "norm_grad(grad_out, x, weight, eps)");
  const Tensor &g = tensor(args[0], "grad_out"), &x = tensor(args[1], "x");
  const Tensor weight = maybe(args[2], "weight");
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  expect_rows(x), expect_affine(weight, x, "weight");
  TORCH_CHECK_VALUE(g.sizes() == x.sizes() && g.device() == x.device() && g.scalar_type() == x.scalar_type() && g.layout() == at::kStrided, "gradients are of ",
                    x.scalar_type(), ", sizes ", x.sizes(), " on ", x.device(), "; not ", g.scalar_type(), " ", g.sizes(), " on ", g.device());
  Grads d;
  try {
    const pybind11::gil_scoped_release no_gil;
    d = final_gradients(g, x, weight, weight.defined() ? weight.scalar_type() : x.scalar_type(), eps, {true, true, true});
  } catch (const Failed &e) {
    return raise(e.rc);
  }
  PyObject *t = PyTuple_New(3);
  if (t == nullptr) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(d.x)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(d.weight)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(d.bias)));
  return t;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- AdamW
namespace {

PyObject *key(const char *name) { return PyUnicode_InternFromString(name); }
// (made once; the interpreter keeps them)
struct Keys {
  PyObject *params = key("params"), *lr = key("lr"), *betas = key("betas"), *eps = key("eps"), *weight_decay = key("weight_decay"), *step = key("step"),
           *mean = key("exp_avg"), *square = key("exp_avg_sq"), *exponents = key("exponents");
};
const Keys &keys() {
  static const Keys k;
  return k;
}
PyObject *item(PyObject *dict, PyObject *k) {
  PyObject *v = PyDict_Check(dict) ? PyDict_GetItemWithError(dict, k) : nullptr;
  if (v == nullptr && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(v != nullptr, "AdamW: no '", PyUnicode_AsUTF8(k), "' where it is kept");
  return v;
}
double number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) throw python_error();
  return v;
}
// Whether elements lie in memory in the order of those of p, which is contiguous or not (`whole`).
bool beside(const Tensor &t, const Tensor &p, bool whole) {
  return t.is_contiguous() ? whole || t.dim() == 1 : t.sizes() == p.sizes() && t.strides() == p.strides();
}

// Parameters with a gradient (all of them: `all`), their moments and groups.
struct Step {
  std::vector<orca_adamw_tensor_t> tensors;
  std::vector<orca_adamw_group_t> groups;
  std::vector<const Tensor *> params;      // (held by the groups)
  std::vector<Tensor> copies;              // of gradients that lie in another order
  c10::Device device;

  void add_group(PyObject *g) {
    const Keys &k = keys();
    PyObject *lr = item(g, k.lr), *betas = item(g, k.betas);
    TORCH_CHECK_VALUE(PySequence_Check(betas) && PySequence_Size(betas) == 2, "AdamW: two betas");
    orca_adamw_group_t h = {};
    for (int i = 0; i < 2; ++i) {
      PyObject *b = PySequence_GetItem(betas, i);
      if (b == nullptr) throw python_error();
      const double v = PyFloat_AsDouble(b);
      Py_DECREF(b);
      if (PyErr_Occurred()) throw python_error();
      TORCH_CHECK_VALUE(v >= 0 && v < 1, "AdamW: betas are from 0 to below 1, not ", v);
      (i == 0 ? h.beta1 : h.beta2) = v;
    }
    if (THPVariable_Check(lr) && THPVariable_Unpack(lr).is_cuda()) {
      const Tensor &t = THPVariable_Unpack(lr);
      TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.numel() == 1 && t.device() == device, "AdamW: lr on the device is one fp32 value on ", device);
      h.d_lr = t.data_ptr<float>();
    } else {
      h.lr = number(lr);
      TORCH_CHECK_VALUE(h.lr >= 0, "AdamW: lr ", h.lr);
    }
    h.eps = number(item(g, k.eps));
    h.weight_decay = number(item(g, k.weight_decay));
    TORCH_CHECK_VALUE((h.eps == 0 || (h.eps >= 1.2e-38 && h.eps <= 3.4e38)) && h.weight_decay >= 0, "AdamW: eps ", h.eps, ", weight_decay ", h.weight_decay);
    groups.push_back(h);
  }
  // What is kept of a parameter: its entries in their order, for a search for each takes longer (a step over 293 tensors 37 us, 35 this way).
  struct Kept { PyObject *step = nullptr, *mean = nullptr, *square = nullptr, *exponents = nullptr; };
  static Kept kept(PyObject *state, int bits) {
    const Keys &k = keys();
    Kept s;
    TORCH_CHECK_TYPE(PyDict_Check(state), "AdamW: a parameter's state is a dict");
    PyObject *name, *value;
    int missing = bits == 8 ? 4 : 3;
    for (Py_ssize_t at = 0; missing != 0 && PyDict_Next(state, &at, &name, &value);)
      if (name == k.step) s.step = value, --missing;
      else if (name == k.mean) s.mean = value, --missing;
      else if (name == k.square) s.square = value, --missing;
      else if (name == k.exponents) s.exponents = value, missing -= bits == 8;
    if (s.step == nullptr) s.step = item(state, k.step);
    if (s.mean == nullptr) s.mean = item(state, k.mean);
    if (s.square == nullptr) s.square = item(state, k.square);
    if (s.exponents == nullptr && bits == 8) s.exponents = item(state, k.exponents);
    return s;
  }
  const Tensor &moment(PyObject *o, PyObject *k, at::ScalarType type, int64_t n) const {
    TORCH_CHECK_TYPE(THPVariable_Check(o), "AdamW: '", PyUnicode_AsUTF8(k), "' is a tensor");
    const Tensor &t = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == device && t.numel() == n, "AdamW: '", PyUnicode_AsUTF8(k), "' is ", n, " of ", type, " on ", device,
                      "; not ", t.numel(), " of ", t.scalar_type(), " on ", t.device());
    return t;
  }
  void add(const Tensor &p, PyObject *state, bool all, int bits) {
    const Tensor &given = p.grad();
    if (!all && !given.defined()) return;
    const Keys &k = keys();
    TORCH_CHECK_VALUE(p.device() == device && is_real(p) && p.is_non_overlapping_and_dense() && !p.is_neg(),
                      "AdamW: parameters are dense, in fp32, bf16 or fp16, on ", device, "; not ", p.scalar_type(), " ", p.sizes(), " on ", p.device());
    TORCH_CHECK(all || !p.is_inference() || c10::InferenceMode::is_enabled(), "AdamW: a parameter made in inference mode changes in inference mode only");
    const int64_t n = p.numel();
    const at::ScalarType type = bits == 8 ? at::kByte : at::kFloat;
    const Kept s = kept(state, bits);
    const Tensor &m = moment(s.mean, k.mean, type, n), &v = moment(s.square, k.square, type, n), &step = moment(s.step, k.step, at::kInt, 1);
    const bool whole = p.is_contiguous();
    TORCH_CHECK_VALUE(beside(m, p, whole) && beside(v, p, whole), "AdamW: moments lie in memory as their parameter does");
    orca_adamw_tensor_t t = {p.data_ptr(), nullptr, m.data_ptr(), v.data_ptr(), nullptr, step.data_ptr<int32_t>(), n, type_of(p), (int32_t)groups.size() - 1};
    if (bits == 8) {
      const Tensor &e = moment(s.exponents, k.exponents, at::kByte, 2 * ((n + 255) / 256));
      TORCH_CHECK_VALUE(e.is_contiguous(), "AdamW: exponents are contiguous");
      t.exponents = e.data_ptr<uint8_t>();
    }
    if (!all) {
      TORCH_CHECK_VALUE(given.layout() == at::kStrided && given.device() == device && given.scalar_type() == p.scalar_type() && given.sizes() == p.sizes(),
                        "AdamW: a gradient is dense, of its parameter's type and sizes");
      if (given.is_neg() || !(given.is_contiguous() ? whole : given.strides() == p.strides())) {
        copies.push_back(at::empty_like(p).copy_(given));
        t.grad = copies.back().data_ptr();
      } else {
        t.grad = given.data_ptr();
      }
    }
    tensors.push_back(t);
    params.push_back(&p);
  }
  // A count that two tensors had would be counted twice.  (Those of a group lie in order, as they were made.)
  void expect_own_steps() const {
    bool rising = true;
    for (size_t i = 1; i < tensors.size(); ++i) rising &= std::less<const int32_t *>()(tensors[i - 1].step, tensors[i].step);
    if (rising) return;
    std::vector<const int32_t *> steps;
    steps.reserve(tensors.size());
    for (const orca_adamw_tensor_t &t : tensors) steps.push_back(t.step);
    std::sort(steps.begin(), steps.end(), std::less<const int32_t *>());
    TORCH_CHECK_VALUE(std::adjacent_find(steps.begin(), steps.end()) == steps.end(), "AdamW: each parameter has a 'step' of its own");
  }
  // (groups of the optimiser, states of its parameters by parameter: in their order as a rule, for a search for each takes longer)
  Step(PyObject *param_groups, PyObject *states, const Tensor &work, bool all, int bits) : device(work.device()) {
    TORCH_CHECK_TYPE(PyList_Check(param_groups) && PyDict_Check(states), "AdamW: a list of groups, a dict of states");
    const Py_ssize_t n = PyDict_Size(states);
    tensors.reserve(n), params.reserve(n);
    Py_ssize_t at = 0, next = 0;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(param_groups); ++i) {
      PyObject *g = PyList_GET_ITEM(param_groups, i), *list = item(g, keys().params);
      TORCH_CHECK_TYPE(PyList_Check(list), "AdamW: a group's parameters are a list");
      add_group(g);
      for (Py_ssize_t j = 0; j < PyList_GET_SIZE(list); ++j, ++at) {
        PyObject *p = PyList_GET_ITEM(list, j), *of = nullptr, *state = nullptr;
        if (C10_UNLIKELY(!PyDict_Next(states, &next, &of, &state) || of != p)) {
          state = PyDict_GetItemWithError(states, p);
          if (state == nullptr && PyErr_Occurred()) throw python_error();
          TORCH_CHECK_VALUE(state != nullptr, "AdamW: a parameter has no state: parameters are added by add_param_group");
        }
        add(tensor(p, "a parameter"), state, all, bits);
      }
    }
    if (at == n) return;
    Py_ssize_t of_params = 0;      // (there may be others' entries)
    PyObject *of, *state;
    for (next = 0; PyDict_Next(states, &next, &of, &state);) of_params += THPVariable_Check(of);
    TORCH_CHECK_VALUE(at == of_params, "AdamW: parameters are not taken out of their groups");
  }
};

}  // namespace

// (param_groups, state, bits, max_norm or negative, norm, work)
PyObject *adamw(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 6, "adamw(param_groups, state, bits, max_norm, norm, work)");
  const Tensor &out = tensor(args[4], "norm"), &work = tensor(args[5], "work");
  const int bits = (int)PyLong_AsLong(args[2]);
  const double max_norm = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(work.device());
  const Step s(args[0], args[1], work, false, bits);
  s.expect_own_steps();
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    rc = orca_adamw_step(s.tensors.data(), (int32_t)s.tensors.size(), s.groups.data(), (int32_t)s.groups.size(), bits, max_norm, out.data_ptr<float>(),
                         work.data_ptr(), stream_of(work));
  }
  if (rc != ORCA_OK) return raise(rc);
  for (const Tensor *p : s.params) p->unsafeGetTensorImpl()->bump_version();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (param_groups, state, work): values of moments in 8 bits
PyObject *moments(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 3, "moments(param_groups, state, work)");
  const Tensor &work = tensor(args[2], "work");
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(work.device());
  Step s(args[0], args[1], work, true, 8);
  // one buffer of bf16 for all of them, each from a multiple of 256 bytes on: an allocation each takes longer than the kernel
  constexpr int64_t ON = 128;
  int64_t total = 0;
  for (const orca_adamw_tensor_t &t : s.tensors) total += 2 * ((t.n + ON - 1) / ON * ON);
  const Tensor all = at::empty({total}, work.options().dtype(at::kBFloat16));
  std::vector<Tensor> values[2];
  int64_t offset = 0;
  for (size_t i = 0; i < s.tensors.size(); ++i)
    for (int k = 0; k < 2; ++k) {
      auto impl = c10::make_intrusive<at::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
      impl->set_sizes_and_strides(s.params[i]->sizes(), s.params[i]->strides());
      impl->set_storage_offset(offset);
      values[k].push_back(Tensor(std::move(impl)));
      (k == 0 ? s.tensors[i].param : *(void **)&s.tensors[i].grad) = all.data_ptr<at::BFloat16>() + offset;
      offset += (s.tensors[i].n + ON - 1) / ON * ON;
    }
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    rc = orca_adamw_moments(s.tensors.data(), (int32_t)s.tensors.size(), stream_of(work));
  }
  if (rc != ORCA_OK) return raise(rc);
  PyObject *both = PyTuple_New(2);
  for (int i = 0; both != nullptr && i < 2; ++i) {
    PyObject *list = PyList_New((Py_ssize_t)values[i].size());
    PyTuple_SET_ITEM(both, i, list);
    if (list == nullptr) {
      Py_DECREF(both);
      return nullptr;
    }
    for (size_t j = 0; j < values[i].size(); ++j) PyList_SET_ITEM(list, (Py_ssize_t)j, THPVariable_Wrap(std::move(values[i][j])));
  }
  return both;
  END_HANDLE_TH_ERRORS
}

}  // namespace orca_torch
