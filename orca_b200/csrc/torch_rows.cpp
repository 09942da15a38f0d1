// The calls of rows by id (orca_packed_*, orca_rows_*) on PyTorch's tensors: the Python module orca_b200._rows.
//
// What the GPU does for a small batch takes less than what Python does around a call: checks of the tensors, outputs, workspaces,
// the stream (us a call, from Python / from here: one row attended over 19.7 / 6.4, a batch put and read back 23 / 12; a lookup of 600 ids
// with its gradient 112 / 53, of which 43 are torch.autograd.grad itself).  Ids and host data are prepared by orca_b200/packed.py
// and orca_b200/lookup.py, which are the only callers.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/orca_b200.h"

namespace {

using at::Tensor;
namespace ag = torch::autograd;

struct How {
  int64_t n_rows;
  double scale;
  int64_t padding;      // -1: none
  Tensor status;        // may be undefined
};

int type_of(const Tensor &t) {
  return t.scalar_type() == at::kFloat ? ORCA_F32 : t.scalar_type() == at::kBFloat16 ? ORCA_BF16 : ORCA_F16;
}
struct Failed : std::runtime_error {      // (a RuntimeError in a backward pass; calls make OrcaError of it, which is one)
  int rc;
  explicit Failed(int rc) : std::runtime_error("orca_b200 error " + std::to_string(rc) + ": " + orca_last_error()), rc(rc) {}
};
void check(int rc) {
  if (rc != ORCA_OK) throw Failed(rc);
}
PyObject *raise(int rc) {      // (what orca_b200._lib.check raises)
  pybind11::module_::import("orca_b200._lib").attr("check")(rc);
  return nullptr;
}
cudaStream_t stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()); }
int32_t *status_of(const How &how) { return how.status.defined() ? how.status.data_ptr<int32_t>() : nullptr; }

Tensor rows_of(const Tensor &table, const Tensor &ids, const How &how) {
  const c10::cuda::CUDAGuard guard(table.device());
  const int64_t width = table.size(1);
  const Tensor t = table.stride(1) == 1 && table.stride(0) >= width ? table : table.contiguous();
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(width);
  Tensor out = at::empty(shape, t.options());
  check(orca_rows_lookup(t.data_ptr(), t.size(0), std::max(t.stride(0), width), (int32_t)width, type_of(t), ids.data_ptr(),
                         ids.scalar_type() == at::kLong, ids.numel(), (float)how.scale, out.data_ptr(), status_of(how),
                         stream_of(table)));
  return out;
}

// grad_out [ids.shape, width]
Tensor table_grad(const Tensor &grad_out, const Tensor &ids, const How &how) {
  const c10::cuda::CUDAGuard guard(grad_out.device());
  const int64_t width = grad_out.size(-1), n = ids.numel();
  Tensor g = grad_out.dim() == 2 ? grad_out : grad_out.reshape({n, width});
  int64_t stride = n > 1 ? g.stride(0) : width;
  if (n > 0 && ((width > 1 && g.stride(1) != 1) || (stride > 0 && stride < width))) g = g.contiguous(), stride = width;
  Tensor grad = at::empty({how.n_rows, width}, g.options());
  if (width == 0) return grad;
  const int64_t need = orca_rows_grad_workspace_bytes(n, how.n_rows, (int32_t)width);
  Tensor ws;
  if (need > 0) ws = at::empty({need}, g.options().dtype(at::kByte));
  check(orca_rows_grad(g.data_ptr(), stride, (int32_t)width, type_of(g), ids.data_ptr(), ids.scalar_type() == at::kLong, n, how.n_rows,
                       (float)how.scale, how.padding, grad.data_ptr(), status_of(how), ws.defined() ? ws.data_ptr() : nullptr, need,
                       stream_of(g)));
  return grad;
}

// The same as a result that has no derivative: a tangent of grad_out is refused, and so is, by whoever asks for it, a backward pass.
Tensor final_grad(const Tensor &grad_out, const Tensor &ids, const How &how) {
  TORCH_CHECK_NOT_IMPLEMENTED(!grad_out._fw_grad(0).defined(), "the gradient of lookup_rows has no forward derivative");
  Tensor grad;
  {
    const at::NoGradGuard no_grad;
    grad = table_grad(grad_out, ids, how);
  }
  if (at::GradMode::is_enabled() && grad_out.requires_grad())
    ag::set_history(grad, std::make_shared<ag::Error>("the gradient of lookup_rows has no derivative", ag::collect_next_edges(grad_out)));
  return grad;
}

struct LookupBackward : public ag::Node {
  How how;
  ag::SavedVariable ids;
  bool released = false;

  ag::variable_list apply(ag::variable_list &&grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, ag::ERR_BACKWARD_TWICE);
    const Tensor &g = grads[0];
    if (!g.defined()) return {Tensor()};
    refuse_capture(g);
    return {final_grad(g, ids.unpack(), how)};
  }
  // The gradient goes on to a node that may belong to an older graph on another stream (the accumulator of a leaf lives as long as any
  // graph of it).  Its stream would be drawn into the capture, or cannot be, and the process ends: refused before.
  void refuse_capture(const Tensor &g) const {
    const auto next = next_edge(0).function->stream();
    if (!next || *next == c10::cuda::getCurrentCUDAStream(g.device().index()).unwrap()) return;
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
                "lookup_rows: this backward pass is captured in a graph while an older graph of the table lives; release that, or call lookup_grad");
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    ids.reset_data();
    released = true;
  }
  std::string name() const override { return "LookupRowsBackward"; }
};

// (table, ids, scale, padding or -1, status or None)
PyObject *lookup(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 5 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]), "lookup(table, ids, scale, padding, status)");
  const Tensor &table = THPVariable_Unpack(args[0]), &ids = THPVariable_Unpack(args[1]);
  How how = {table.size(0), PyFloat_AsDouble(args[2]), PyLong_AsLongLong(args[3]), {}};
  if (PyErr_Occurred()) return nullptr;
  if (args[4] != Py_None) how.status = THPVariable_Unpack(args[4]);
  Tensor out;
  try {
    const pybind11::gil_scoped_release no_gil;
    TORCH_CHECK_NOT_IMPLEMENTED(!table._fw_grad(0).defined(), "lookup_rows has no forward derivative");
    const bool differentiate = at::GradMode::is_enabled() && table.requires_grad();
    {
      const at::NoGradGuard no_grad;
      out = rows_of(table, ids, how);
    }
    if (differentiate) {
      auto node = std::make_shared<LookupBackward>();
      node->how = std::move(how);
      node->ids = ag::SavedVariable(ids, false);
      node->set_next_edges(ag::collect_next_edges(table));
      ag::set_history(out, node);
    }
  } catch (const Failed &e) {
    return raise(e.rc);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (grad_out, ids, rows, scale, padding or -1, status or None)
PyObject *grad(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 6 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]), "grad(grad_out, ids, rows, scale, padding, status)");
  const Tensor &g = THPVariable_Unpack(args[0]), &ids = THPVariable_Unpack(args[1]);
  How how = {PyLong_AsLongLong(args[2]), PyFloat_AsDouble(args[3]), PyLong_AsLongLong(args[4]), {}};
  if (PyErr_Occurred()) return nullptr;
  if (args[5] != Py_None) how.status = THPVariable_Unpack(args[5]);
  Tensor out;
  try {
    const pybind11::gil_scoped_release no_gil;
    out = final_grad(g, ids, how);
  } catch (const Failed &e) {
    return raise(e.rc);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- rows in 4 bits
const Tensor &tensor(PyObject *o, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " is a tensor");
  return THPVariable_Unpack(o);
}
// A tensor of `type` with these sizes (-1: any) beside `words`.
void expect(const Tensor &t, const Tensor &words, at::ScalarType type, at::IntArrayRef sizes, const char *name) {
  bool fits = t.device() == words.device() && t.scalar_type() == type && t.dim() == (int64_t)sizes.size();
  for (size_t i = 0; fits && i < sizes.size(); ++i) fits = sizes[i] < 0 || t.size((int64_t)i) == sizes[i];
  TORCH_CHECK_VALUE(fits, name, " is a tensor of ", type, ", sizes ", sizes, " (-1: any), on ", words.device(), "; not ", t.scalar_type(), " ",
                    t.sizes(), " on ", t.device());
}
void expect_whole(const Tensor &t, const char *name) {
  TORCH_CHECK_VALUE(t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0, name, " is contiguous and 16-byte aligned");
}
// Attention over packed rows has no derivatives: what asks for one would be cut off from the result.
void expect_constant(const Tensor &t, const char *name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined(), "attention over packed rows has no gradient: ",
                              name, " asks for one");
}

// What both forms of attention take: {words, status, qt, edges, time_w}, and what they return.
struct Attend {
  Tensor words, status, qt, edges, time_w, ctx, valid;
  int packed;
  Attend(PyObject *const *args)
      : words(tensor(args[0], "words")), status(tensor(args[1], "status")), qt(tensor(args[2], "qt")), edges(tensor(args[3], "edges")),
        time_w(tensor(args[4], "time_w")) {
    packed = edges.scalar_type() == at::kInt;
    expect(qt, words, at::kFloat, {-1, ORCA_QT_LD}, "qt");
    expect(time_w, words, at::kFloat, {ORCA_DIM}, "time_w");
    expect(edges, words, packed ? at::kInt : at::kFloat, {-1, packed ? ORCA_PACKED_WORDS : ORCA_DIM}, "edges: PackedRows, or it");
    expect_whole(qt, "qt"), expect_whole(time_w, "time_w"), expect_whole(edges, "edges");
    TORCH_CHECK_VALUE(edges.size(0) > 0, "edges without a row");
    expect_constant(qt, "qt"), expect_constant(time_w, "time_w"), expect_constant(edges, "edges");
  }
  int64_t rows() const { return qt.size(0); }
  void outputs() {
    ctx = at::empty({rows(), ORCA_QT_DIM}, at::TensorOptions().dtype(at::kFloat).device(words.device()));
    valid = at::empty({rows()}, at::TensorOptions().dtype(at::kByte).device(words.device()));
  }
  Tensor workspace(int64_t bytes) const { return bytes > 0 ? at::empty({bytes}, valid.options()) : Tensor(); }
  const uint32_t *table() const { return (const uint32_t *)words.data_ptr(); }
};
PyObject *pair(Tensor a, Tensor b) {
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
  PyObject *t = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x), Py_XDECREF(y);
  return t;
}

// (words, status, qt, edges, time_w, nbr, eid, delta)
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 8, "attend(words, status, qt, edges, time_w, nbr, eid, delta)");
  Attend a(args);
  const Tensor &nbr = tensor(args[5], "nbr"), &eid = tensor(args[6], "eid"), &delta = tensor(args[7], "delta");
  expect(nbr, a.words, at::kInt, {a.rows(), -1}, "nbr");
  expect(eid, a.words, at::kInt, nbr.sizes(), "eid");
  expect(delta, a.words, at::kFloat, nbr.sizes(), "delta");
  expect_constant(delta, "delta");
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::NoGradGuard no_grad;
    const c10::cuda::CUDAGuard guard(a.words.device());
    const Tensor nbr_ = nbr.contiguous(), eid_ = eid.contiguous(), delta_ = delta.contiguous();
    const int64_t k = nbr.size(1), need = orca_packed_attend_workspace_bytes((int32_t)a.rows(), k);
    a.outputs();
    const Tensor ws = a.workspace(need);
    rc = orca_packed_attend(a.qt.data_ptr<float>(), a.table(), a.words.size(0), a.edges.data_ptr(), a.edges.size(0), a.packed,
                            a.time_w.data_ptr<float>(), nbr_.data_ptr<int32_t>(), eid_.data_ptr<int32_t>(), delta_.data_ptr<float>(), k,
                            (int32_t)a.rows(), a.ctx.data_ptr<float>(), a.valid.data_ptr<uint8_t>(), a.status.data_ptr<int32_t>(),
                            ws.defined() ? ws.data_ptr() : nullptr, need, stream_of(a.words));
  }
  return rc == ORCA_OK ? pair(a.ctx, a.valid) : raise(rc);
  END_HANDLE_TH_ERRORS
}

// (words, status, qt, edges, time_w, indptr, adj_nbr, adj_eid, adj_ts, nodes of the graph, nodes, times, last or 0)
PyObject *attend_lists(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 13, "attend_lists(words, status, qt, edges, time_w, indptr, adj_nbr, adj_eid, adj_ts, n_nodes, nodes, times, last)");
  Attend a(args);
  const Tensor &indptr = tensor(args[5], "indptr"), &adj_nbr = tensor(args[6], "adj_nbr"), &adj_eid = tensor(args[7], "adj_eid"),
               &adj_ts = tensor(args[8], "adj_ts"), &nodes = tensor(args[10], "nodes"), &times = tensor(args[11], "timestamps");
  const int64_t n_nodes = PyLong_AsLongLong(args[9]), last = PyLong_AsLongLong(args[12]);
  if (PyErr_Occurred()) return nullptr;
  expect(indptr, a.words, at::kLong, {n_nodes + 1}, "the adjacency's indptr");
  expect(adj_nbr, a.words, at::kInt, {-1}, "the adjacency's adj_nbr");
  expect(adj_eid, a.words, at::kInt, adj_nbr.sizes(), "the adjacency's adj_eid");
  expect(adj_ts, a.words, at::kDouble, adj_nbr.sizes(), "the adjacency's adj_ts");
  // (the kernel reads the graph's arrays where they lie: a view with other strides has its values elsewhere, or beyond its storage)
  for (const Tensor *t : {&indptr, &adj_nbr, &adj_eid, &adj_ts}) TORCH_CHECK_VALUE(t->is_contiguous(), "the adjacency's arrays are contiguous");
  expect(nodes, a.words, at::kInt, {a.rows()}, "nodes");
  expect(times, a.words, at::kDouble, {a.rows()}, "timestamps");
  expect_constant(times, "timestamps"), expect_constant(adj_ts, "the adjacency's adj_ts");
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::NoGradGuard no_grad;
    const c10::cuda::CUDAGuard guard(a.words.device());
    const Tensor nodes_ = nodes.contiguous(), times_ = times.contiguous();
    const int64_t need = orca_packed_attend_last_workspace_bytes((int32_t)a.rows(), last);
    a.outputs();
    const Tensor ws = a.workspace(need);
    rc = orca_packed_attend_lists(a.qt.data_ptr<float>(), a.table(), a.words.size(0), a.edges.data_ptr(), a.edges.size(0), a.packed,
                                  a.time_w.data_ptr<float>(), indptr.data_ptr<int64_t>(), adj_nbr.data_ptr<int32_t>(),
                                  adj_eid.data_ptr<int32_t>(), adj_ts.data_ptr<double>(), n_nodes, nodes_.data_ptr<int32_t>(),
                                  times_.data_ptr<double>(), last, (int32_t)a.rows(), a.ctx.data_ptr<float>(), a.valid.data_ptr<uint8_t>(),
                                  a.status.data_ptr<int32_t>(), ws.defined() ? ws.data_ptr() : nullptr, need, stream_of(a.words));
  }
  return rc == ORCA_OK ? pair(a.ctx, a.valid) : raise(rc);
  END_HANDLE_TH_ERRORS
}

// (words, status, record or None, x, ids or None): without ids row i goes to row i
PyObject *push(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 5, "push(words, status, record, x, ids)");
  const Tensor &words = tensor(args[0], "words"), &status = tensor(args[1], "status"), &x = tensor(args[3], "x");
  const bool by_id = args[4] != Py_None;
  const int64_t n = x.size(0);
  if (by_id) TORCH_CHECK_VALUE(tensor(args[4], "ids").size(0) == n, n, " rows for ", tensor(args[4], "ids").size(0), " ids");
  if (n == 0) Py_RETURN_NONE;
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(words.device());
    rc = orca_packed_push((uint32_t *)words.data_ptr(), words.size(0), x.data_ptr(), type_of(x), std::max<int64_t>(x.stride(0), ORCA_DIM),
                          by_id ? THPVariable_Unpack(args[4]).data_ptr<int32_t>() : nullptr, (int32_t)n,
                          by_id ? THPVariable_Unpack(args[2]).data_ptr<int32_t>() : nullptr, status.data_ptr<int32_t>(), stream_of(words));
  }
  if (rc != ORCA_OK) return raise(rc);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (words, status, ids)
PyObject *pull(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 3, "pull(words, status, ids)");
  const Tensor &words = tensor(args[0], "words"), &status = tensor(args[1], "status"), &ids = tensor(args[2], "ids");
  Tensor out;
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(words.device());
    out = at::empty({ids.size(0), ORCA_DIM}, words.options().dtype(at::kFloat));
    rc = orca_packed_pull((const uint32_t *)words.data_ptr(), words.size(0), ids.data_ptr<int32_t>(), ids.size(0), out.data_ptr<float>(),
                          status.data_ptr<int32_t>(), stream_of(words));
  }
  return rc == ORCA_OK ? THPVariable_Wrap(std::move(out)) : raise(rc);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- the module
#define CALL(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(lookup), CALL(grad), CALL(attend), CALL(attend_lists), CALL(push), CALL(pull), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", nullptr, -1, methods};

}  // namespace

// (`made_for`: looked for in the file before it is loaded, orca_b200/build.py)
PyMODINIT_FUNC PyInit__rows() {
  PyObject *m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "made_for", ORCA_ROWS_MADE_FOR) != 0) Py_CLEAR(m);
  return m;
}
