// orca_rows_lookup as an operation that PyTorch differentiates: the Python module orca_b200._rows.
//
// A lookup of a batch's ids takes the GPU 9 us, forward and backward; torch.autograd.Function alone takes the host 50, so that the
// node of the graph and what the two calls need around them (outputs, workspace, streams) are written here.  Arguments are checked
// by orca_b200/lookup.py, which is the only caller.
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
void check(int rc) {
  TORCH_CHECK(rc == ORCA_OK, "orca_b200 error ", rc, ": ", orca_last_error());
}
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
                         c10::cuda::getCurrentCUDAStream(table.device().index())));
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
                       c10::cuda::getCurrentCUDAStream(g.device().index())));
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
    Tensor grad;
    {
      const at::NoGradGuard no_grad;
      grad = table_grad(g, ids.unpack(), how);
    }
    // (a derivative of the gradient is refused by whoever asks for it)
    if (at::GradMode::is_enabled() && g.requires_grad())
      ag::set_history(grad, std::make_shared<ag::Error>("the gradient of lookup_rows has no derivative", ag::collect_next_edges(g)));
    return {grad};
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
  {
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
  {
    const pybind11::gil_scoped_release no_gil;
    const at::NoGradGuard no_grad;
    out = table_grad(g, ids, how);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"lookup", (PyCFunction)(void (*)())lookup, METH_FASTCALL, nullptr},
                         {"grad", (PyCFunction)(void (*)())grad, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__rows() { return PyModule_Create(&module); }
