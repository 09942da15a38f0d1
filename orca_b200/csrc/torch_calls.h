// What the sources of the module orca_b200._rows share: PyTorch's headers, errors, streams, and its calls.
#pragma once

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

namespace orca_torch {

using at::Tensor;
namespace ag = torch::autograd;

inline int type_of(const Tensor &t) {
  return t.scalar_type() == at::kFloat ? ORCA_F32 : t.scalar_type() == at::kBFloat16 ? ORCA_BF16 : ORCA_F16;
}
struct Failed : std::runtime_error {      // (a RuntimeError in a backward pass; calls make OrcaError of it, which is one)
  int rc;
  explicit Failed(int rc) : std::runtime_error("orca_b200 error " + std::to_string(rc) + ": " + orca_last_error()), rc(rc) {}
};
inline void check(int rc) {
  if (rc != ORCA_OK) throw Failed(rc);
}
inline PyObject *raise(int rc) {      // (what orca_b200._lib.check raises)
  pybind11::module_::import("orca_b200._lib").attr("check")(rc);
  return nullptr;
}
inline cudaStream_t stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()); }
inline const Tensor &tensor(PyObject *o, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " is a tensor");
  return THPVariable_Unpack(o);
}

// A gradient goes on to nodes that may belong to an older graph on another stream (the accumulator of a leaf lives as long as any
// graph of it).  Their stream would be drawn into a capture, or cannot be, and the process ends: refused before.
inline void refuse_capture(const ag::Node &node, const Tensor &g, const char *why) {
  const c10::Stream current = c10::cuda::getCurrentCUDAStream(g.device().index()).unwrap();
  for (size_t i = 0; i < node.num_outputs(); ++i) {
    const ag::Edge &edge = node.next_edge(i);
    if (!edge.is_valid() || !node.task_should_compute_output(i)) continue;
    const auto next = edge.function->stream();
    if (!next || *next == current) continue;
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, why);
    return;
  }
}

// torch_train.cpp
PyObject *norm(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *norm_grad(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *adamw(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *moments(PyObject *, PyObject *const *args, Py_ssize_t n_args);

}  // namespace orca_torch
