// adapters_binding.cpp — the adapter operators (gsdf_adapters/gsdf_adapters.h) for gs_sdf_amd.adapters.
#include <torch/extension.h>

#include "gsdf_adapters/gsdf_adapters.h"

namespace py = pybind11;

namespace {
uint64_t number(const py::handle &h, const char *name) {
  PyObject *i = PyNumber_Index(h.ptr());
  const unsigned long long v = i != nullptr ? PyLong_AsUnsignedLongLong(i) : 0;
  Py_XDECREF(i);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK(false, name, ": expected a whole number in [0, 2^64)");
  }
  return v;
}
gsdf_adapters::Offset offset_of(const py::handle &h) {
  gsdf_adapters::Offset o;
  if (THPVariable_Check(h.ptr())) o.word = THPVariable_Unpack(h.ptr());
  else o.number = number(h, "offset");
  return o;
}
}  // namespace

PYBIND11_MODULE(_gsdf_adapters, m) {
  typedef const torch::Tensor &T;
  typedef const std::optional<torch::Tensor> &O;
  m.def("lowrank_adapt", [](T x, T a, T b, T ids, O scales, O base, double p, py::handle seed, py::handle offset) {
    return gsdf_adapters::lowrank_adapt(x, a, b, ids, scales, base, p, number(seed, "seed"), offset_of(offset));
  });
  m.def("lowrank_adapt_", &gsdf_adapters::lowrank_adapt_);
  m.def("dropout", [](T x, double p, py::handle seed, py::handle offset, O residual) {
    return gsdf_adapters::dropout(x, p, number(seed, "seed"), offset_of(offset), residual);
  });
  m.def("router_balance", &gsdf_adapters::router_balance);
}
