// Addresses, sizes and types of lists of torch tensors, read in C++: a thousand gradients cost some
// 30 microseconds here and ten times that through Python attributes.  Built against the installed
// torch (prism_b200/build.py names the library after its version).
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "prism_bsa.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PRISM_BF16;
    case at::kHalf: return PRISM_FP16;
    case at::kFloat: return PRISM_FP32;
    default: return -1;
  }
}

// The tensor of a list item if it is a contiguous strided CUDA tensor, else NULL.
const at::Tensor* plain_tensor(PyObject* item) {
  if (!THPVariable_Check(item)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(item);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() ? &t : nullptr;
}

}  // namespace

// For n = the length of both lists (outs may be grads): table[0, n) the addresses of grads,
// [n, 2n) of outs, [2n, 3n) the element counts, codes[n] the prism_dtype_t.  Returns the index of
// the one device that all are on; -1 where an item is not a contiguous CUDA tensor of one of the
// three types, or an output has another type, size or device than its gradient (the caller looks
// closer).
extern "C" int prism_tensor_pairs(PyObject* grads, PyObject* outs, int64_t n, int64_t* table, int* codes) noexcept {
  try {
    if (!PyList_CheckExact(grads) || !PyList_CheckExact(outs) || PyList_GET_SIZE(grads) != n ||
        PyList_GET_SIZE(outs) != n || n < 1)
      return -1;
    int device = -1;
    for (int64_t i = 0; i < n; ++i) {
      const at::Tensor* g = plain_tensor(PyList_GET_ITEM(grads, i));
      const at::Tensor* o = outs == grads ? g : plain_tensor(PyList_GET_ITEM(outs, i));
      if (g == nullptr || o == nullptr) return -1;
      const int code = dtype_code(*g), at = g->get_device();
      if (i == 0) device = at;
      if (code < 0 || at != device || o->get_device() != device || o->scalar_type() != g->scalar_type() ||
          o->numel() != g->numel())
        return -1;
      table[i] = reinterpret_cast<int64_t>(g->data_ptr());
      table[n + i] = reinterpret_cast<int64_t>(o->data_ptr());
      table[2 * n + i] = g->numel();
      codes[i] = code;
    }
    return device;
  } catch (...) {
    PyErr_Clear();
    return -1;
  }
}
