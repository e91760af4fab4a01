// Addresses, sizes and types of a Python list of tensors (host code): what nr_grad_norm / nr_grad_scale take, read in one call.
// Asking every tensor for four things from Python costs a microsecond each, which for a few hundred gradients is more than the
// kernels take.  Called with the interpreter lock held (ctypes.PyDLL); nothing is thrown across the boundary.
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <vector>

namespace {
enum { kNotTensors = -1, kType = -2, kDevice = -3, kLayout = -4, kFailed = -5, kTracked = -6 };
}

// ptr, numel [len(list)], dtype [len(list)] (NR_DTYPE_*) <- the list's.  Returns the one device that they are on; or kNotTensors;
// kType: one is not fp32 / bf16 / fp16; kTracked: autograd follows one, backwards or forwards; kDevice: not all on one GPU; kLayout:
// one is not contiguous (its address is not taken).
extern "C" int nr_tensor_list(PyObject* list, int64_t* ptr, int64_t* numel, int32_t* dtype) {
  try {
    if (!PyList_Check(list)) return kNotTensors;
    int device = -1;
    bool dense = true;
    const bool grad_mode = c10::GradMode::is_enabled();
    const Py_ssize_t n = PyList_GET_SIZE(list);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      if (!THPVariable_Check(o)) return kNotTensors;
      const at::Tensor& t = THPVariable_Unpack(o);
      switch (t.scalar_type()) {
        case at::kFloat: dtype[i] = 0; break;
        case at::kBFloat16: dtype[i] = 1; break;
        case at::kHalf: dtype[i] = 2; break;
        default: return kType;
      }
      if ((grad_mode && t.requires_grad()) || t._fw_grad(0).defined()) return kTracked;
      if (!t.is_cuda() || (device >= 0 && t.get_device() != device)) return kDevice;
      device = (int)t.get_device();
      numel[i] = t.numel();
      if (t.layout() != at::kStrided || !t.is_contiguous()) dense = false;
      else ptr[i] = numel[i] > 0 ? reinterpret_cast<int64_t>(t.data_ptr()) : 0;
    }
    return dense ? device : kLayout;
  } catch (...) {
    return kFailed;
  }
}

// The list's tensors have been written through their addresses: autograd's version counters go up, as after any write in place, so
// that a backward pass that saved one of them raises.  (A tensor of inference mode has no counter.)
extern "C" int nr_mark_written(PyObject* list) {
  try {
    const Py_ssize_t n = PyList_GET_SIZE(list);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(list, i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    return 0;
  } catch (...) {
    return kFailed;
  }
}

// 1 if two of the non-empty tensors start at the same address.
extern "C" int nr_same_address(const int64_t* ptr, int64_t n) {
  try {
    std::vector<int64_t> p;
    p.reserve((size_t)n);
    for (int64_t i = 0; i < n; ++i)
      if (ptr[i] != 0) p.push_back(ptr[i]);
    std::sort(p.begin(), p.end());
    return std::adjacent_find(p.begin(), p.end()) != p.end() ? 1 : 0;
  } catch (...) {
    return kFailed;
  }
}
