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

// "torch V python X.Y": what this library was compiled against, and the only ones it may be loaded beside.
extern "C" const char* nr_built_for() { return NR_BUILT_FOR; }

// ptr, numel [len(list)], dtype [len(list)] (NR_DTYPE_*) <- the list's.  Returns the one device that they are on; or kNotTensors;
// kType: one is not fp32 / bf16 / fp16; kTracked: autograd follows one, backwards or forwards; kDevice: not all on one GPU; kLayout:
// one is not contiguous, or holds its values negated (its address is not taken).
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
      if (t.layout() != at::kStrided || !t.is_contiguous() || t.is_neg()) dense = false;
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

namespace {
struct Range {
  uint64_t from, to;
  bool operator<(const Range& o) const { return from < o.from; }
};
Range range_of(const int64_t* ptr, const int64_t* numel, const int32_t* dtype, int64_t i) {
  const uint64_t from = (uint64_t)ptr[i];
  return {from, from + (uint64_t)numel[i] * (dtype[i] == 0 ? 4 : 2)};
}
enum { kApart = 0, kWrittenTwice = 1, kWrittenAndRead = 2 };
}  // namespace

// Whether writing dst[0 .. n) while src[0 .. n) is read depends on who comes first: kWrittenTwice if two of dst share memory,
// kWrittenAndRead if one of dst shares memory with one of src and is not that one itself, with its type, at the same place of the
// list (in place: every element is read and written by one thread).  Empty tensors share nothing.
extern "C" int nr_shared_memory(const int64_t* src, const int32_t* src_dtype, const int64_t* dst, const int32_t* dst_dtype, const int64_t* numel,
                                int64_t n) {
  try {
    std::vector<Range> out;
    out.reserve((size_t)n);
    uint64_t low = UINT64_MAX, high = 0;  // (of src, without what is in place)
    for (int64_t i = 0; i < n; ++i) {
      if (numel[i] <= 0) continue;
      out.push_back(range_of(dst, numel, dst_dtype, i));
      if (src[i] == dst[i] && src_dtype[i] == dst_dtype[i]) continue;
      const Range r = range_of(src, numel, src_dtype, i);
      low = std::min(low, r.from);
      high = std::max(high, r.to);
    }
    if (out.empty()) return kApart;
    if (!std::is_sorted(out.begin(), out.end())) std::sort(out.begin(), out.end());
    for (size_t k = 1; k < out.size(); ++k)
      if (out[k].from < out[k - 1].to) return kWrittenTwice;
    if (high <= out.front().from || low >= out.back().to) return kApart;
    for (int64_t i = 0; i < n; ++i) {  // (the ranges of out are apart, so their ends ascend too: the first that ends behind r's start)
      if (numel[i] <= 0 || (src[i] == dst[i] && src_dtype[i] == dst_dtype[i])) continue;
      const Range r = range_of(src, numel, src_dtype, i);
      if (r.to <= out.front().from || r.from >= out.back().to) continue;  // (all of them beside a bucket)
      const auto at = std::upper_bound(out.begin(), out.end(), r.from, [](uint64_t a, const Range& o) { return a < o.to; });
      if (at != out.end() && at->from < r.to) return kWrittenAndRead;
    }
    return kApart;
  } catch (...) {
    return kFailed;
  }
}

// All that clipping asks of its two lists (or of one, in place), in one call: block <- [address n | elements n | place's address n | type n
// (int32) | place's type n (int32)].  Returns the device and marks the places as written if nothing stands against taking the lists as
// they are; else kNotTensors, without a mark: the caller finds out what with the functions above.
extern "C" int nr_clip_lists(PyObject* grads, PyObject* outs, int64_t* block) {
  try {
    const int64_t n = (int64_t)PyList_GET_SIZE(grads);
    if ((int64_t)PyList_GET_SIZE(outs) != n) return kNotTensors;
    int64_t *numel = block + n, *dst = block + 2 * n;
    int32_t *type = reinterpret_cast<int32_t*>(block + 3 * n), *dst_type = type + n;
    const int device = nr_tensor_list(grads, block, numel, type);
    if (device < 0) return kNotTensors;
    if (outs == grads) {
      std::copy(block, block + n, dst);
      std::copy(type, type + n, dst_type);
    } else {
      std::vector<int64_t> count((size_t)n);
      if (nr_tensor_list(outs, dst, count.data(), dst_type) != device || !std::equal(count.begin(), count.end(), numel)) return kNotTensors;
    }
    if (nr_shared_memory(block, type, dst, dst_type, numel, n) != kApart || nr_mark_written(outs) != 0) return kNotTensors;
    return device;
  } catch (...) {
    return kNotTensors;
  }
}
