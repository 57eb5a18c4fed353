// Host side of the calls that take lists of tensors: checks a Python list and lays out its table
// (ganamd_tensor rows) in one pass.  From Python the same costs about 0.4 us a tensor and list,
// more than the kernels take for a thousand tensors; here some 20 ns.
//
// Called through ctypes.PyDLL (the GIL is held).  No exception leaves: every entry point catches.
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

namespace {

int code(at::ScalarType t) {         // GANAMD_F32, _BF16, _F16
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// One tensor of the list `name`: what is wrong with it, or nothing.
std::string look(PyObject* o, const char* name, int& device) {
  const std::string what(name);
  if (!THPVariable_Check(o)) return what + " are tensors; got " + Py_TYPE(o)->tp_name;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) return what + " are dense tensors";
  if (!t.is_cuda()) return what + " are on one GPU; got one on " + t.device().str();
  if (device < 0) device = t.get_device();
  if (t.get_device() != device) return what + " are on one GPU; got several";
  if (code(t.scalar_type()) < 0) return what + " are float32, bfloat16 or float16; got " + toString(t.scalar_type());
  if (!t.is_non_overlapping_and_dense()) return what + " are stored densely, each element once";
  return "";
}

std::string table(PyObject* ts, PyObject* outs, long n, int64_t* rows) {
  int device = -1;
  for (long i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(ts, i);
    std::string bad = look(o, "gradients", device);
    if (!bad.empty()) return bad;
    const at::Tensor& t = THPVariable_Unpack(o);
    const at::Tensor* d = &t;
    if (outs != ts) {
      PyObject* q = PyList_GET_ITEM(outs, i);
      bad = look(q, "outputs", device);
      if (!bad.empty()) return bad;
      d = &THPVariable_Unpack(q);
      if (d->numel() != t.numel()) return "an output has another number of elements than its gradient";
      if (!(t.is_contiguous() && d->is_contiguous()) && t.strides() != d->strides())
        return "a gradient that is not contiguous needs an output of its own strides";
      if (code(d->scalar_type()) != code(t.scalar_type()) && d->scalar_type() != at::kFloat)
        return "an output is of its gradient's type or float32";
    }
    rows[4 * i] = reinterpret_cast<int64_t>(t.const_data_ptr());
    rows[4 * i + 1] = reinterpret_cast<int64_t>(d->const_data_ptr());
    rows[4 * i + 2] = t.numel();
    rows[4 * i + 3] = code(t.scalar_type()) | static_cast<int64_t>(code(d->scalar_type())) << 32;
  }
  return "";
}

}  // namespace

extern "C" {

// tensors, outs: Python lists (outs may be tensors itself: no outputs of their own); rows: room for
// len(tensors) ganamd_tensor.  Returns None, or a text that says why the list is refused.
PyObject* host_tensor_table(PyObject* tensors, PyObject* outs, int64_t* rows) {
  try {
    if (!PyList_Check(tensors) || !PyList_Check(outs)) return PyUnicode_FromString("lists of tensors are wanted");
    const long n = PyList_GET_SIZE(tensors);
    if (PyList_GET_SIZE(outs) != n)
      return PyUnicode_FromFormat("%ld gradients, %ld outputs", n, (long)PyList_GET_SIZE(outs));
    const std::string bad = table(tensors, outs, n, rows);
    if (bad.empty()) Py_RETURN_NONE;
    return PyUnicode_FromString(bad.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "host_tensor_table");
  }
  return nullptr;
}

// Whether any tensor of a list requires a gradient (1, 0; -1 with a Python error set).
int host_requires_grad(PyObject* tensors) {
  try {
    for (long i = 0; i < PyList_GET_SIZE(tensors); ++i)
      if (THPVariable_Unpack(PyList_GET_ITEM(tensors, i)).requires_grad()) return 1;
    return 0;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "host_requires_grad");
    return -1;
  }
}

}  // extern "C"
