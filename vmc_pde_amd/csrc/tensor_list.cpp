// Reads the addresses and sizes of many torch tensors at once, for the calls that take a table of them (vmcpde_tensor of include/vmcpde.h).
//
// Host code only, a library of its own beside libvmcpde.so, whose boundary stays free of torch types.  Python needs some 60 ns for every attribute
// of every tensor: with a dozen of them, clipping the 51 leaves of a flow's parameter vector cost five times the kernel's time.  Nothing is decided
// here: whatever is not plain (other types, devices, layouts) is handed back to the Python code, which handles or refuses it.
#include <torch/csrc/autograd/python_variable.h>

namespace {

// VMCPDE_F64 .. VMCPDE_BF16, or -1
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kDouble: return 0;
    case at::kFloat: return 1;
    case at::kHalf: return 2;
    case at::kBFloat16: return 3;
    default: return -1;
  }
}

}  // namespace

extern "C" {

// tensors: a list; out: a list of the same length, or None = the tensors themselves.  Fills table[4 * k ..] = { address, address to write to, elements,
// type code }, device[0] = the device's index.  Returns 1 where every entry is a dense tensor on one GPU, of a supported type, contiguous, not recorded by
// automatic differentiation (`recording`: that is to be asked of what is written to), and every out like its tensor; else 0 -- and 0 for whatever goes wrong.
int vmcpde_read_tensors(PyObject* tensors, PyObject* out, int recording, int64_t* table, int64_t capacity, int64_t* device) {
  try {
    if (!PyList_CheckExact(tensors)) return 0;
    const Py_ssize_t n = PyList_GET_SIZE(tensors);
    const bool own = out == Py_None;
    if (n == 0 || n > capacity || (!own && (!PyList_CheckExact(out) || PyList_GET_SIZE(out) != n))) return 0;
    for (Py_ssize_t k = 0; k < n; ++k) {
      PyObject* p = PyList_GET_ITEM(tensors, k);
      PyObject* q = own ? p : PyList_GET_ITEM(out, k);
      if (!THPVariable_Check(p) || !THPVariable_Check(q)) return 0;
      const at::Tensor& t = THPVariable_Unpack(p);
      const at::Tensor& o = THPVariable_Unpack(q);
      if (!t.defined() || !o.defined() || t.layout() != at::kStrided || o.layout() != at::kStrided || !t.is_cuda() || !o.is_cuda()) return 0;
      if (k == 0) device[0] = t.get_device();
      const int code = code_of(t.scalar_type());
      if (code < 0 || o.scalar_type() != t.scalar_type() || t.get_device() != device[0] || o.get_device() != device[0]) return 0;
      if (!t.is_contiguous() || !o.is_contiguous() || o.sizes() != t.sizes() || (recording && o.requires_grad())) return 0;
      table[4 * k] = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()));
      table[4 * k + 1] = static_cast<int64_t>(reinterpret_cast<uintptr_t>(o.data_ptr()));
      table[4 * k + 2] = t.numel();
      table[4 * k + 3] = code;
    }
    return 1;
  } catch (...) {
    return 0;
  }
}

}  // extern "C"
