// The layer operators as a Python module: tensors in, tensors out, one call into libvmcpde.so's C entry points.
//
// Host code only, a library of its own beside libvmcpde.so, whose boundary stays free of torch types.  A small call is bound by the host: Python's checks
// and attribute reads and torch's allocations through Python took 5 of the 8.6 us of a token's norm and 28 us of a small training step's two.
// Nothing is decided here: whatever is not plain (another device, layouts that need a copy, arguments that have to be refused) returns
// None before anything is launched, and vmc_pde_amd/layers.py, which can do all of it, handles or refuses the call.  What fails behind that is raised: made a second time,
// clipping in place would clip what is clipped already.
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>

#include <algorithm>
#include <cstring>
#include <vector>

#include "../../include/vmcpde.h"

namespace {

struct {
  decltype(&vmcpde_dense_workspace_bytes) dense_workspace;
  decltype(&vmcpde_dense) dense;
  decltype(&vmcpde_dense_backward) dense_backward;
  decltype(&vmcpde_layer_norm) layer_norm;
  decltype(&vmcpde_layer_norm_backward_workspace_bytes) layer_norm_workspace;
  decltype(&vmcpde_layer_norm_backward) layer_norm_backward;
  decltype(&vmcpde_global_norm_workspace_bytes) global_norm_workspace;
  decltype(&vmcpde_global_norm) global_norm;
} entry;

// vmc_pde_amd._native's exception and the library's message
PyObject* error_class = PyExc_RuntimeError;
decltype(&vmcpde_last_error) last_error;

struct NotPlain {};
struct Raised {};      // a Python exception is set
inline void need(bool plain) {
  if (!plain) throw NotPlain();
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kDouble: return VMCPDE_F64;
    case at::kFloat: return VMCPDE_F32;
    case at::kHalf: return VMCPDE_F16;
    case at::kBFloat16: return VMCPDE_BF16;
    default: throw NotPlain();
  }
}
at::ScalarType wide_of(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }
at::ScalarType slope_of(at::ScalarType t) { return t == at::kBFloat16 ? at::kHalf : t == at::kHalf ? at::kFloat : t; }

// The arguments of a call, in order.  The last two are the current device and its current stream.
struct Arguments {
  PyObject* const* given;
  const Py_ssize_t count;
  const int64_t device;
  const bool recording, tangents;      // tangents: whether a forward-mode level (there is only the first) is entered, outside of which no tensor has one
  Arguments(PyObject* const* a, Py_ssize_t n, Py_ssize_t wanted) : given(a), count(n), device(n == wanted ? PyLong_AsLongLong(a[n - 2]) : -1), recording(c10::GradMode::is_enabled()),
                                                                      tangents(torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr) {
    need(n == wanted && device >= 0);
  }
  void* stream() const { return PyLong_AsVoidPtr(given[count - 1]); }
  // a tensor on the device that automatic differentiation does not record, and without a forward-mode tangent
  const at::Tensor& tensor(int k) const { return checked(given[k], true); }
  const at::Tensor& checked(PyObject* p, bool written) const {
    need(THPVariable_Check(p));
    const at::Tensor& t = THPVariable_Unpack(p);
    need(t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !t.is_neg() && !(written && recording && t.requires_grad()) &&
         !(tangents && t._fw_grad(/* level */ 0).defined()));
    return t;
  }
  const at::Tensor* tensor_or_none(int k) const { return given[k] == Py_None ? nullptr : &tensor(k); }
  bool flag(int k) const {
    need(PyBool_Check(given[k]));
    return given[k] == Py_True;
  }
  double number(int k) const {
    need(PyFloat_CheckExact(given[k]) || PyLong_CheckExact(given[k]));
    const double v = PyFloat_AsDouble(given[k]);
    need(!(v == -1.0 && PyErr_Occurred()));
    return v;
  }
};

// row pitch of t as a matrix of `cols` columns
int64_t pitch_of(const at::Tensor& t, int64_t cols) {
  if (t.is_contiguous()) return cols;
  const auto sizes = t.sizes(), strides = t.strides();
  const int64_t last = t.dim() - 1;
  need(last >= 1 && (cols == 1 || strides[last] == 1));
  for (int64_t k = 0; k + 1 < last; ++k) need(strides[k] == strides[k + 1] * sizes[k + 1]);
  need(strides[last - 1] >= cols);
  return strides[last - 1];
}

struct Kernel { int64_t n_in, n_out, ld; int32_t transposed; };
Kernel layout_of(const at::Tensor& t) {
  need(t.dim() == 2);
  const int64_t n_in = t.size(0), n_out = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
  need(n_in >= 1 && n_out >= 1);
  if ((s1 == 1 || n_out == 1) && (s0 >= n_out || n_in == 1)) return {n_in, n_out, std::max(s0, n_out), 0};
  need((s0 == 1 || n_in == 1) && (s1 >= n_in || n_out == 1));
  return {n_in, n_out, std::max(s1, n_in), 1};
}

void vector_of(const at::Tensor& t, int64_t n) { need(t.dim() == 1 && t.size(0) == n && t.is_contiguous()); }

struct Workspace {
  at::Tensor held;
  void* p = nullptr;
  Workspace(int64_t bytes, const at::Tensor& like) {
    need(bytes >= 0);
    if (bytes) {
      held = at::empty({bytes}, like.options().dtype(at::kByte));
      p = held.data_ptr();
    }
  }
};

// One call into the library.  What it refuses (-1, with nothing launched) the Python code calls again and reports; other errors may have come behind a launch.
template <typename F>
void call(const char* name, F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  need(rc != -1);
  if (rc == 0) return;
  PyErr_Format(error_class, "%s failed (rc=%d): %s", name, rc, last_error ? last_error() : "");
  throw Raised();
}

// (behind the call: nothing may send it back to the Python code)
PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  try {
    return THPVariable_Wrap(t);
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(error_class, "a result could not be handed to Python");
    return nullptr;
  }
}
PyObject* wrap(const at::Tensor& a, const at::Tensor& b) { return Py_BuildValue("(NN)", wrap(a), wrap(b)); }
PyObject* wrap(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) { return Py_BuildValue("(NNN)", wrap(a), wrap(b), wrap(c)); }

template <typename F>
PyObject* plainly(F f) {
  try {
    return f();
  } catch (const Raised&) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (x, kernel, bias, activation's code, scale, residual, want_slope, device, stream)
PyObject* dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return plainly([&]() -> PyObject* {
    const Arguments in(args, n, 9);
    const at::Tensor &x = in.tensor(0), &kernel = in.tensor(1);
    const at::Tensor *bias = in.tensor_or_none(2), *residual = in.tensor_or_none(5);
    const Kernel w = layout_of(kernel);
    const auto dtype = x.scalar_type();
    vmcpde_dense_args a = {};
    a.dtype = code_of(dtype);
    a.activation = (int32_t)PyLong_AsLong(args[3]);
    a.kernel_t = w.transposed;
    need(x.dim() >= 1 && x.size(-1) == w.n_in && kernel.scalar_type() == dtype && a.activation >= VMCPDE_ACT_NONE && a.activation <= VMCPDE_ACT_SILU);
    auto shape = x.sizes().vec();
    shape.back() = w.n_out;
    a.rows = x.numel() / w.n_in;
    a.n_in = w.n_in;
    a.n_out = w.n_out;
    a.x = x.data_ptr();
    a.ldx = pitch_of(x, w.n_in);
    a.kernel = kernel.data_ptr();
    a.ldk = w.ld;
    if (bias) {
      vector_of(*bias, w.n_out);
      need(bias->scalar_type() == dtype);
      a.bias = bias->data_ptr();
    }
    if (residual) {
      need(residual->scalar_type() == dtype && residual->sizes() == at::IntArrayRef(shape));
      a.residual = residual->data_ptr();
      a.ldr = pitch_of(*residual, w.n_out);
    }
    a.scale = in.number(4);
    const bool want_slope = in.flag(6);
    const at::Tensor y = at::empty(shape, x.options());
    at::Tensor slope;
    a.y = y.data_ptr();
    a.ldy = w.n_out;
    if (want_slope && a.activation != VMCPDE_ACT_NONE) {
      slope = at::empty(shape, x.options().dtype(slope_of(dtype)));
      a.slope = slope.data_ptr();
    }
    const int64_t bytes = entry.dense_workspace(&a, 0);
    const Workspace space(bytes, x);
    void* stream = in.stream();
    call("vmcpde_dense", [&] { return entry.dense(&a, space.p, bytes, stream); });
    return want_slope ? wrap(y, slope) : wrap(y);
  });
}

// (dy, x, kernel, slope, scale, want_x, want_kernel, want_bias, device, stream)
PyObject* dense_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return plainly([&]() -> PyObject* {
    const Arguments in(args, n, 10);
    const at::Tensor &dy = in.tensor(0), &x = in.tensor(1), &kernel = in.tensor(2);
    const at::Tensor* slope = in.tensor_or_none(3);
    const Kernel w = layout_of(kernel);
    const auto dtype = dy.scalar_type();
    need(x.dim() >= 1 && x.size(-1) == w.n_in && x.scalar_type() == dtype && kernel.scalar_type() == dtype);
    auto shape = x.sizes().vec();
    shape.back() = w.n_out;
    need(dy.sizes() == at::IntArrayRef(shape));
    vmcpde_dense_args a = {};
    a.dtype = code_of(dtype);
    a.kernel_t = w.transposed;
    a.rows = x.numel() / w.n_in;
    a.n_in = w.n_in;
    a.n_out = w.n_out;
    a.x = x.data_ptr();
    a.ldx = pitch_of(x, w.n_in);
    a.kernel = kernel.data_ptr();
    a.ldk = w.ld;
    a.scale = in.number(4);
    if (slope) {
      need(slope->scalar_type() == slope_of(dtype) && slope->sizes() == at::IntArrayRef(shape) && slope->is_contiguous());
      a.slope = slope->data_ptr();
    }
    a.dy = dy.data_ptr();
    a.ldd = pitch_of(dy, w.n_out);
    const bool want_x = in.flag(5), want_kernel = in.flag(6), want_bias = in.flag(7);
    at::Tensor dx, dkernel, dbias;
    if (want_x) a.dx = (dx = at::empty(x.sizes(), x.options())).data_ptr();
    if (want_kernel) a.dkernel = (dkernel = at::empty({w.n_in, w.n_out}, x.options())).data_ptr();
    if (want_bias) a.dbias = (dbias = at::empty({w.n_out}, x.options())).data_ptr();
    const int64_t bytes = entry.dense_workspace(&a, 1);
    const Workspace space(bytes, x);
    void* stream = in.stream();
    call("vmcpde_dense_backward", [&] { return entry.dense_backward(&a, space.p, bytes, stream); });
    return wrap(dx, dkernel, dbias);
  });
}

// the type of a norm's weights beside elements of type `dtype`
at::ScalarType weights_of(const at::Tensor& t, at::ScalarType dtype, int64_t cols) {
  const auto type = t.scalar_type();
  need(type == dtype || (type == at::kFloat && (dtype == at::kHalf || dtype == at::kBFloat16)));
  vector_of(t, cols);
  return type;
}

// (x, weight, bias, eps, want_stats, device, stream)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return plainly([&]() -> PyObject* {
    const Arguments in(args, n, 7);
    const at::Tensor& x = in.tensor(0);
    const at::Tensor *weight = in.tensor_or_none(1), *bias = in.tensor_or_none(2);
    need(x.dim() >= 1 && x.size(-1) >= 1);
    const auto dtype = x.scalar_type();
    vmcpde_norm_args a = {};
    a.cols = x.size(-1);
    a.rows = x.numel() / a.cols;
    auto weights = dtype;
    if (weight) {
      weights = weights_of(*weight, dtype, a.cols);
      a.weight = weight->data_ptr();
    }
    if (bias) {
      const auto type = weights_of(*bias, dtype, a.cols);
      need(!weight || type == weights);
      weights = type;
      a.bias = bias->data_ptr();
    }
    a.dtype = code_of(dtype);
    a.weight_dtype = code_of(weights);
    a.x = x.data_ptr();
    a.ldx = pitch_of(x, a.cols);
    a.eps = in.number(3);
    const bool want_stats = in.flag(4);
    const at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor mean, rstd;
    a.y = y.data_ptr();
    a.ldy = a.cols;
    if (want_stats) {
      const auto leading = x.sizes().slice(0, x.dim() - 1);
      a.mean = (mean = at::empty(leading, x.options().dtype(wide_of(dtype)))).data_ptr();
      a.rstd = (rstd = at::empty(leading, x.options().dtype(wide_of(dtype)))).data_ptr();
      need(a.rows > 0);                       // (no rows, no addresses: the Python code's)
    }
    void* stream = in.stream();
    call("vmcpde_layer_norm", [&] { return entry.layer_norm(&a, stream); });
    return want_stats ? wrap(y, mean, rstd) : wrap(y);
  });
}

// (dy, x, mean, rstd, weight, want_x, want_weight, want_bias, device, stream); without a weight its gradient has x's type
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return plainly([&]() -> PyObject* {
    const Arguments in(args, n, 10);
    const at::Tensor &dy = in.tensor(0), &x = in.tensor(1), &mean = in.tensor(2), &rstd = in.tensor(3);
    const at::Tensor* weight = in.tensor_or_none(4);
    need(x.dim() >= 1 && x.size(-1) >= 1);
    const auto dtype = dy.scalar_type();
    const auto leading = x.sizes().slice(0, x.dim() - 1);
    need(x.scalar_type() == dtype && dy.sizes() == x.sizes());
    for (const at::Tensor* t : {&mean, &rstd}) need(t->scalar_type() == wide_of(dtype) && t->sizes() == leading && t->is_contiguous());
    vmcpde_norm_args a = {};
    a.cols = x.size(-1);
    a.rows = x.numel() / a.cols;
    auto weights = dtype;
    if (weight) {
      weights = weights_of(*weight, dtype, a.cols);
      a.weight = weight->data_ptr();
    }
    a.dtype = code_of(dtype);
    a.weight_dtype = code_of(weights);
    a.x = x.data_ptr();
    a.ldx = pitch_of(x, a.cols);
    a.mean = mean.data_ptr();
    a.rstd = rstd.data_ptr();
    a.dy = dy.data_ptr();
    a.ldd = pitch_of(dy, a.cols);
    const bool want_x = in.flag(5), want_weight = in.flag(6), want_bias = in.flag(7);
    at::Tensor dx, dweight, dbias;
    if (want_x) a.dx = (dx = at::empty(x.sizes(), x.options())).data_ptr();
    if (want_weight) a.dweight = (dweight = at::empty({a.cols}, x.options().dtype(weights))).data_ptr();
    if (want_bias) a.dbias = (dbias = at::empty({a.cols}, x.options().dtype(weights))).data_ptr();
    const int64_t bytes = want_weight || want_bias ? entry.layer_norm_workspace(&a) : 0;
    const Workspace space(bytes, x);
    void* stream = in.stream();
    call("vmcpde_layer_norm_backward", [&] { return entry.layer_norm_backward(&a, space.p, bytes, stream); });
    return wrap(dx, dweight, dbias);
  });
}

// (tensors, out, max_norm, device, stream): tensors a list; out a list of the same length, or None = the tensors themselves; max_norm None: the norm only
PyObject* global_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return plainly([&]() -> PyObject* {
    const Arguments in(args, n, 5);
    PyObject *tensors = args[0], *out = args[1];
    const bool clip = args[2] != Py_None, own = out == Py_None;
    need(PyList_CheckExact(tensors) && PyList_GET_SIZE(tensors) > 0 && (own || (PyList_CheckExact(out) && PyList_GET_SIZE(out) == PyList_GET_SIZE(tensors))));
    const Py_ssize_t count = PyList_GET_SIZE(tensors);
    need(count < (1 << 30));
    std::vector<vmcpde_tensor> table((size_t)count);
    at::TensorOptions options;
    for (Py_ssize_t k = 0; k < count; ++k) {
      const at::Tensor& t = in.checked(PyList_GET_ITEM(tensors, k), clip && own);
      const at::Tensor& o = own ? t : in.checked(PyList_GET_ITEM(out, k), clip);
      need(t.is_contiguous() && (own || (o.is_contiguous() && o.sizes() == t.sizes() && o.scalar_type() == t.scalar_type())));
      table[(size_t)k] = {t.data_ptr(), o.data_ptr(), t.numel(), code_of(t.scalar_type()), 0};
      if (k == 0) options = t.options();
    }
    const double max_norm = clip ? in.number(2) : 0.0;
    const at::Tensor norm = at::empty({}, options.dtype(at::kDouble));
    const int64_t bytes = entry.global_norm_workspace(table.data(), (int32_t)count);
    const Workspace space(bytes, norm);
    void* stream = in.stream();
    double* to = static_cast<double*>(norm.data_ptr());
    call("vmcpde_global_norm", [&] { return entry.global_norm(table.data(), (int32_t)count, clip, max_norm, to, space.p, bytes, stream); });
    if (clip) {                               // written in place: a recorded graph that saved one of these has to see it
      PyObject* const written = own ? tensors : out;
      for (Py_ssize_t k = 0; k < PyList_GET_SIZE(written); ++k)      // (looked at anew: another thread may have changed the list meanwhile)
        if (THPVariable_Check(PyList_GET_ITEM(written, k))) {
          const at::Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(written, k));
          if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
    }
    return wrap(norm);
  });
}

// the addresses of the eight entry points, in the order of `entry`
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t COUNT = sizeof(entry) / sizeof(void*);
  if (n != COUNT) {
    PyErr_SetString(PyExc_TypeError, "bind takes the addresses of the layer operators' entry points");
    return nullptr;
  }
  void* address[COUNT];
  for (Py_ssize_t k = 0; k < COUNT; ++k) {
    address[k] = PyLong_AsVoidPtr(args[k]);
    if (PyErr_Occurred()) return nullptr;
  }
  static_assert(sizeof(address) == sizeof(entry), "function addresses only");
  std::memcpy(&entry, address, sizeof(entry));
  Py_RETURN_NONE;
}

// (the exception class to raise, the address of vmcpde_last_error)
PyObject* raising(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* address = n == 2 && PyExceptionClass_Check(args[0]) ? PyLong_AsVoidPtr(args[1]) : nullptr;
  if (!address) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "raising takes an exception class and the address of vmcpde_last_error");
    return nullptr;
  }
  Py_INCREF(args[0]);      // (kept as long as the module, which is never unloaded)
  error_class = args[0];
  static_assert(sizeof(last_error) == sizeof(address), "a function's address");
  std::memcpy(&last_error, &address, sizeof(address));
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),       METHOD(raising),       METHOD(dense),       METHOD(dense_backward), METHOD(layer_norm), METHOD(layer_norm_backward),
                         METHOD(global_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "vmcpde_layer_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch and Python that this was compiled against; of any other only this may be asked
PyMODINIT_FUNC PyInit_vmcpde_layer_calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", VMCPDE_BUILT_FOR)) Py_CLEAR(m);
  return m;
}
