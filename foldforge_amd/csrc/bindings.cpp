// CPython calls of the C-ABI (include/foldforge_amd.h): one function per entry point, its
// arguments converted by the entry point's own parameter types, so a call costs about a
// microsecond of host time where ctypes with 25 to 30 arguments takes eight. Checks stay in
// kernels.py; the one that runs over every parameter of every call (device, dtype, layout,
// shape) is params_ok below.
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <tuple>
#include <type_traits>
#include <utility>

#include "foldforge_amd.h"

namespace {

// A pointer argument: a tensor's data, an address as int (a stream) or None (NULL).
void* pointer_from(PyObject* o) {
  if (o == Py_None) return nullptr;
  if (THPVariable_Check(o)) return THPVariable_Unpack(o).data_ptr();
  return PyLong_AsVoidPtr(o);  // sets TypeError for anything else
}

template <typename T>
T from(PyObject* o) {
  if constexpr (std::is_pointer_v<T>) {
    return static_cast<T>(pointer_from(o));
  } else if constexpr (std::is_floating_point_v<T>) {
    return static_cast<T>(PyFloat_AsDouble(o));
  } else if constexpr (std::is_same_v<T, size_t>) {
    return PyLong_AsSize_t(o);
  } else {
    const long long v = PyLong_AsLongLong(o);
    if (static_cast<long long>(static_cast<T>(v)) != v && !PyErr_Occurred())
      PyErr_SetString(PyExc_OverflowError, "integer argument out of range");
    return static_cast<T>(v);
  }
}

template <auto Fn>
struct Call;
template <typename R, typename... A, R (*Fn)(A...)>
struct Call<Fn> {
  template <size_t... I>
  static PyObject* apply(PyObject* const* args, std::index_sequence<I...>) {
    const std::tuple<A...> v{from<A>(args[I])...};
    if (PyErr_Occurred()) return nullptr;
    R r;
    // launches may wait for queue space: other Python threads run meanwhile, as under ctypes
    Py_BEGIN_ALLOW_THREADS;
    r = std::apply(Fn, v);
    Py_END_ALLOW_THREADS;
    if constexpr (std::is_same_v<R, size_t>)
      return PyLong_FromSize_t(r);
    else
      return PyLong_FromLong(r);
  }
  static PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != static_cast<Py_ssize_t>(sizeof...(A)))
      return PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", (Py_ssize_t)sizeof...(A), n);
    return apply(args, std::index_sequence_for<A...>{});
    END_HANDLE_TH_ERRORS
  }
};

// params_ok(x, tensors, shapes): whether every tensor is a contiguous fp32 strided tensor on
// x's device of the given shape (False: the caller looks closer, and raises or copies).
PyObject* params_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !THPVariable_Check(args[0]) || !PyTuple_Check(args[1]) || !PyTuple_Check(args[2]) ||
      PyTuple_GET_SIZE(args[1]) != PyTuple_GET_SIZE(args[2]))
    return PyErr_Format(PyExc_TypeError, "params_ok(tensor, tuple of tensors, tuple of shapes)");
  const at::Device device = THPVariable_Unpack(args[0]).device();
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[1]); ++i) {
    PyObject* o = PyTuple_GET_ITEM(args[1], i);
    PyObject* shape = PyTuple_GET_ITEM(args[2], i);
    if (!THPVariable_Check(o) || !PyTuple_Check(shape)) Py_RETURN_FALSE;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kFloat || t.layout() != at::kStrided || t.device() != device ||
        t.dim() != PyTuple_GET_SIZE(shape) || !t.is_contiguous())
      Py_RETURN_FALSE;
    for (int64_t d = 0; d < t.dim(); ++d) {
      const long long want = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
      if (want == -1 && PyErr_Occurred()) return nullptr;
      if (t.size(d) != want) Py_RETURN_FALSE;
    }
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// activation_ok(codes, scales): whether they are an 8-bit activation: contiguous e4m3 codes [.., c], c > 0, and contiguous
// uint8 scales [.., ceil(c / 32)] on one device.
PyObject* activation_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) return PyErr_Format(PyExc_TypeError, "activation_ok(codes, scales)");
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_FALSE;
  const at::Tensor &c = THPVariable_Unpack(args[0]), &s = THPVariable_Unpack(args[1]);
  const int64_t dims = c.dim();
  if (c.scalar_type() != at::kFloat8_e4m3fn || s.scalar_type() != at::kByte || c.device() != s.device() || dims == 0 ||
      s.dim() != dims || !c.is_contiguous() || !s.is_contiguous() || c.size(dims - 1) <= 0 ||
      s.size(dims - 1) != (c.size(dims - 1) + 31) / 32)
    Py_RETURN_FALSE;
  for (int64_t d = 0; d + 1 < dims; ++d)
    if (c.size(d) != s.size(d)) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

bool plain(const at::Tensor& t, at::Device device) {
  return t.layout() == at::kStrided && t.device() == device && t.is_contiguous();
}
bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
// FFK_DTYPE_* of a bf16 / fp32 tensor, -1 for another.
int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? FFK_DTYPE_BF16 : t.scalar_type() == at::kFloat ? FFK_DTYPE_F32 : -1;
}

// adapted_sizes(x, weight, bias, down, up, scale, offsets, adapter): (rows, d_in, d_out, adapters, rank, requests, weight's
// dtype, adapters' dtype) where every tensor (bias and scale may be None) is as a projection with adapters takes it, None
// where not (the caller looks closer; sizes out of the kernels' range are left to it).
PyObject* adapted_sizes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "adapted_sizes: 8 tensors");
  for (int i = 0; i < 8; ++i)
    if (!THPVariable_Check(args[i]) && !((i == 2 || i == 5) && args[i] == Py_None)) Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]), &down = THPVariable_Unpack(args[3]),
                   &up = THPVariable_Unpack(args[4]), &offsets = THPVariable_Unpack(args[6]),
                   &adapter = THPVariable_Unpack(args[7]);
  const at::Device device = x.device();
  const int wc = dtype_code(w), ac = dtype_code(down);
  if (!x.is_cuda() || !plain(x, device) || x.scalar_type() != at::kBFloat16 || x.dim() == 0 || wc < 0 || ac < 0 ||
      dtype_code(up) != ac || w.dim() != 2 || down.dim() != 3 || up.dim() != 3 || !plain(w, device) ||
      !plain(down, device) || !plain(up, device) || !plain(offsets, device) || !plain(adapter, device) ||
      offsets.dim() != 1 || adapter.dim() != 1 || offsets.scalar_type() != at::kInt ||
      adapter.scalar_type() != at::kInt || offsets.numel() != adapter.numel() + 1)
    Py_RETURN_NONE;
  const int64_t d_out = w.size(0), d_in = w.size(1), adapters = down.size(0), rank = down.size(1);
  if (d_in <= 0 || d_out <= 0 || x.size(x.dim() - 1) != d_in || down.size(2) != d_in || up.size(0) != adapters ||
      up.size(1) != d_out || up.size(2) != rank || !aligned(x) || !aligned(w) || !aligned(down) || !aligned(up))
    Py_RETURN_NONE;
  const int64_t sizes[2] = {d_out, adapters};
  for (int i = 0; i < 2; ++i) {
    PyObject* o = args[i ? 5 : 2];
    if (o == Py_None) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != sizes[i] || !plain(t, device)) Py_RETURN_NONE;
  }
  return Py_BuildValue("(LLLLLLii)", (long long)(x.numel() / d_in), (long long)d_in, (long long)d_out, (long long)adapters,
                       (long long)rank, (long long)adapter.numel(), wc, ac);
  END_HANDLE_TH_ERRORS
}

// like(x, other): whether both are contiguous bf16 / fp32 tensors of one shape, type and GPU, with a last axis (other may be
// None).
PyObject* like(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) return PyErr_Format(PyExc_TypeError, "like(tensor, tensor or None)");
  if (!THPVariable_Check(args[0]) || !(args[1] == Py_None || THPVariable_Check(args[1]))) Py_RETURN_FALSE;
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  if (!x.is_cuda() || !plain(x, x.device()) || dtype_code(x) < 0 || x.dim() == 0 || x.size(x.dim() - 1) == 0)
    Py_RETURN_FALSE;
  if (args[1] != Py_None) {
    const at::Tensor& o = THPVariable_Unpack(args[1]);
    if (!plain(o, x.device()) || o.scalar_type() != x.scalar_type() || o.sizes() != x.sizes()) Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// empties(tensor, ((shape, kind), ...)): new tensors on the tensor's device, kind 0 bf16, 1 fp32, 2 uint8, 3 e4m3 (a
// call's outputs and workspace in one step: four torch.empty cost 5 us of the caller's time).
PyObject* empties(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  static constexpr at::ScalarType kKinds[] = {at::kBFloat16, at::kFloat, at::kByte, at::kFloat8_e4m3fn};
  if (n != 2 || !THPVariable_Check(args[0]) || !PyTuple_Check(args[1]))
    return PyErr_Format(PyExc_TypeError, "empties(tensor, tuple of (shape, kind))");
  const at::TensorOptions options = at::TensorOptions().device(THPVariable_Unpack(args[0]).device());
  const Py_ssize_t count = PyTuple_GET_SIZE(args[1]);
  PyObject* out = PyTuple_New(count);
  if (out == nullptr) return nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* spec = PyTuple_GET_ITEM(args[1], i);
    PyObject* shape = PyTuple_Check(spec) && PyTuple_GET_SIZE(spec) == 2 ? PyTuple_GET_ITEM(spec, 0) : nullptr;
    const long kind = shape ? PyLong_AsLong(PyTuple_GET_ITEM(spec, 1)) : -1;
    if (shape == nullptr || !PyTuple_Check(shape) || kind < 0 || kind > 3) {
      Py_DECREF(out);
      return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_TypeError, "empties: (shape, kind), kind 0 to 3");
    }
    c10::SmallVector<int64_t, 6> sizes;
    for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(shape); ++k) {
      sizes.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, k)));
      if (sizes.back() < 0) {
        Py_DECREF(out);
        return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "empties: negative size");
      }
    }
    try {
      PyTuple_SET_ITEM(out, i, THPVariable_Wrap(at::empty(sizes, options.dtype(kKinds[kind]))));
    } catch (...) {
      Py_DECREF(out);
      throw;
    }
  }
  return out;
  END_HANDLE_TH_ERRORS
}

#define FFK_CALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&Call<&name>::run)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"params_ok", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&params_ok)), METH_FASTCALL, nullptr},
    {"activation_ok", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&activation_ok)), METH_FASTCALL, nullptr},
    {"adapted_sizes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&adapted_sizes)), METH_FASTCALL, nullptr},
    {"like", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&like)), METH_FASTCALL, nullptr},
    {"empties", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&empties)), METH_FASTCALL, nullptr},
    FFK_CALL(ffk_layer_norm),
    FFK_CALL(ffk_layer_norm_linear),
    FFK_CALL(ffk_swiglu_ffn_workspace),
    FFK_CALL(ffk_swiglu_ffn),
    FFK_CALL(ffk_triangle_multiplication_workspace),
    FFK_CALL(ffk_triangle_multiplication),
    FFK_CALL(ffk_triangle_attention_workspace),
    FFK_CALL(ffk_triangle_attention),
    FFK_CALL(ffk_triangle_attention_transition_workspace),
    FFK_CALL(ffk_triangle_attention_transition),
    FFK_CALL(ffk_flash_attention_bias),
    FFK_CALL(ffk_transition_workspace),
    FFK_CALL(ffk_transition),
    FFK_CALL(ffk_attention_pair_bias_workspace),
    FFK_CALL(ffk_attention_pair_bias),
    FFK_CALL(ffk_msa_pair_weighted_averaging_workspace),
    FFK_CALL(ffk_msa_pair_weighted_averaging),
    FFK_CALL(ffk_outer_product_mean_workspace),
    FFK_CALL(ffk_outer_product_mean),
    FFK_CALL(ffk_outer_product_mean_grouped_workspace),
    FFK_CALL(ffk_outer_product_mean_grouped),
    FFK_CALL(ffk_quantize_activation),
    FFK_CALL(ffk_restore_activation),
    FFK_CALL(ffk_dropout_add),
    FFK_CALL(ffk_adapted_linear_workspace),
    FFK_CALL(ffk_adapted_linear),
    FFK_CALL(ffk_adapted_linear_backward_workspace),
    FFK_CALL(ffk_adapted_linear_backward),
    FFK_CALL(ffk_layer_norm_checkpoint),
    FFK_CALL(ffk_layer_norm_backward_workspace),
    FFK_CALL(ffk_layer_norm_backward),
    FFK_CALL(ffk_transition_backward_workspace),
    FFK_CALL(ffk_transition_backward),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_bindings", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bindings(void) { return PyModule_Create(&module_def); }
