// Compiled front of the packed-request operators: the calls of kernels.py for
// tensors that need no conversion, without the cost of checking and converting
// them in Python (20 to 25 us of host time a call, more than the kernels take
// for single tokens).  Each function returns None for anything else -- other
// layouts, types, devices, or arguments that are wrong -- and kernels.py then
// goes its own way, which converts, or raises with a message.  Nothing is kept
// between calls but the addresses of the devices' error words.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>

#include "../../include/bsa.h"

// What _native.py compares with the running torch before it loads this file.
extern "C" __attribute__((used, visibility("default"))) const char bsa_binding_torch[] =
    "bsa-binding-torch=" BSA_TORCH_VERSION;

namespace {

constexpr int kDevices = 64;
int32_t* g_err_words[kDevices] = {};

// The entry points, from the library that _native.py has loaded (bind).
decltype(&::bsa_last_error) last_error;
decltype(&::bsa_residual_norm) norm_entry;
decltype(&::bsa_lora_add_workspace_bytes) lora_bytes;
decltype(&::bsa_lora_add) lora_entry;
decltype(&::bsa_packed_attention_workspace_bytes) attention_bytes;
decltype(&::bsa_packed_attention) attention_entry;

// A tensor argument: null for None, `bad` for anything else that is no tensor
// on the CUDA device `device` (-1: not known yet, then set).
struct Arg {
  const at::Tensor* t = nullptr;
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  void* data() const { return t != nullptr ? t->data_ptr() : nullptr; }
};

bool take(PyObject* o, int& device, Arg& out) {
  out.t = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_conj() || t.is_neg() || t.requires_grad())
    return false;
  const int d = t.get_device();
  if (device < 0) device = d;
  if (d != device) return false;
  out.t = &t;
  return true;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? BSA_F32 : t == at::kBFloat16 ? BSA_BF16 : t == at::kHalf ? BSA_F16 : -1;
}

bool contiguous_i32(const Arg& a) {
  return a->dim() == 1 && a->scalar_type() == at::kInt && a->is_contiguous();
}

// The device is the current one, with an error word.
bool ready(int device) {
  return norm_entry != nullptr && device >= 0 && device < kDevices && g_err_words[device] != nullptr &&
         c10::cuda::current_device() == device;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

PyObject* failed(const char* name, int rc) {
  PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, last_error());
  return nullptr;
}

template <typename Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// residual_norm(x, y, gate, shift, scale, weight, bias, post_weight, post_bias,
//               row_starts, norm, post_norm, eps, normed_code or -1)
PyObject* residual_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 14) Py_RETURN_NONE;
    int device = -1;
    Arg a[10];
    for (int i = 0; i < 10; ++i)
      if (!take(args[i], device, a[i])) Py_RETURN_NONE;
    const Arg &x = a[0], &y = a[1], &starts = a[9];
    const long norm = PyLong_AsLong(args[10]), post = PyLong_AsLong(args[11]);
    const double eps = PyFloat_AsDouble(args[12]);
    long normed_code = PyLong_AsLong(args[13]);
    if (PyErr_Occurred()) return nullptr;
    if (normed_code < -1 || !x || !ready(device) || x->dim() != 2 || x->stride(1) != 1 || x->numel() == 0) Py_RETURN_NONE;
    const int64_t rows = x->size(0), width = x->size(1);
    const int xc = dtype_code(x->scalar_type());
    if (xc < 0) Py_RETURN_NONE;
    if (y) {
      if (y->dim() != 2 || y->sizes() != x->sizes() || y->stride(1) != 1) Py_RETURN_NONE;
      if (normed_code < 0) normed_code = dtype_code(y->scalar_type());
      if (dtype_code(y->scalar_type()) != normed_code) Py_RETURN_NONE;
    } else {
      if (normed_code < 0) normed_code = xc;
      if (a[2] || post != BSA_NORM_NONE) Py_RETURN_NONE;
    }
    if (normed_code < 0 || (xc != BSA_F32 && normed_code != xc)) Py_RETURN_NONE;
    int64_t requests = 0;
    if (starts) {
      if (!contiguous_i32(starts) || starts->size(0) < 2) Py_RETURN_NONE;
      requests = starts->size(0) - 1;
    }
    int mods = -1;
    for (int i = 2; i < 5; ++i) {
      if (!a[i]) continue;
      const int code = dtype_code(a[i]->scalar_type());
      if (a[i]->dim() != 2 || a[i]->size(1) != width || a[i]->stride(1) != 1 || code < 0 ||
          (mods >= 0 && code != mods))
        Py_RETURN_NONE;
      if (requests == 0) requests = a[i]->size(0);
      if (a[i]->size(0) != requests) Py_RETURN_NONE;
      mods = code;
    }
    if (requests == 0) requests = 1;
    if (!starts && requests != 1 && requests != rows) Py_RETURN_NONE;
    if (requests > INT32_MAX) Py_RETURN_NONE;
    int codes[2] = {-1, -1};    // affine, post
    for (int i = 5; i < 9; ++i) {
      if (!a[i]) continue;
      int& code = codes[(i - 5) / 2];
      const int c = dtype_code(a[i]->scalar_type());
      if (a[i]->dim() != 1 || a[i]->size(0) != width || !a[i]->is_contiguous() || c < 0 ||
          (code >= 0 && c != code))
        Py_RETURN_NONE;
      code = c;
    }
    if (post == BSA_NORM_NONE && (a[7] || a[8])) Py_RETURN_NONE;
    at::Tensor residual;
    if (y) residual = at::empty({rows, width}, x->options());
    const at::ScalarType nt =
        normed_code == BSA_F32 ? at::kFloat : normed_code == BSA_BF16 ? at::kBFloat16 : at::kHalf;
    at::Tensor normed = at::empty({rows, width}, x->options().dtype(nt));
    const int rc = norm_entry(
        x.data(), xc, x->stride(0), y.data(), static_cast<int32_t>(normed_code),
        y ? y->stride(0) : 0, rows, static_cast<int32_t>(width),
        static_cast<const int32_t*>(starts.data()), static_cast<int32_t>(requests), a[2].data(),
        a[2] ? a[2]->stride(0) : 0, a[3].data(), a[3] ? a[3]->stride(0) : 0, a[4].data(),
        a[4] ? a[4]->stride(0) : 0, mods < 0 ? 0 : mods, a[5].data(), a[6].data(),
        codes[0] < 0 ? 0 : codes[0], a[7].data(), a[8].data(), codes[1] < 0 ? 0 : codes[1],
        static_cast<int32_t>(norm), static_cast<int32_t>(post), static_cast<float>(eps),
        y ? residual.data_ptr() : nullptr, normed.data_ptr(), g_err_words[device], stream_of(device));
    if (rc != BSA_OK) return failed("bsa_residual_norm", rc);
    PyObject* first = args[0];
    if (y) first = THPVariable_Wrap(std::move(residual)); else Py_INCREF(first);
    PyObject* second = THPVariable_Wrap(std::move(normed));
    PyObject* pair = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
  });
}

bool rows_8(const Arg& t) {
  return t->dim() == 2 && t->stride(1) == 1 && t->stride(0) % 8 == 0 && t->stride(0) >= t->size(1) &&
         reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
}

// lora_add(y, x, lora_a, lora_b, row_starts, adapters, scales, out)
PyObject* lora_add(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 8) Py_RETURN_NONE;
    int device = -1;
    Arg a[8];
    for (int i = 0; i < 8; ++i)
      if (!take(args[i], device, a[i])) Py_RETURN_NONE;
    const Arg &y = a[0], &x = a[1], &la = a[2], &lb = a[3], &starts = a[4], &ids = a[5], &scales = a[6],
              &out = a[7];
    if (!y || !x || !la || !lb || !starts || !ids || !ready(device)) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i)
      if (a[i]->scalar_type() != at::kBFloat16) Py_RETURN_NONE;
    if (!rows_8(y) || !rows_8(x) || y->size(0) != x->size(0) || y->numel() == 0 || x->numel() == 0)
      Py_RETURN_NONE;
    const int64_t rows = y->size(0), cols = y->size(1), k = x->size(1);
    if (la->dim() != 3 || !la->is_contiguous() || la->size(2) != k || lb->dim() != 3 ||
        !lb->is_contiguous() || reinterpret_cast<uintptr_t>(la->data_ptr()) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(lb->data_ptr()) % 16 != 0)
      Py_RETURN_NONE;
    const int64_t count = la->size(0), rank = la->size(1);
    if (lb->size(0) != count || lb->size(1) != cols || lb->size(2) != rank || count > INT32_MAX ||
        cols > INT32_MAX || k > INT32_MAX)
      Py_RETURN_NONE;
    if (!contiguous_i32(starts) || !contiguous_i32(ids) || starts->size(0) != ids->size(0) + 1 ||
        ids->size(0) == 0 || ids->size(0) > INT32_MAX)
      Py_RETURN_NONE;
    if (scales && (scales->scalar_type() != at::kFloat || scales->dim() != 1 || scales->size(0) != count ||
                   !scales->is_contiguous()))
      Py_RETURN_NONE;
    if (out && (out->scalar_type() != at::kBFloat16 || out->sizes() != y->sizes() || !rows_8(out)))
      Py_RETURN_NONE;
    at::Tensor fresh;
    if (!out) fresh = at::empty({rows, cols}, y->options());
    const at::Tensor& dst = out ? *out.t : fresh;
    const int64_t bytes = lora_bytes(rows, static_cast<int32_t>(ids->size(0)),
                                                       static_cast<int32_t>(k), static_cast<int32_t>(rank));
    at::Tensor work = at::empty({bytes}, y->options().dtype(at::kByte));
    const int rc = lora_entry(
        y.data(), y->stride(0), x.data(), x->stride(0), la.data(), lb.data(),
        static_cast<const float*>(scales.data()), static_cast<const int32_t*>(starts.data()),
        static_cast<const int32_t*>(ids.data()), rows, static_cast<int32_t>(ids->size(0)),
        static_cast<int32_t>(count), static_cast<int32_t>(k), static_cast<int32_t>(cols),
        static_cast<int32_t>(rank), work.data_ptr(), bytes, dst.data_ptr(), dst.stride(0),
        g_err_words[device], stream_of(device));
    if (rc != BSA_OK) return failed("bsa_lora_add", rc);
    if (out) {
      Py_INCREF(args[7]);
      return args[7];
    }
    return THPVariable_Wrap(std::move(fresh));
  });
}

bool strided_heads(const Arg& t) {
  return t->dim() == 3 && t->scalar_type() == at::kBFloat16 && t->size(2) == 128 && t->stride(2) == 1 &&
         t->stride(0) % 8 == 0 && t->stride(1) % 8 == 0 && t->stride(0) >= 128 &&
         (t->size(1) == 1 || (t->stride(1) >= 128 && t->stride(0) >= t->stride(1))) &&
         reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
}

// packed_attention(q, k, v, q_starts, k_starts, causal, scale)
PyObject* packed_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) Py_RETURN_NONE;
    int device = -1;
    Arg a[5];
    for (int i = 0; i < 5; ++i)
      if (!take(args[i], device, a[i])) Py_RETURN_NONE;
    const Arg &q = a[0], &k = a[1], &v = a[2], &qs = a[3];
    if (!q || !k || !v || !qs || !ready(device)) Py_RETURN_NONE;
    const Arg& ks = a[4] ? a[4] : a[3];
    const int causal = PyObject_IsTrue(args[5]);
    const double scale = PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) return nullptr;
    if (!strided_heads(q) || !strided_heads(k) || !strided_heads(v) || k->sizes() != v->sizes() ||
        q->numel() == 0 || k->numel() == 0)
      Py_RETURN_NONE;
    if (!contiguous_i32(qs) || !contiguous_i32(ks) || qs->size(0) != ks->size(0) || qs->size(0) < 2 ||
        qs->size(0) > INT32_MAX || (!a[4] && q->size(0) != k->size(0)))
      Py_RETURN_NONE;
    const int64_t tq = q->size(0), tk = k->size(0), heads = q->size(1), kv = k->size(1);
    if (heads % kv != 0 || heads > INT32_MAX) Py_RETURN_NONE;
    const int32_t requests = static_cast<int32_t>(qs->size(0) - 1);
    at::Tensor out = at::empty({tq, heads, 128}, q->options());
    const int64_t bytes = attention_bytes(
        tq, tk, requests, static_cast<int32_t>(heads), static_cast<int32_t>(kv));
    at::Tensor work;
    if (bytes > 0) work = at::empty({bytes}, q->options().dtype(at::kByte));
    const int rc = attention_entry(
        q.data(), q->stride(0), q->stride(1), k.data(), k->stride(0), k->stride(1), v.data(),
        v->stride(0), v->stride(1), static_cast<const int32_t*>(qs.data()),
        static_cast<const int32_t*>(ks.data()), tq, tk, requests, static_cast<int32_t>(heads),
        static_cast<int32_t>(kv), 128, causal, static_cast<float>(scale),
        bytes > 0 ? work.data_ptr() : nullptr, bytes, out.data_ptr(), g_err_words[device],
        stream_of(device));
    if (rc != BSA_OK) return failed("bsa_packed_attention", rc);
    return THPVariable_Wrap(std::move(out));
  });
}

// set_err_word(device, address)
PyObject* set_err_word(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "set_err_word takes a device and an address");
    return nullptr;
  }
  const long device = PyLong_AsLong(args[0]);
  void* address = PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (device < 0 || device >= kDevices) {
    PyErr_SetString(PyExc_ValueError, "device out of range");
    return nullptr;
  }
  g_err_words[device] = static_cast<int32_t*>(address);
  Py_RETURN_NONE;
}

// bind(addresses of the six entry points above, in that order)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* at[6];
  for (Py_ssize_t i = 0; i < 6 && n == 6; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  if (n != 6 || PyErr_Occurred()) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
    return nullptr;
  }
  last_error = reinterpret_cast<decltype(last_error)>(at[0]);
  norm_entry = reinterpret_cast<decltype(norm_entry)>(at[1]);
  lora_bytes = reinterpret_cast<decltype(lora_bytes)>(at[2]);
  lora_entry = reinterpret_cast<decltype(lora_entry)>(at[3]);
  attention_bytes = reinterpret_cast<decltype(attention_bytes)>(at[4]);
  attention_entry = reinterpret_cast<decltype(attention_entry)>(at[5]);
  Py_RETURN_NONE;
}

#define BSA_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {BSA_METHOD(residual_norm), BSA_METHOD(lora_add), BSA_METHOD(packed_attention),
                         BSA_METHOD(set_err_word), BSA_METHOD(bind), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr,
                      nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
