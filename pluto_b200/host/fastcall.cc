// CPython binding of the C ABI for the per-call paths of pluto_b200.layers: one vectorcall function
// per entry point, arguments converted straight to the C types.  A ctypes call spends 1 to 5 us on
// the same (it grows with the number of arguments, and decode has 24); with launches at 3 to 4 us
// that is a large part of what a single-token call costs.
//
// Pointers come as integers (tensor.data_ptr()), None, or bytes objects (the cache descriptor that
// kv_cache() below packs).  The GIL is released around the call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstdio>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/pluto_b200.h"

namespace {

template <typename T>
bool convert(PyObject* o, T& value) {
  if constexpr (std::is_pointer_v<T>) {
    if (o == Py_None) {
      value = nullptr;
    } else if (PyBytes_Check(o)) {
      value = reinterpret_cast<T>(PyBytes_AS_STRING(o));
    } else {
      const unsigned long long bits = PyLong_AsUnsignedLongLong(o);
      if (bits == ~0ull && PyErr_Occurred()) return false;
      value = reinterpret_cast<T>(static_cast<uintptr_t>(bits));
    }
  } else if constexpr (std::is_floating_point_v<T>) {
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) return false;
    value = static_cast<T>(d);
  } else {
    const long long n = PyLong_AsLongLong(o);
    if (n == -1 && PyErr_Occurred()) return false;
    if constexpr (std::is_same_v<T, int>) {
      if (n < INT32_MIN || n > INT32_MAX) {
        PyErr_SetString(PyExc_OverflowError, "argument does not fit a C int");
        return false;
      }
    }
    value = static_cast<T>(n);
  }
  return true;
}

PyObject* to_python(int v) { return PyLong_FromLong(v); }
PyObject* to_python(size_t v) { return PyLong_FromSize_t(v); }

template <auto Function>
struct Entry;
template <typename R, typename... A, R (*Function)(A...)>
struct Entry<Function> {
  template <size_t... I>
  static PyObject* call(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<std::remove_const_t<A>...> values;
    if (!(convert(args[I], std::get<I>(values)) && ...)) return nullptr;
    R result;
    Py_BEGIN_ALLOW_THREADS
    result = Function(std::get<I>(values)...);
    Py_END_ALLOW_THREADS
    return to_python(result);
  }
  static PyObject* fastcall(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (count != static_cast<Py_ssize_t>(sizeof...(A))) {
      PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", static_cast<Py_ssize_t>(sizeof...(A)), count);
      return nullptr;
    }
    return call(args, std::index_sequence_for<A...>{});
  }
};

// kv_cache(k_base, v_base, block_table, max_blocks, page_size, page_stride, token_stride, dtype,
// num_pages) -> bytes: struct pluto_kv_cache of one pool.
PyObject* kv_cache(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 9) {
    PyErr_SetString(PyExc_TypeError, "kv_cache takes 9 arguments");
    return nullptr;
  }
  pluto_kv_cache c = {};
  if (!convert(args[0], c.k_base) || !convert(args[1], c.v_base) || !convert(args[2], c.block_table) ||
      !convert(args[3], c.max_blocks) || !convert(args[4], c.page_size) || !convert(args[5], c.page_stride) ||
      !convert(args[6], c.token_stride) || !convert(args[7], c.dtype) || !convert(args[8], c.num_pages))
    return nullptr;
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&c), sizeof(c));
}

// ---- tensors, by the attributes that a Python caller would ask for ---------------------------------------------
struct Names {
  PyObject *shape, *stride, *dtype, *data_ptr, *get_device, *is_contiguous, *element_size;
};
Names names;
PyObject* refusal;    // class of the error: (code name, message, code)
PyObject* dtypes[4];  // fp32, bf16, E4M3, int32
constexpr int kInt32 = 3;

// bind_tensors(error class, fp32, bf16, E4M3, int32): the objects that the functions below compare with and raise.
PyObject* bind_tensors(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 5) {
    PyErr_SetString(PyExc_TypeError, "bind_tensors takes 5 arguments");
    return nullptr;
  }
  names = {PyUnicode_InternFromString("shape"), PyUnicode_InternFromString("stride"), PyUnicode_InternFromString("dtype"),
           PyUnicode_InternFromString("data_ptr"), PyUnicode_InternFromString("get_device"), PyUnicode_InternFromString("is_contiguous"),
           PyUnicode_InternFromString("element_size")};
  for (int i = 0; i < 5; ++i) Py_INCREF(args[i]);
  refusal = args[0];
  for (int i = 0; i < 4; ++i) dtypes[i] = args[1 + i];
  Py_RETURN_NONE;
}

bool refuse(const char* message) {   // false, with the error set
  if (PyErr_Occurred()) return false;
  if (PyObject* e = PyObject_CallFunction(refusal, "ssi", "InvalidArgument", message, -1)) {
    PyErr_SetObject(refusal, e);
    Py_DECREF(e);
  }
  return false;
}

struct Sizes {
  Py_ssize_t rank;
  long long n[4];
  bool operator==(const Sizes& o) const {
    if (rank != o.rank) return false;
    for (Py_ssize_t i = 0; i < rank && i < 4; ++i)
      if (n[i] != o.n[i]) return false;
    return true;
  }
};
bool take_sizes(PyObject* tuple, Sizes& out) {   // takes the reference; at most four dimensions are kept
  if (tuple == nullptr) return false;
  out.rank = PyTuple_Check(tuple) ? PyTuple_GET_SIZE(tuple) : 0;
  for (Py_ssize_t i = 0; i < out.rank && i < 4; ++i) out.n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
  Py_DECREF(tuple);
  return !PyErr_Occurred();
}
bool shape_of(PyObject* t, Sizes& out) { return take_sizes(PyObject_GetAttr(t, names.shape), out); }
bool strides_of(PyObject* t, Sizes& out) { return take_sizes(PyObject_CallMethodNoArgs(t, names.stride), out); }
long long number_of(PyObject* t, PyObject* method) {   // -2 with an error set
  PyObject* v = PyObject_CallMethodNoArgs(t, method);
  if (v == nullptr) return -2;
  const long long n = PyLong_AsLongLong(v);
  Py_DECREF(v);
  return PyErr_Occurred() ? -2 : n;
}
template <typename T>
bool address_of(PyObject* t, T*& out) {
  PyObject* v = PyObject_CallMethodNoArgs(t, names.data_ptr);
  if (v == nullptr) return false;
  out = reinterpret_cast<T*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(v)));
  Py_DECREF(v);
  return !PyErr_Occurred();
}
int dtype_of(PyObject* t) {   // index into dtypes, -1 for others, -2 with an error set
  PyObject* d = PyObject_GetAttr(t, names.dtype);
  if (d == nullptr) return -2;
  Py_DECREF(d);   // (torch keeps its dtypes alive)
  for (int i = 0; i < 4; ++i)
    if (d == dtypes[i]) return i;
  return -1;
}
// A contiguous int32 tensor of the given shape on the device; its address.
bool int32_of(PyObject* t, const Sizes& want, long long device, const char* what, const int32_t*& out) {
  Sizes shape;
  if (dtype_of(t) == kInt32 && shape_of(t, shape) && shape == want && number_of(t, names.get_device) == device && number_of(t, names.is_contiguous) == 1)
    return address_of(t, out);
  char message[160];
  if (want.rank == 1) snprintf(message, sizeof(message), "%s must be a contiguous int32 tensor of shape [%lld] on the current device", what, want.n[0]);
  else snprintf(message, sizeof(message), "%s must be a contiguous int32 tensor of shape [%lld, %lld] on the current device", what, want.n[0], want.n[1]);
  return refuse(message);
}

// int32_address(t, device, what, n0[, n1]) -> address of an optional contiguous int32 tensor of that shape, or None.
PyObject* int32_address(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 4 && count != 5) {
    PyErr_SetString(PyExc_TypeError, "int32_address takes 4 or 5 arguments");
    return nullptr;
  }
  if (args[0] == Py_None) Py_RETURN_NONE;
  Sizes want{count - 3, {}};
  long long device;
  if (!convert(args[1], device) || !convert(args[3], want.n[0]) || (count == 5 && !convert(args[4], want.n[1]))) return nullptr;
  const char* what = PyUnicode_AsUTF8(args[2]);
  const int32_t* out;
  if (what == nullptr || !int32_of(args[0], want, device, what, out)) return nullptr;
  return PyLong_FromVoidPtr(const_cast<int32_t*>(out));
}

bool fill_draft_pool(PyObject* const* args, pluto_kv_cache& c, pluto_kv_scales& s) {
  PyObject *k = args[0], *v = args[1], *table = args[2];
  long long batch, device;
  if (!convert(args[5], batch) || !convert(args[6], device)) return false;
  const int code = dtype_of(k);
  if (code < 0 || code > PLUTO_E4M3 || dtype_of(v) != code) return refuse("a cache pool stores fp32, bf16 or E4M3");
  Sizes shape, other, strides, other_strides;
  if (!shape_of(k, shape) || !shape_of(v, other) || !strides_of(k, strides) || !strides_of(v, other_strides)) return false;
  if (shape.rank != 4 || !(other == shape) || !(other_strides == strides) || strides.n[3] != 1 || strides.n[2] != shape.n[3])
    return refuse("cache pools are [pages, page_size, kv_heads, head_dim] of one shape, heads contiguous");
  if (number_of(k, names.get_device) != device || number_of(v, names.get_device) != device) return refuse("the cache is not on the current device");
  c.dtype = code;
  if (shape.n[0] > INT32_MAX || shape.n[1] > INT32_MAX) return refuse("cache pools have at most 2^31 - 1 pages of as many slots");
  c.num_pages = static_cast<int>(shape.n[0]);
  c.page_size = static_cast<int>(shape.n[1]);
  c.page_stride = static_cast<size_t>(strides.n[0]);
  c.token_stride = static_cast<size_t>(strides.n[1]);
  if (!address_of(k, c.k_base) || !address_of(v, c.v_base)) return false;
  if (table == Py_None) {
    if (shape.n[0] < batch) return refuse("a cache without a block table has a page for every sequence");
  } else {
    Sizes blocks;
    if (!shape_of(table, blocks)) return false;
    // (a table without columns has no address, which would pass for no table: a page of its own for every sequence)
    if (blocks.rank != 2 || blocks.n[1] < 1 || blocks.n[1] > INT32_MAX) return refuse("a block table is [batch, blocks], of one block or more");
    if (!int32_of(table, Sizes{2, {batch, blocks.n[1]}}, device, "block table", c.block_table)) return false;
    c.max_blocks = static_cast<int>(blocks.n[1]);
  }
  if ((code == PLUTO_E4M3) != (args[3] != Py_None) || (code == PLUTO_E4M3) != (args[4] != Py_None))
    return refuse("an 8-bit cache needs its scales, and only that");
  if (code != PLUTO_E4M3) return true;
  const Sizes rows{3, {shape.n[0], shape.n[1], shape.n[2]}};
  uint8_t** bases[2] = {&s.k, &s.v};
  for (int side = 0; side < 2; ++side) {
    PyObject* t = args[3 + side];
    if (!shape_of(t, other) || !strides_of(t, side ? other_strides : strides)) return false;
    if (!(other == rows) || number_of(t, names.element_size) != 1 || number_of(t, names.get_device) != device ||
        (side ? !(other_strides == strides) : strides.n[2] != 1 && shape.n[2] != 1))
      return refuse("cache scales are one byte each, [pages, page_size, kv_heads], heads contiguous");
    if (!address_of(t, *bases[side])) return false;
  }
  s.page_stride = static_cast<size_t>(strides.n[0]);
  s.token_stride = static_cast<size_t>(strides.n[1]);
  return true;
}

// draft_pool(k_pool, v_pool, block_table, k_scales, v_scales, batch, device) -> (bytes of struct pluto_kv_cache, bytes of
// struct pluto_kv_scales or None): the pool that the functions of drafted tokens take, after every check of its tensors.
PyObject* draft_pool(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 7) {
    PyErr_SetString(PyExc_TypeError, "draft_pool takes 7 arguments");
    return nullptr;
  }
  pluto_kv_cache c = {};
  pluto_kv_scales s = {};
  if (!fill_draft_pool(args, c, s)) return nullptr;
  return c.dtype != PLUTO_E4M3 ? Py_BuildValue("y#O", reinterpret_cast<const char*>(&c), static_cast<Py_ssize_t>(sizeof(c)), Py_None)
                               : Py_BuildValue("y#y#", reinterpret_cast<const char*>(&c), static_cast<Py_ssize_t>(sizeof(c)),
                                               reinterpret_cast<const char*>(&s), static_cast<Py_ssize_t>(sizeof(s)));
}

template <auto Function>
constexpr PyMethodDef entry(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&Entry<Function>::fastcall)), METH_FASTCALL, nullptr};
}
#define ENTRY(name) entry<&name>(#name)

PyMethodDef methods[] = {
    ENTRY(pluto_attn_fwd),
    ENTRY(pluto_attn_bwd),
    ENTRY(pluto_attn_bwd_workspace_bytes),
    ENTRY(pluto_attn_probs),
    ENTRY(pluto_gqa_prefill_fwd),
    ENTRY(pluto_gqa_prefill_fwd_workspace_bytes),
    ENTRY(pluto_gqa_gate_bwd),
    ENTRY(pluto_gqa_prefill_bwd),
    ENTRY(pluto_gqa_prefill_bwd_workspace_bytes),
    ENTRY(pluto_qk_prepare_bwd),
    ENTRY(pluto_qk_prepare_bwd_workspace_bytes),
    ENTRY(pluto_qk_prepare),
    ENTRY(pluto_gqa_decode),
    ENTRY(pluto_gqa_decode_workspace_bytes),
    ENTRY(pluto_gqa_decode_noalloc),
    ENTRY(pluto_gqa_decode_probs),
    ENTRY(pluto_cached_attention_step),
    ENTRY(pluto_cached_attention_step_workspace_bytes),
    ENTRY(pluto_kv8_append),
    ENTRY(pluto_kv8_read),
    ENTRY(pluto_kv_keep),
    ENTRY(pluto_draft_prepare),
    ENTRY(pluto_gqa_tree_decode),
    ENTRY(pluto_gqa_tree_decode_workspace_bytes),
    ENTRY(pluto_verify_drafts),
    ENTRY(pluto_gdn_token_step),
    ENTRY(pluto_gdn_token_step_scratch_bytes),
    ENTRY(pluto_gdn_gates),
    ENTRY(pluto_gdn_conv_silu),
    ENTRY(pluto_gdn_prefill),
    ENTRY(pluto_gdn_prefill_workspace_bytes),
    ENTRY(pluto_gdn_step),
    ENTRY(pluto_gdn_out_norm_gate),
    ENTRY(pluto_gdn_out_norm_gate_bwd),
    ENTRY(pluto_gdn_out_norm_gate_bwd_workspace_bytes),
    ENTRY(pluto_gdn_recurrence_bwd),
    ENTRY(pluto_gdn_recurrence_bwd_workspace_bytes),
    ENTRY(pluto_gdn_conv_silu_bwd),
    ENTRY(pluto_linear_imported_fwd),
    ENTRY(pluto_dense_fwd),
    ENTRY(pluto_dense_bwd),
    ENTRY(pluto_dense_workspace_bytes),
    ENTRY(pluto_block_linear_fwd),
    ENTRY(pluto_block_linear_bwd),
    ENTRY(pluto_block_linear_workspace_bytes),
    ENTRY(pluto_dequantize_matrix),
    {"kv_cache", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&kv_cache)), METH_FASTCALL, nullptr},
    {"bind_tensors", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind_tensors)), METH_FASTCALL, nullptr},
    {"int32_address", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&int32_address)), METH_FASTCALL, nullptr},
    {"draft_pool", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&draft_pool)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
