// Python calls of the shared-prefix serving operators on torch tensors
// (dolittle_b200/shared.py documents them).  They are made once per block and
// decode step, where the interpreter's share of an argument-by-argument call
// through ctypes (13 us) outlasted the kernels of a small batch: here the
// checks, the allocations and the call take a few microseconds.  The C ABI
// itself is reached through the addresses given to bind().
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/dolittle_b200.h"

namespace {

decltype(&dl_attention_shared_workspace_bytes) attention_workspace_bytes;
decltype(&dl_attention_shared) attention_shared;
decltype(&dl_cache_evict_workspace_bytes) evict_workspace_bytes;
decltype(&dl_cache_evict) cache_evict;
decltype(&dl_last_error) last_error;
PyObject* refusal;  // DolittleError(status, message)

struct ArgumentError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw ArgumentError(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int64_t size_t_of(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw ArgumentError(std::string(name) + " must be an integer");
  }
  if (v < 0) throw ArgumentError(std::string(name) + " must not be negative");
  return v;
}

struct Caches {
  int64_t positions, heads, width, count, row, outer;
  void *key, *value;
};

// Key and value caches [(caches,) positions, heads, width]: bfloat16, one
// shape and layout, the heads of a position contiguous.  torch leaves the
// stride of a dimension of size 1 arbitrary; it is not used.
Caches caches(PyObject* k, PyObject* v, const std::string& name, int dims, c10::Device device) {
  const at::Tensor &key = tensor(k, "key caches"), &value = tensor(v, "value caches");
  if (key.scalar_type() != at::kBFloat16 || value.scalar_type() != at::kBFloat16 || key.dim() != dims ||
      value.sizes() != key.sizes() || key.device() != device || value.device() != device)
    throw ArgumentError(name + "_key and " + name + "_value must be bfloat16 tensors of one shape and " +
                        std::to_string(dims) + " dimensions, on the query's device");
  const auto n = key.sizes(), s = key.strides();
  Caches c;
  c.width = n[dims - 1];
  c.heads = n[dims - 2];
  c.positions = n[dims - 3];
  c.count = dims == 4 ? n[0] : 1;
  c.row = c.positions > 1 ? s[dims - 3] : c.heads * c.width;
  c.outer = c.count > 1 ? s[0] : c.row * c.positions;
  if ((s[dims - 1] != 1 && c.width > 1) || (s[dims - 2] != c.width && c.heads > 1))
    throw ArgumentError(name + "_key: the heads of a position must be contiguous");
  for (int i = 0; i < dims; ++i)
    if (n[i] > 1 && value.strides()[i] != s[i])
      throw ArgumentError(name + "_key and " + name + "_value must have the same strides");
  c.key = key.data_ptr();
  c.value = value.data_ptr();
  return c;
}

template <class T>
T* flat(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef sizes, c10::Device device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.sizes() != sizes || t.device() != device || !t.is_contiguous()) {
    std::string shape;
    for (int64_t n : sizes) shape += (shape.empty() ? "" : ", ") + std::to_string(n);
    throw ArgumentError(std::string(name) + " must be a contiguous " + at::toString(type) + " tensor (" + shape +
                        ") on the query's device");
  }
  return static_cast<T*>(t.data_ptr());
}

// A reference of our own.
struct Reference {
  PyObject* object = nullptr;
  Reference() = default;
  Reference(const Reference&) = delete;
  Reference& operator=(const Reference&) = delete;
  ~Reference() { Py_XDECREF(object); }
  void hold(PyObject* o) {
    Py_INCREF(o);
    object = o;
  }
  operator PyObject*() const { return object; }
};

struct Refused {
  dl_status status;
};
void require(dl_status s) {
  if (s != DL_OK) throw Refused{s};
}

// Runs `body`, whose result is a new reference, with every failure as a Python exception.
template <class F>
PyObject* guarded(F&& body) {
  try {
    return body();
  } catch (const ArgumentError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Refused& r) {
    if (PyObject* error = PyObject_CallFunction(refusal, "is", int(r.status), last_error())) {
      PyErr_SetObject(refusal, error);
      Py_DECREF(error);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* wrap(PyObject* given, const at::Tensor& made) {
  if (given == Py_None) return THPVariable_Wrap(made);
  Py_INCREF(given);
  return given;
}

at::Tensor scratch(size_t bytes, c10::Device device) {
  return at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(device));
}

// query, prefix_key, prefix_value, suffix_key, suffix_value, prefix_lengths,
// suffix_lengths, prefix_weights, suffix_weights, out, lse
PyObject* py_attention_shared(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11) throw ArgumentError("attention_shared takes 11 arguments");
    const at::Tensor& q = tensor(arg[0], "query");
    if (q.scalar_type() != at::kBFloat16 || q.dim() != 4)
      throw ArgumentError("query must be a bfloat16 CUDA tensor [batch, rows, heads, width]");
    const int64_t batch = q.size(0), rows = q.size(1), heads = q.size(2), width = q.size(3);
    // The stride between tokens, also where an expanded query has 0: the C
    // ABI's 0 is dense rows, which the storage of one token does not hold.
    const int64_t stride = rows > 1 ? q.stride(1) : batch > 1 ? q.stride(0) : heads * width;
    if ((q.stride(3) != 1 && width > 1) || (q.stride(2) != width && heads > 1) || stride < heads * width ||
        (rows > 1 && batch > 1 && q.stride(0) != rows * stride))
      throw ArgumentError("query: heads contiguous, one stride between tokens, at least a token's heads");
    if (!q.is_cuda()) throw ArgumentError("query must be a bfloat16 CUDA tensor [batch, rows, heads, width]");
    const c10::Device device = q.device();
    dl_shared_attention a = {};
    a.batch = batch;
    a.rows = rows;
    a.query_heads = heads;
    a.width = width;
    a.query_stride = stride;
    if (arg[1] != Py_None) {
      const Caches c = caches(arg[1], arg[2], "prefix", 3, device);
      if (c.width != width) throw ArgumentError("prefix caches must have the query's head width");
      a.kv_heads = c.heads;
      a.prefix_key = c.key;
      a.prefix_value = c.value;
      a.prefix_capacity = c.positions;
      a.prefix_row_stride = c.row;
      a.prefix_lengths = flat<int64_t>(arg[5], "prefix_lengths", at::kLong, {batch}, device);
    }
    if (arg[3] != Py_None) {
      const Caches c = caches(arg[3], arg[4], "suffix", 4, device);
      if (c.count != batch || c.width != width || (arg[1] != Py_None && c.heads != int64_t(a.kv_heads)))
        throw ArgumentError(
            "suffix caches must be [batch, positions, the prefix's KV heads, the query's head width]");
      a.kv_heads = c.heads;
      a.suffix_key = c.key;
      a.suffix_value = c.value;
      a.suffix_capacity = c.positions;
      a.suffix_row_stride = c.row;
      a.suffix_sequence_stride = c.outer;
      a.suffix_lengths = flat<int64_t>(arg[6], "suffix_lengths", at::kLong, {batch}, device);
    }
    if (arg[1] == Py_None && arg[3] == Py_None) throw ArgumentError("a prefix or a suffix cache is required");
    float *pw = nullptr, *sw = nullptr, *lse_ptr = nullptr;
    if (arg[7] != Py_None)
      pw = flat<float>(arg[7], "prefix_weights", at::kFloat, {int64_t(a.kv_heads), int64_t(a.prefix_capacity)}, device);
    if (arg[8] != Py_None)
      sw = flat<float>(arg[8], "suffix_weights", at::kFloat,
                       {batch, int64_t(a.kv_heads), int64_t(a.suffix_capacity)}, device);
    at::Tensor out, lse;
    void* out_ptr;
    const auto options = at::TensorOptions().device(device);
    if (arg[9] == Py_None) {
      out = at::empty(q.sizes(), options.dtype(at::kBFloat16));
      out_ptr = out.data_ptr();
    } else {
      out_ptr = flat<void>(arg[9], "out", at::kBFloat16, q.sizes(), device);
    }
    if (arg[10] == Py_None) {
      lse = at::empty({batch, rows, heads}, options.dtype(at::kFloat));
      lse_ptr = lse.data_ptr<float>();
    } else {
      lse_ptr = flat<float>(arg[10], "lse", at::kFloat, {batch, rows, heads}, device);
    }
    const c10::cuda::OptionalCUDAGuard guard(device);
    // A refused call has a workspace of 0 bytes, and the call itself says why.
    const at::Tensor workspace = scratch(attention_workspace_bytes(&a, pw || sw), device);
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    dl_status status;
    Py_BEGIN_ALLOW_THREADS
    status = attention_shared(&a, q.data_ptr(), out_ptr, lse_ptr, pw, sw, workspace.data_ptr(), stream);
    Py_END_ALLOW_THREADS
    require(status);
    PyObject* result = PyTuple_New(2);
    if (!result) return nullptr;
    PyTuple_SET_ITEM(result, 0, wrap(arg[9], out));
    PyTuple_SET_ITEM(result, 1, wrap(arg[10], lse));
    return result;
  });
}

// key, value, weights, positions, lengths, budget, first, recent, out (a
// sequence of five tensors, or None: in place)
PyObject* py_cache_evict(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 9) throw ArgumentError("cache_evict takes 9 arguments");
    // The results' own references, until they are returned: a sequence may
    // make its elements on access and keep none, or change meanwhile.
    Reference out[5];
    if (arg[8] == Py_None) {
      for (int i = 0; i < 5; ++i) out[i].hold(arg[i]);
    } else {
      if (!PySequence_Check(arg[8]) || PySequence_Size(arg[8]) != 5)
        throw ArgumentError("out must be (key, value, weights, positions, lengths)");
      for (int i = 0; i < 5; ++i) {
        out[i].object = PySequence_GetItem(arg[8], i);
        if (!out[i]) throw ArgumentError("out must be (key, value, weights, positions, lengths)");
      }
    }
    const at::Tensor& key = tensor(arg[0], "key caches");
    if (!key.is_cuda()) throw ArgumentError("the caches must be CUDA tensors");
    const c10::Device device = key.device();
    const Caches c = caches(arg[0], arg[1], "cache", 4, device);
    const Caches o = arg[8] == Py_None ? c : caches(out[0], out[1], "out", 4, device);
    if (o.count != c.count || o.heads != c.heads || o.width != c.width)
      throw ArgumentError("the output caches must be [caches, positions, heads, width] like the inputs");
    dl_cache_eviction e = {};
    e.caches = c.count;
    e.kv_heads = c.heads;
    e.width = c.width;
    e.capacity = c.positions;
    e.budget = size_t_of(arg[5], "budget");
    e.first = size_t_of(arg[6], "first");
    e.recent = size_t_of(arg[7], "recent");
    e.key = c.key;
    e.value = c.value;
    e.row_stride = c.row;
    e.cache_stride = c.outer;
    e.weights = flat<float>(arg[2], "weights", at::kFloat, {c.count, c.heads, c.positions}, device);
    e.positions = flat<int32_t>(arg[3], "positions", at::kInt, {c.count, c.heads, c.positions}, device);
    e.lengths = flat<int64_t>(arg[4], "lengths", at::kLong, {c.count}, device);
    e.key_out = o.key;
    e.value_out = o.value;
    e.out_capacity = o.positions;
    e.out_row_stride = o.row;
    e.out_cache_stride = o.outer;
    e.weights_out = flat<float>(out[2], "weights (output)", at::kFloat, {c.count, c.heads, o.positions}, device);
    e.positions_out = flat<int32_t>(out[3], "positions (output)", at::kInt, {c.count, c.heads, o.positions}, device);
    e.lengths_out = flat<int64_t>(out[4], "lengths (output)", at::kLong, {c.count}, device);
    const c10::cuda::OptionalCUDAGuard guard(device);
    const at::Tensor workspace = scratch(evict_workspace_bytes(&e), device);
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    dl_status status;
    Py_BEGIN_ALLOW_THREADS
    status = cache_evict(&e, workspace.data_ptr(), stream);
    Py_END_ALLOW_THREADS
    require(status);
    return PyTuple_Pack(5, out[0].object, out[1].object, out[2].object, out[3].object, out[4].object);
  });
}

// Addresses of the five C functions in the order above, then DolittleError.
PyObject* py_bind(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "bind takes 6 arguments");
    return nullptr;
  }
  void* f[5];
  for (int i = 0; i < 5; ++i) {
    f[i] = PyLong_AsVoidPtr(arg[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function");
      return nullptr;
    }
  }
  attention_workspace_bytes = reinterpret_cast<decltype(attention_workspace_bytes)>(f[0]);
  attention_shared = reinterpret_cast<decltype(attention_shared)>(f[1]);
  evict_workspace_bytes = reinterpret_cast<decltype(evict_workspace_bytes)>(f[2]);
  cache_evict = reinterpret_cast<decltype(cache_evict)>(f[3]);
  last_error = reinterpret_cast<decltype(last_error)>(f[4]);
  Py_INCREF(arg[5]);
  Py_XSETREF(refusal, arg[5]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"attention_shared", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention_shared)),
     METH_FASTCALL, nullptr},
    {"cache_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_cache_evict)), METH_FASTCALL,
     nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_shared", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_shared() { return PyModule_Create(&module); }
