// The Python side of the 4-bit cache's calls: torch tensors checked and handed to the C ABI (xtg_cuda_kv4_*), outputs and
// workspaces allocated by torch on the current stream. A call here costs 4 to 9 us of host time, the launches included;
// through ctypes it cost 10 to 17, more than the small calls run on the GPU. The C ABI's functions come from the library
// that the package loaded (bind), so this module links torch only.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../../include/xtg_cuda.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

PyObject* error_class = nullptr;
decltype(&xtg_cuda_kv4_store) store_fn = nullptr;
decltype(&xtg_cuda_kv4_load) load_fn = nullptr;
decltype(&xtg_cuda_kv4_workspace) workspace_fn = nullptr;
decltype(&xtg_cuda_kv4_attention) attention_fn = nullptr;

void require(bool ok, const std::string& why) {
  if (!ok) throw Refused("kv4: " + why);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  require(THPVariable_Check(o), std::string(name) + " is a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused(std::string("kv4: ") + name + " is an integer");
  }
  return v;
}

int small(PyObject* o, const char* name) {
  const int64_t v = integer(o, name);
  require(v >= INT32_MIN && v <= INT32_MAX, std::string(name) + " is a 32-bit integer");
  return (int)v;
}

int code_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

void require_index(const char* name, const at::Tensor& t, int dims, c10::Device dev) {
  require(t.scalar_type() == at::kInt && t.dim() == dims && t.device() == dev && t.is_contiguous(),
          std::string(name) + " is a contiguous int32 tensor of " + std::to_string(dims) +
              " dimension(s) on the pool's device");
}

// pool, table, pos, cu_rows, err (a tensor or None) -> the C ABI's descriptor
xtg_cuda_kv4 where(PyObject* const* args, int64_t rows, c10::Device& dev) {
  const at::Tensor &pool = tensor(args[0], "pool"), &table = tensor(args[1], "table"), &pos = tensor(args[2], "pos"),
                   &cu_rows = tensor(args[3], "cu_rows");
  dev = pool.device();
  require(pool.scalar_type() == at::kByte && pool.dim() == 3 && pool.is_contiguous() && dev.is_cuda(),
          "pool is a contiguous uint8 CUDA tensor [pages][kv_heads][72 head_dim]");
  const int64_t block = pool.size(2);
  require(block == 72 * 64 || block == 72 * 128 || block == 72 * 256,
          "head_dim 64, 128 or 256 (pool.shape[2] / 72)");
  require_index("table", table, 2, dev);
  require_index("pos", pos, 1, dev);
  require_index("cu_rows", cu_rows, 1, dev);
  const int64_t seqs = table.size(0);
  require(pos.size(0) == seqs && cu_rows.size(0) == seqs + 1, "table [seqs][max_pages], pos [seqs], cu_rows [seqs + 1]");
  require(pool.size(1) <= INT32_MAX && seqs < INT32_MAX && table.size(1) <= INT32_MAX, "sizes below 2^31");
  int32_t* err = nullptr;
  if (args[4] != Py_None) {
    const at::Tensor& e = tensor(args[4], "err");
    require(e.scalar_type() == at::kInt && e.numel() == 1 && e.device() == dev, "err is one int32 on the pool's device");
    err = e.data_ptr<int32_t>();
  }
  return {pool.data_ptr<uint8_t>(), pool.size(0), (int)pool.size(1), (int)(block / 72), table.data_ptr<int32_t>(),
          (int)table.size(1), (int)seqs, pos.data_ptr<int32_t>(), cu_rows.data_ptr<int32_t>(), rows, err};
}

// The dtype code of rows t [rows][heads][head_dim] with contiguous head dims (heads 0: any number)
int rows_type(const char* name, const at::Tensor& t, int64_t heads, const xtg_cuda_kv4& c, c10::Device dev) {
  const int code = code_of(t.scalar_type());
  require(code >= 0, std::string(name) + " is float32, bfloat16 or float16");
  require(t.dim() == 3 && t.size(2) == c.head_dim && (heads == 0 || t.size(1) == heads) && t.device() == dev,
          std::string(name) + " is [rows][heads][head_dim] of the pool's head_dim on the pool's device");
  require(t.stride(2) == 1, std::string(name) + "'s head dims must be contiguous");
  return code;
}

// The stride of dimension d; that of a single row or head, which nothing steps by, may be any number.
int64_t stride(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Runs f (which gets the current stream and a message buffer) with device dev current.
template <class F>
void call(c10::Device dev, F&& f) {
  char why[1024] = "";
  const c10::cuda::CUDAGuard guard(dev);
  if (f(c10::cuda::getCurrentCUDAStream(dev.index()).stream(), why, (int)sizeof(why)) != 0) throw Refused(why);
}

// A METH_FASTCALL function of n arguments; C++ exceptions end here, as the package's error class.
template <class F>
PyObject* entry(const char* name, Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  try {
    require(attention_fn != nullptr, "bind first");
    require(given == wanted, std::string(name) + " takes " + std::to_string(wanted) + " arguments");
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, "kv4: unknown error");
  }
  return nullptr;
}

// bind(error class, addresses of the four C functions)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* cls;
  unsigned long long store, load, workspace, attention;
  if (!PyArg_ParseTuple(args, "OKKKK", &cls, &store, &load, &workspace, &attention)) return nullptr;
  Py_INCREF(cls);
  Py_XDECREF(error_class);
  error_class = cls;
  store_fn = reinterpret_cast<decltype(store_fn)>(store);
  load_fn = reinterpret_cast<decltype(load_fn)>(load);
  workspace_fn = reinterpret_cast<decltype(workspace_fn)>(workspace);
  attention_fn = reinterpret_cast<decltype(attention_fn)>(attention);
  Py_RETURN_NONE;
}

// store(pool, table, pos, cu_rows, err, k, v)
PyObject* store(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("store", n, 7, [&]() -> PyObject* {
    const at::Tensor &k = tensor(args[5], "k"), &v = tensor(args[6], "v");
    c10::Device dev(c10::kCPU);
    require(k.dim() == 3 && v.dim() == 3 && k.size(0) == v.size(0), "k and v have the same type and rows");
    const xtg_cuda_kv4 c = where(args, k.size(0), dev);
    const int type = rows_type("k", k, c.kv_heads, c, dev);
    require(rows_type("v", v, c.kv_heads, c, dev) == type, "k and v have the same type and rows");
    call(dev, [&](void* stream, char* why, int len) {
      return store_fn(&c, k.data_ptr(), v.data_ptr(), type, stride(k, 0), stride(k, 1), stride(v, 0), stride(v, 1),
                      stream, why, len);
    });
    Py_RETURN_NONE;
  });
}

// load(pool, table, pos, cu_rows, err, rows, dtype code) -> (k, v)
PyObject* load(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("load", n, 7, [&]() -> PyObject* {
    c10::Device dev(c10::kCPU);
    const int64_t rows = integer(args[5], "rows");
    const int type = small(args[6], "dtype");
    require(type >= 0 && type <= 2, "dtype is float32, bfloat16 or float16");
    require(rows >= 0, "rows is not negative");
    const xtg_cuda_kv4 c = where(args, rows, dev);
    const at::ScalarType types[3] = {at::kFloat, at::kBFloat16, at::kHalf};
    const auto options = at::TensorOptions().dtype(types[type]).device(dev);
    at::Tensor k = at::empty({rows, c.kv_heads, c.head_dim}, options), v = at::empty({rows, c.kv_heads, c.head_dim}, options);
    call(dev, [&](void* stream, char* why, int len) {
      return load_fn(&c, k.data_ptr(), v.data_ptr(), type + XTG_CUDA_KV4_ZERO_REST, stream, why, len);
    });
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(v)));
    return both;
  });
}

// attention(pool, table, pos, cu_rows, err, q, scale, window, rows_per_seq or None, out or None) -> out
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("attention", n, 10, [&]() -> PyObject* {
    const at::Tensor& q = tensor(args[5], "q");
    const double scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      throw Refused("kv4: scale is a number");
    }
    const int window = small(args[7], "window");
    c10::Device dev(c10::kCPU);
    require(q.dim() == 3, "q is [rows][heads][head_dim] of the pool's head_dim on the pool's device");
    const xtg_cuda_kv4 c = where(args, q.size(0), dev);
    const int type = rows_type("q", q, 0, c, dev);
    require(q.size(1) <= INT32_MAX, "sizes below 2^31");
    const int64_t mean = c.seqs > 0 ? (c.rows + c.seqs - 1) / c.seqs : 1;
    const int per_seq = args[8] == Py_None ? (int)std::min<int64_t>(std::max<int64_t>(mean, 1), INT32_MAX)
                                           : small(args[8], "rows_per_seq");
    at::Tensor out;
    int out_type = type;
    if (args[9] == Py_None) {   // nothing unwritten is returned
      out_type += XTG_CUDA_KV4_ZERO_REST;
      out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    } else {
      out = tensor(args[9], "out");
      require(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == dev && out.is_contiguous(),
              "out is contiguous, of q's shape and type");
    }
    call(dev, [&](void* stream, char* why, int len) {
      const int64_t bytes = workspace_fn((int)q.size(1), c.kv_heads, c.head_dim, per_seq);
      require(bytes >= 0, "q heads a multiple of KV heads, rows_per_seq at least 1");
      const at::Tensor work = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
      return attention_fn(&c, q.data_ptr(), out.data_ptr(), out_type, (int)q.size(1), stride(q, 0), stride(q, 1), (float)scale,
                          window, per_seq, work.data_ptr(), bytes, stream, why, len);
    });
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(store)), METH_FASTCALL, nullptr},
    {"load", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(load)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv4_torch() { return PyModule_Create(&module); }
