// The Python side of the 16-bit paged caches' calls: torch tensors checked and handed to the C ABI (xtg_cuda_kv16_*), as
// kv4_torch.cpp does for the 4-bit cache.
#define XTG_NAME "kv16"
#include "torch_call.h"

namespace {

decltype(&xtg_cuda_kv16_append) append_fn = nullptr;
decltype(&xtg_cuda_kv16_workspace) workspace_fn = nullptr;
decltype(&xtg_cuda_kv16_attention) attention_fn = nullptr;

// k_pool, v_pool (None: k_pool is a latent cache's pool), table, pos, cu_rows, err -> the C ABI's descriptor
xtg_cuda_kv16 where(PyObject* const* args, int64_t rows, c10::Device& dev) {
  const at::Tensor& k = tensor(args[0], "the pool");
  const bool latent = args[1] == Py_None;
  const at::Tensor &table = tensor(args[2], "table"), &pos = tensor(args[3], "pos"), &cu_rows = tensor(args[4], "cu_rows");
  dev = k.device();
  xtg_cuda_kv16 c = {};
  c.dtype = code_of(k.scalar_type());
  require(dev.is_cuda() && c.dtype >= 1, "the pool is a CUDA tensor of bfloat16 or float16");
  require(k.dim() == (latent ? 3 : 4) && k.stride(-1) == 1,
          latent ? "the pool is [pages][page][latent + 64] with contiguous dims"
                 : "k_pool is [pages][kv_heads][page][head_dim] with contiguous dims");
  for (int64_t n : k.sizes()) require(n >= 1 && n <= INT32_MAX, "pool sizes in 1 .. 2^31 - 1");
  c.k = k.data_ptr();
  c.pages = k.size(0);
  c.page = (int)k.size(-2);
  c.kv_heads = latent ? 1 : (int)k.size(1);
  c.head_dim = (int)k.size(-1);
  c.v_dim = c.head_dim - 64;
  c.k_page = stride(k, 0);
  c.k_head = latent ? 0 : stride(k, 1);
  c.k_slot = stride(k, latent ? 1 : 2);
  if (!latent) {
    const at::Tensor& v = tensor(args[1], "v_pool");
    require(v.dim() == 4 && v.scalar_type() == k.scalar_type() && v.device() == dev && v.size(0) == k.size(0) &&
                v.size(1) == k.size(1) && v.size(2) == k.size(2) && v.size(3) >= 1 && v.size(3) <= INT32_MAX &&
                v.stride(3) == 1,
            "v_pool is [pages][kv_heads][page][v_dim], of k_pool's type, sizes and device, with contiguous dims");
    c.v = v.data_ptr();
    c.v_dim = (int)v.size(3);
    c.v_page = stride(v, 0);
    c.v_head = stride(v, 1);
    c.v_slot = stride(v, 2);
  }
  require_index("table", table, 2, dev);
  require_index("pos", pos, 1, dev);
  require_index("cu_rows", cu_rows, 1, dev);
  const int64_t seqs = table.size(0);
  require(pos.size(0) == seqs && cu_rows.size(0) == seqs + 1, "table [seqs][max_pages], pos [seqs], cu_rows [seqs + 1]");
  require(seqs < INT32_MAX && table.size(1) <= INT32_MAX, "sizes below 2^31");
  c.table = table.data_ptr<int32_t>();
  c.max_pages = (int)table.size(1);
  c.seqs = (int)seqs;
  c.pos = pos.data_ptr<int32_t>();
  c.cu_rows = cu_rows.data_ptr<int32_t>();
  c.rows = rows;
  if (args[5] != Py_None) {
    const at::Tensor& e = tensor(args[5], "err");
    require(e.scalar_type() == at::kInt && e.numel() == 1 && e.device() == dev, "err is one int32 on the pool's device");
    c.err = e.data_ptr<int32_t>();
  }
  return c;
}

// t is [rows][heads][dims] (heads 0: any number; below 0: [rows][dims]) with contiguous dims
void require_rows(const char* name, const at::Tensor& t, int64_t rows, int64_t heads, int64_t dims, at::ScalarType type,
                  c10::Device dev) {
  const bool ok = heads < 0 ? t.dim() == 2 : t.dim() == 3 && (heads == 0 || t.size(1) == heads);
  require(ok && t.size(0) == rows && t.size(-1) == dims && t.device() == dev && t.stride(-1) == 1,
          std::string(name) + (heads < 0 ? " is [rows][" : " is [rows][heads][") + std::to_string(dims) +
              "] with contiguous dims on the pool's device");
  require(t.scalar_type() == type, std::string(name) + " has the type of the call's other rows (of the cache for attention)");
  require(t.dim() < 3 || t.size(1) <= INT32_MAX, "sizes below 2^31");
}

// bind(error class, addresses of the three C functions)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* cls;
  unsigned long long append, workspace, attention;
  if (!PyArg_ParseTuple(args, "OKKK", &cls, &append, &workspace, &attention)) return nullptr;
  Py_INCREF(cls);
  Py_XDECREF(error_class);
  error_class = cls;
  append_fn = reinterpret_cast<decltype(append_fn)>(append);
  workspace_fn = reinterpret_cast<decltype(workspace_fn)>(workspace);
  attention_fn = reinterpret_cast<decltype(attention_fn)>(attention);
  Py_RETURN_NONE;
}

// append(k_pool, v_pool or None, table, pos, cu_rows, err, k, v, freq or None, q or None, first, interleaved) -> q's rows
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("append", n, 12, [&]() -> PyObject* {
    const at::Tensor &k = tensor(args[6], "k"), &v = tensor(args[7], "v");
    c10::Device dev(c10::kCPU);
    require(k.dim() >= 1, "k has rows");
    const xtg_cuda_kv16 c = where(args, k.size(0), dev);
    const bool latent = !c.v;
    xtg_cuda_kv16_rows r = {};
    r.dtype = code_of(k.scalar_type());
    require(r.dtype >= 0, "k is float32, bfloat16 or float16");
    const int64_t dims = latent ? 64 : c.head_dim;
    require_rows("k", k, c.rows, latent ? -1 : c.kv_heads, dims, k.scalar_type(), dev);
    require_rows(latent ? "the latent vectors" : "v", v, c.rows, latent ? -1 : c.kv_heads, c.v_dim, k.scalar_type(), dev);
    r.k = k.data_ptr();
    r.v = v.data_ptr();
    r.k_row = stride(k, 0);
    r.v_row = stride(v, 0);
    if (!latent) {
      r.k_head = stride(k, 1);
      r.v_head = stride(v, 1);
    }
    if (args[8] != Py_None) {
      const at::Tensor& freq = tensor(args[8], "freq");
      require(freq.scalar_type() == at::kFloat && freq.dim() == 1 && freq.device() == dev && freq.is_contiguous() &&
                  freq.size(0) <= 128,
              "freq is a contiguous float32 tensor [rotary / 2] on the pool's device, at most 128 pairs");
      r.freq = freq.data_ptr<float>();
      r.rotary = 2 * (int)freq.size(0);
      r.first = small(args[10], "first");
    }
    const int interleaved = PyObject_IsTrue(args[11]);
    if (interleaved < 0) {
      PyErr_Clear();
      throw Refused("kv16: interleaved is a truth value");
    }
    r.interleaved = interleaved;
    at::Tensor out;
    if (args[9] != Py_None) {
      const at::Tensor& q = tensor(args[9], "q");
      require_rows("q", q, c.rows, 0, dims, k.scalar_type(), dev);
      require(q.size(1) >= 1, "q has heads");
      r.q = q.data_ptr();
      r.heads = (int)q.size(1);
      r.q_row = stride(q, 0);
      r.q_head = stride(q, 1);
      out = at::empty(q.sizes(), at::TensorOptions().dtype(c.dtype == 1 ? at::kBFloat16 : at::kHalf).device(dev));
      r.q_out = out.data_ptr();
    }
    call(dev, [&](void* stream, char* why, int len) { return append_fn(&c, &r, stream, why, len); });
    if (args[9] == Py_None) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// attention(k_pool, v_pool or None, table, pos, cu_rows, err, q, q_rot or None, scale, window, rows_per_seq or None, out or
// None) -> out
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("attention", n, 12, [&]() -> PyObject* {
    const at::Tensor& q = tensor(args[6], "q");
    const double scale = PyFloat_AsDouble(args[8]);
    if (scale == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      throw Refused("kv16: scale is a number");
    }
    xtg_cuda_kv16_attn r = {};
    r.scale = (float)scale;
    r.window = small(args[9], "window");
    c10::Device dev(c10::kCPU);
    require(q.dim() == 3, "q is [rows][heads][dims]");
    const xtg_cuda_kv16 c = where(args, q.size(0), dev);
    const bool latent = !c.v;
    const at::ScalarType type = c.dtype == 1 ? at::kBFloat16 : at::kHalf;
    require_rows("q", q, c.rows, 0, latent ? c.v_dim : c.head_dim, type, dev);
    r.q = q.data_ptr();
    r.heads = (int)q.size(1);
    r.q_row = stride(q, 0);
    r.q_head = stride(q, 1);
    if (latent) {
      const at::Tensor& rot = tensor(args[7], "q_rot");
      require(q.size(1) >= 1, "q has heads");
      require_rows("q_rot", rot, c.rows, q.size(1), 64, type, dev);
      r.q_rot = rot.data_ptr();
      r.r_row = stride(rot, 0);
      r.r_head = stride(rot, 1);
    }
    const int64_t mean = c.seqs > 0 ? (c.rows + c.seqs - 1) / c.seqs : 1;
    r.rows_per_seq = args[10] == Py_None ? (int)std::min<int64_t>(std::max<int64_t>(mean, 1), INT32_MAX)
                                         : small(args[10], "rows_per_seq");
    at::Tensor out;
    if (args[11] == Py_None) {   // nothing unwritten is returned
      r.zero_rest = 1;
      out = at::empty({c.rows, q.size(1), c.v_dim}, at::TensorOptions().dtype(type).device(dev));
    } else {
      out = tensor(args[11], "out");
      require(out.dim() == 3 && out.size(0) == c.rows && out.size(1) == q.size(1) && out.size(2) == c.v_dim &&
                  out.scalar_type() == type && out.device() == dev && out.is_contiguous(),
              "out is contiguous, [rows][heads][v_dim] of the cache's type");
    }
    r.out = out.data_ptr();
    call(dev, [&](void* stream, char* why, int len) {
      r.workspace_bytes = workspace_fn(r.heads, c.kv_heads, c.head_dim, c.v_dim, latent, r.rows_per_seq);
      require(r.workspace_bytes >= 0,
              "q heads a multiple of KV heads, rows_per_seq at least 1, (head_dim, v_dim) (64, 64), (128, 128), (192, 128) or "
              "(256, 256), of a latent cache (320, 256) or (576, 512)");
      const at::Tensor work = at::empty({r.workspace_bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
      r.workspace = work.data_ptr();
      return attention_fn(&c, &r, stream, why, len);
    });
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv16_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv16_torch() { return PyModule_Create(&module); }
