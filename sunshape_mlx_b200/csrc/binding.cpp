// Native lane of the paged operators' Python wrappers.
//
// Their kernels take a few microseconds on small inputs, less than a Python
// wrapper spends on checking tensors, allocating outputs and converting
// arguments. A function here does all of that for the ordinary call: it
// checks what the wrapper checks, allocates, launches through the C ABI on the
// current stream and returns the outputs. Where anything is not as expected
// (wrong types or shapes, nothing to do, tensors of another device, a status
// that is not 0) it returns None and has done nothing; the wrapper then goes
// its own way, which raises the error that belongs to the case.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/sunshape_b200.h"

namespace {

using at::Tensor;

// One call's view of its arguments. `ok` turns false at the first thing that is not as expected.
struct Call {
  PyObject* const* args;
  bool ok = true;
  int64_t device = -1;

  bool want(bool cond) { return ok = ok && cond; }
  const Tensor& tensor(int i) {
    static const Tensor none;
    if (!want(THPVariable_Check(args[i]))) return none;
    const Tensor& t = THPVariable_Unpack(args[i]);
    if (!want(t.is_cuda() && t.layout() == at::kStrided)) return none;
    if (device < 0) device = t.get_device();
    want(t.get_device() == device);
    return t;
  }
  // An input of which a result would have to keep the graph: the wrapper refuses it.
  void no_graph(const Tensor& t) {
    if (ok) want(!(t.requires_grad() && at::GradMode::is_enabled()));
  }
  int64_t integer(int i) {
    if (!want(PyLong_Check(args[i]))) return 0;
    const int64_t v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  double number(int i) {
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  bool truth(int i) {
    const int v = PyObject_IsTrue(args[i]);
    if (v < 0) {
      PyErr_Clear();
      ok = false;
    }
    return v == 1;
  }
  const Tensor& int32(int i, int dims) {
    const Tensor& t = tensor(i);
    if (ok) want(t.scalar_type() == at::kInt && t.dim() == dims && t.numel() > 0 && t.stride(dims - 1) == 1);
    return t;
  }
  // Pages of head_dim d; returns the tokens of a page. The pool has pages and kv heads then.
  int64_t pool(const Tensor& t, int64_t d) {
    if (!ok || !want(t.scalar_type() == at::kByte && t.dim() == 3 && t.stride(2) == 1 && t.size(0) > 0 && t.size(1) > 0 &&
                     (d == 64 || d == 128 || d == 256)))
      return 0;
    const int64_t bytes = t.size(2);
    return want(bytes >= 20 * d && bytes % (20 * d) == 0) ? bytes * 4 / (5 * d) : 0;
  }
  bool here() { return ok && want(device == c10::cuda::current_device()); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
};

int code_of(at::ScalarType t) {
  return t == at::kFloat ? SS_F32 : t == at::kHalf ? SS_F16 : t == at::kBFloat16 ? SS_BF16 : -1;
}

PyObject* wrap(std::initializer_list<Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// Runs a body that returns a new reference, or null for "not here"; no exception leaves it.
template <class F>
PyObject* lane(PyObject* const* args, Py_ssize_t n, Py_ssize_t expected, F&& body) {
  if (n == expected) {
    try {
      Call c{args};
      if (PyObject* r = body(c)) return r;
      if (PyErr_Occurred()) PyErr_Clear();
    } catch (...) {  // such as no memory for the outputs: the wrapper's own way reports it
    }
  }
  Py_RETURN_NONE;
}

// (seq_lens, q_lens, block_table, free_pages, n_free, page_size, n_tokens)
PyObject* plan_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return lane(args, nargs, 7, [](Call& c) -> PyObject* {
    const Tensor &lens = c.int32(0, 1), &q = c.int32(1, 1), &table = c.int32(2, 2), &free_pages = c.int32(3, 1), &left = c.int32(4, 1);
    const int64_t page = c.integer(5), tokens = c.integer(6);
    if (!c.ok) return nullptr;
    const int64_t n = lens.size(0);
    if (!c.want(q.size(0) == n && table.size(0) == n && left.size(0) == 1 && table.stride(0) >= table.size(1) && page >= 16 &&
                page % 16 == 0 && page < (1ll << 31) && tokens >= 0 && tokens < (1ll << 31) && n <= 16384) || !c.here())
      return nullptr;
    Tensor slots = at::empty({tokens}, lens.options().dtype(at::kLong));
    Tensor out = at::empty({2 * n + 3 + 2 * tokens}, lens.options());
    int32_t* p = out.data_ptr<int32_t>();
    int32_t *pos = p + n + 1, *req = pos + tokens, *now = req + tokens;
    if (ss_plan_step(lens.data_ptr<int32_t>(), q.data_ptr<int32_t>(), (int)n, table.data_ptr<int32_t>(), table.stride(0),
                     (int)table.size(1), free_pages.data_ptr<int32_t>(), (int)free_pages.size(0), left.data_ptr<int32_t>(), (int)page,
                     tokens, p, pos, req, slots.data_ptr<int64_t>(), now, now + n, now + n + 1, c.stream()))
      return nullptr;
    auto part = [&](int64_t at, int64_t count) { return out.as_strided({count}, {1}, at); };
    return wrap({part(0, n + 1), part(n + 1, tokens), part(n + 1 + tokens, tokens), slots, part(n + 1 + 2 * tokens, n),
                 part(2 * n + 1 + 2 * tokens, 1), part(2 * n + 2 + 2 * tokens, 1)});
  });
}

// (keys, values, slots, pages): True
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return lane(args, nargs, 4, [](Call& c) -> PyObject* {
    const Tensor &k = c.tensor(0), &v = c.tensor(1), &slots = c.tensor(2), &pages = c.tensor(3);
    if (!c.ok || !c.want(k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.size(0) > 0)) return nullptr;
    const int64_t n = k.size(0), h = k.size(1), d = k.size(2), page = c.pool(pages, d);
    const int dt = code_of(k.scalar_type());
    if (!c.want(dt >= 0 && page > 0 && pages.size(1) == h && k.stride(2) == 1 && v.stride(2) == 1 && slots.scalar_type() == at::kLong &&
                slots.dim() == 1 && slots.size(0) == n && slots.is_contiguous()) || !c.here())
      return nullptr;
    if (ss_int4_append(k.data_ptr(), v.data_ptr(), dt, k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr<int64_t>(), n,
                       (int)h, (int)d, pages.data_ptr(), pages.size(0), pages.stride(0), pages.stride(1), (int)page, c.stream()))
      return nullptr;
    Py_RETURN_TRUE;
  });
}

// (slots, pages, head_dim, dtype code): (keys, values)
PyObject* fetch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return lane(args, nargs, 4, [](Call& c) -> PyObject* {
    const Tensor &slots = c.tensor(0), &pages = c.tensor(1);
    const int64_t d = c.integer(2), dt = c.integer(3);
    if (!c.ok) return nullptr;
    const int64_t page = c.pool(pages, d);
    if (!c.want(page > 0 && dt >= SS_F32 && dt <= SS_BF16 && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) > 0 &&
                slots.is_contiguous()) || !c.here())
      return nullptr;
    const int64_t n = slots.size(0), h = pages.size(1);
    const auto opt = pages.options().dtype(dt == SS_F32 ? at::kFloat : dt == SS_F16 ? at::kHalf : at::kBFloat16);
    Tensor k = at::empty({n, h, d}, opt), v = at::empty({n, h, d}, opt);
    if (ss_int4_fetch(slots.data_ptr<int64_t>(), n, (int)h, (int)d, pages.data_ptr(), pages.size(0), pages.stride(0), pages.stride(1),
                      (int)page, k.data_ptr(), v.data_ptr(), (int)dt, c.stream()))
      return nullptr;
    return wrap({k, v});
  });
}

// (queries, pages, block_table, seq_lens, cu_q, scale, max_q, causal, window, return_lse, workspace): (out,) or (out, lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return lane(args, nargs, 11, [](Call& c) -> PyObject* {
    const Tensor &q = c.tensor(0), &pages = c.tensor(1), &table = c.int32(2, 2), &lens = c.int32(3, 1), &cu = c.int32(4, 1), &ws = c.tensor(10);
    const double scale = c.number(5);
    const int64_t max_q = c.integer(6), window = c.integer(8);
    const bool causal = c.truth(7), with_lse = c.truth(9);
    c.no_graph(q);
    if (!c.ok || !c.want(q.dim() == 3 && q.size(0) > 0)) return nullptr;
    const int64_t n = q.size(0), hq = q.size(1), d = q.size(2), page = c.pool(pages, d), b = lens.size(0);
    if (!c.want(page > 0 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && hq >= 1 && hq % pages.size(1) == 0 &&
                q.stride(2) == 1 && table.size(0) == b && cu.size(0) == b + 1 && max_q >= 1 && max_q < (1ll << 31) && window >= 0 &&
                window < (1ll << 31)) || !c.here())
      return nullptr;
    Tensor out = at::empty({n, hq, d}, q.options()), lse;
    if (with_lse) lse = at::empty({n, hq}, q.options().dtype(at::kFloat));
    ss_int4_attn_args a = {};
    a.q = q.data_ptr(); a.dtype = code_of(q.scalar_type()); a.q_token_stride = q.stride(0); a.q_head_stride = q.stride(1);
    a.n_tokens = n; a.hq = (int)hq; a.hkv = (int)pages.size(1); a.d = (int)d;
    a.pages = pages.data_ptr(); a.n_pages = (int)pages.size(0); a.page_stride = pages.stride(0); a.head_stride = pages.stride(1);
    a.page_size = (int)page;
    a.block_table = table.data_ptr<int32_t>(); a.table_stride = table.stride(0); a.width = (int)table.size(1);
    a.seq_lens = lens.data_ptr<int32_t>(); a.cu_q = cu.data_ptr<int32_t>(); a.n_requests = (int)b; a.max_q = (int)max_q;
    a.scale = (float)scale; a.causal = causal; a.window = (int)window;
    a.out = out.data_ptr(); a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
    a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
    if (ss_int4_attention(&a, c.stream())) return nullptr;
    return with_lse ? wrap({out, lse}) : wrap({out});
  });
}

// (logits, targets, top_k): (logprobs, entropy, top_ids, top_logprobs)
PyObject* logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return lane(args, nargs, 3, [](Call& c) -> PyObject* {
    const Tensor &x = c.tensor(0), &t = c.tensor(1);
    const int64_t k = c.integer(2);
    c.no_graph(x);
    if (!c.ok || !c.want(x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0 && x.size(1) < (1ll << 31))) return nullptr;
    const int64_t n = x.size(0), vocab = x.size(1);
    const int dt = code_of(x.scalar_type());
    if (!c.want(dt >= 0 && (x.stride(1) == 1 || vocab == 1) && t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == n &&
                t.is_contiguous() && k >= 0 && k <= 32) || !c.here())
      return nullptr;
    Tensor out = at::empty({(2 + k) * n}, x.options().dtype(at::kFloat)), ids = at::empty({n, k}, x.options().dtype(at::kInt));
    float* p = out.data_ptr<float>();
    if (ss_token_logprobs(x.data_ptr(), dt, n, x.stride(0), (int)vocab, t.data_ptr<int64_t>(), (int)k, p, p + n, ids.data_ptr<int32_t>(),
                          p + 2 * n, c.stream()))
      return nullptr;
    return wrap({out.as_strided({n}, {1}, 0), out.as_strided({n}, {1}, n), ids, out.as_strided({n, k}, {k, 1}, 2 * n)});
  });
}

#define SS_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {SS_FAST(plan_step), SS_FAST(append), SS_FAST(fetch), SS_FAST(attention), SS_FAST(logprobs),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast", "Native lane of the paged operators' wrappers.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&kModule); }
