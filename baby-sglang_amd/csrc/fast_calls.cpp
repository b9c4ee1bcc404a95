// The scored attention, eviction and logit calls of _hip.py without their Python: a small call's host time is the time of the call (one
// request's decode 6 us on the GPU, its wrapper 10, 4 this way), and most of it goes into asking a dozen tensors for type, shape, strides and
// address one attribute at a time.  Every function here takes the wrapper's arguments, checks that they are the ordinary case -- tensors
// on the current GPU, of the types and strides that the C entry point takes as they are -- and makes the call; it returns the entry point's
// code, or None for anything else, without having called it: the wrapper then goes on as if it were not there, and raises or
// converts.  A CPython extension over PyTorch's C++ interface; the wrappers work without it.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/bsgl_attn.h"

namespace {

// the C entry points, handed over by _hip.py (this module links against nothing of the library's)
decltype(&bsgl_paged_decode_scored) g_decode;
decltype(&bsgl_decode_scored_workspace_bytes) g_decode_bytes;
decltype(&bsgl_paged_prefill_scored) g_prefill;
decltype(&bsgl_prefill_workspace_bytes) g_prefill_bytes;
decltype(&bsgl_evict_tokens) g_evict;
decltype(&bsgl_evict_workspace_bytes) g_evict_bytes;
decltype(&bsgl_logit_controls) g_logits;

// The call itself, without the interpreter's lock: a launch waits where the stream's queue is full, and other threads (the overlap mode's
// worker among them) go on meanwhile, as they do through ctypes.  The arguments are held by the caller.
template <typename F> PyObject* unlocked(F call) {
  struct Unlocked {  // (taken back whichever way the call is left)
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
  };
  int rc;
  {
    Unlocked u;
    rc = call();
  }
  return PyLong_FromLong(rc);
}

// One call's look at its arguments: `ok` falls when anything is not the ordinary case.
struct Look {
  int index;
  void* stream;
  bool ok;
  Look(PyObject* device, PyObject* stream_handle) : index((int)PyLong_AsLong(device)), stream(PyLong_AsVoidPtr(stream_handle)), ok(PyErr_Occurred() == nullptr) {}
  // the tensor, or NULL for None
  const at::Tensor* optional(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_CheckExact(o)) {
      ok = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.get_device() != index || t.layout() != at::kStrided) {
      ok = false;
      return nullptr;
    }
    return &t;
  }
  const at::Tensor* needed(PyObject* o) {
    const at::Tensor* t = optional(o);
    if (t == nullptr) ok = false;
    return t;
  }
  // a dense vector of n elements
  const void* vector(PyObject* o, at::ScalarType type, int64_t n, bool may_be_none = true) {
    const at::Tensor* t = may_be_none ? optional(o) : needed(o);
    if (t == nullptr) return nullptr;
    if (t->scalar_type() != type || t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1)) ok = false;
    return t->data_ptr();
  }
  // a matrix with dense rows that do not overlap; *stride of a single row: its length
  const at::Tensor* table(PyObject* o, at::ScalarType type, int64_t* stride, bool may_be_none = false) {
    const at::Tensor* t = may_be_none ? optional(o) : needed(o);
    if (t == nullptr) return nullptr;
    if (t->scalar_type() != type || t->dim() != 2 || (t->size(1) > 1 && t->stride(1) != 1) || (t->size(0) > 1 && t->stride(0) < t->size(1))) {
      ok = false;
      return nullptr;
    }
    *stride = t->size(0) > 1 ? t->stride(0) : t->size(1);
    return t;
  }
  int64_t integer(PyObject* o, int64_t lo = INT32_MIN, int64_t hi = INT32_MAX) {
    if (!PyLong_CheckExact(o)) {
      ok = false;
      return 0;
    }
    int over = 0;
    const int64_t v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over != 0 || v < lo || v > hi) ok = false;
    return v;
  }
  double number(PyObject* o) {
    if (PyFloat_CheckExact(o)) return PyFloat_AS_DOUBLE(o);
    if (PyLong_CheckExact(o)) return (double)integer(o);
    ok = false;
    return 0;
  }
};

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return BSGL_DTYPE_BF16;
    case at::kHalf: return BSGL_DTYPE_F16;
    case at::kFloat: return BSGL_DTYPE_F32;
    default: return -1;
  }
}

// [rows, heads, dim], every row dense
bool dense_rows(const at::Tensor& t, int64_t rows, int64_t heads, int64_t dim) {
  return t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == dim && t.stride(2) == 1 && t.stride(1) == dim &&
         (rows <= 1 || t.stride(0) >= heads * dim);
}
// a pair of slabs of q's type that share their strides
bool dense_slabs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t dim) {
  return k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.sizes() == v.sizes() && k.strides() == v.strides() &&
         k.size(0) >= 1 && k.size(2) == dim && k.stride(2) == 1 && k.stride(1) == dim;
}

// index, stream, q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens, scale, logit_cap, slopes, visible_from, visible_to,
// token_weights, token_weights_out, n_splits, variant, out, workspace, max_seq_len, k_new, v_new, out_cache_loc
PyObject* decode_scored(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 23) Py_RETURN_NONE;
  Look k(a[0], a[1]);
  const at::Tensor *q = k.needed(a[2]), *ks = k.needed(a[3]), *vs = k.needed(a[4]), *out = k.needed(a[17]);
  if (!k.ok || q->dim() != 3 || ks->dim() != 3 || vs->dim() != 3 || out->dim() != 2) Py_RETURN_NONE;
  const int64_t batch = q->size(0), hq = q->size(1), dim = q->size(2), hkv = ks->size(1);
  const int code = dtype_code(*q);
  bsgl_decode_call c{};
  bsgl_score_mods m{};
  if (batch < 1 || hq < 1 || dim < 1 || hkv < 1 || batch > INT32_MAX || code < 0 || out->scalar_type() != q->scalar_type()) Py_RETURN_NONE;
  if (!dense_rows(*q, batch, hq, dim) || !dense_slabs(*q, *ks, *vs, dim)) Py_RETURN_NONE;
  if (out->size(0) != batch || out->size(1) != hq * dim || out->stride(1) != 1 || (batch > 1 && out->stride(0) < hq * dim)) Py_RETURN_NONE;
  int64_t table_stride = 0, w_stride = 0, wo_stride = 0;
  const at::Tensor* table = k.table(a[5], at::kInt, &table_stride);
  c.req_pool_indices = (const int64_t*)k.vector(a[6], at::kLong, batch, false);
  c.seq_lens = (const int64_t*)k.vector(a[7], at::kLong, batch, false);
  c.scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)k.number(a[8]);
  const double cap = k.number(a[9]);
  m.slopes = (const float*)k.vector(a[10], at::kFloat, hq);
  m.visible_from = (const int32_t*)k.vector(a[11], at::kInt, batch);
  m.visible_to = (const int32_t*)k.vector(a[12], at::kInt, batch);
  const at::Tensor* w = k.table(a[13], at::kFloat, &w_stride, true);
  const at::Tensor* wo = a[14] == Py_None ? w : k.table(a[14], at::kFloat, &wo_stride, true);
  if (a[14] == Py_None) wo_stride = w_stride;
  c.n_splits = (int32_t)k.integer(a[15], 1, 64);
  c.variant = (int32_t)k.integer(a[16]);
  const at::Tensor* ws = k.optional(a[18]);
  c.max_seq_len = (int32_t)k.integer(a[19]);
  c.stream = k.stream;
  const at::Tensor *kn = k.optional(a[20]), *vn = k.optional(a[21]);
  if (kn != nullptr || vn != nullptr || a[22] != Py_None) {
    if (!k.ok || kn == nullptr || vn == nullptr) Py_RETURN_NONE;
    c.out_cache_loc = (const int32_t*)k.vector(a[22], at::kInt, batch, false);
    for (const at::Tensor* t : {kn, vn})
      if (t->scalar_type() != q->scalar_type() || !dense_rows(*t, batch, hkv, dim)) Py_RETURN_NONE;
    c.k_new = kn->data_ptr();
    c.v_new = vn->data_ptr();
    c.k_new_row_stride = batch > 1 ? kn->stride(0) : hkv * dim;
    c.v_new_row_stride = batch > 1 ? vn->stride(0) : hkv * dim;
  }
  if (!k.ok || table->size(0) < 1 || table->size(1) < 1 || !(cap >= 0.0) || !std::isfinite(cap) || (w == nullptr) != (wo == nullptr)) Py_RETURN_NONE;
  if (w != nullptr && (w->sizes() != table->sizes() || wo->sizes() != table->sizes() || w_stride != wo_stride)) Py_RETURN_NONE;
  const size_t need = g_decode_bytes((int32_t)batch, (int32_t)hq, (int32_t)dim, c.n_splits, 0, table->size(1), w != nullptr);
  if (need > 0) {
    if (ws == nullptr || !ws->is_contiguous() || ws->nbytes() < need) Py_RETURN_NONE;  // (the wrapper makes one)
    c.workspace = ws->data_ptr();
    c.workspace_bytes = ws->nbytes();
  }
  c.out = out->data_ptr();
  c.out_row_stride = batch > 1 ? out->stride(0) : hq * dim;
  c.q = q->data_ptr();
  c.q_row_stride = batch > 1 ? q->stride(0) : hq * dim;
  c.k_slab = ks->data_ptr();
  c.v_slab = vs->data_ptr();
  c.slab_row_stride = ks->stride(0);
  c.n_slots = ks->size(0);
  c.req_to_token = (const int32_t*)table->data_ptr();
  c.table_row_stride = table_stride;
  c.table_rows = table->size(0);
  c.table_cols = table->size(1);
  c.batch = (int32_t)batch;
  c.n_q_heads = (int32_t)hq;
  c.n_kv_heads = (int32_t)hkv;
  c.head_dim = (int32_t)dim;
  c.dtype = c.out_dtype = code;
  m.logit_cap = (float)cap;
  if (w != nullptr) {
    m.token_weights = (const float*)w->data_ptr();
    m.token_weights_out = (float*)wo->data_ptr();
    m.weights_row_stride = w_stride;
  }
  return unlocked([&] { return g_decode(&c, &m); });
}

// index, stream, q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens, prefix_lens, extended_lens, scale, logit_cap, slopes,
// visible_from, visible_to, variant, out, workspace
PyObject* prefill_scored(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 18) Py_RETURN_NONE;
  Look k(a[0], a[1]);
  const at::Tensor *q = k.needed(a[2]), *ks = k.needed(a[3]), *vs = k.needed(a[4]), *rows = k.needed(a[6]), *out = k.needed(a[16]), *ws = k.needed(a[17]);
  if (!k.ok || q->dim() != 3 || ks->dim() != 3 || vs->dim() != 3 || rows->dim() != 1 || out->dim() != 2) Py_RETURN_NONE;
  const int64_t tokens = q->size(0), hq = q->size(1), dim = q->size(2), hkv = ks->size(1), batch = rows->size(0);
  const int code = dtype_code(*q);
  if (tokens < 1 || hq < 1 || dim < 1 || hkv < 1 || batch < 1 || tokens > INT32_MAX || batch > INT32_MAX || code < 0 || out->scalar_type() != q->scalar_type())
    Py_RETURN_NONE;
  if (!dense_rows(*q, tokens, hq, dim) || !dense_slabs(*q, *ks, *vs, dim)) Py_RETURN_NONE;
  if (out->size(0) != tokens || out->size(1) != hq * dim || out->stride(1) != 1 || (tokens > 1 && out->stride(0) < hq * dim)) Py_RETURN_NONE;
  int64_t table_stride = 0;
  const at::Tensor* table = k.table(a[5], at::kInt, &table_stride);
  const void *req = k.vector(a[6], at::kLong, batch, false), *lens = k.vector(a[7], at::kLong, batch, false), *prefix = k.vector(a[8], at::kLong, batch, false),
             *ext = k.vector(a[9], at::kLong, batch, false);
  const float scale = a[10] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)k.number(a[10]);
  const double cap = k.number(a[11]);
  bsgl_score_mods m{};
  m.slopes = (const float*)k.vector(a[12], at::kFloat, hq);
  m.visible_from = (const int32_t*)k.vector(a[13], at::kInt, tokens);
  m.visible_to = (const int32_t*)k.vector(a[14], at::kInt, tokens);
  const int32_t variant = (int32_t)k.integer(a[15]);
  if (!k.ok || table->size(0) < 1 || table->size(1) < 1 || !(cap >= 0.0) || !std::isfinite(cap)) Py_RETURN_NONE;
  m.logit_cap = (float)cap;
  if (!ws->is_contiguous() || ws->nbytes() < g_prefill_bytes((int32_t)batch, (int32_t)tokens, (int32_t)hq, (int32_t)dim)) Py_RETURN_NONE;
  return unlocked([&] {
    return g_prefill(out->data_ptr(), tokens > 1 ? out->stride(0) : hq * dim, q->data_ptr(), tokens > 1 ? q->stride(0) : hq * dim, ks->data_ptr(),
                     vs->data_ptr(), ks->stride(0), ks->size(0), (const int32_t*)table->data_ptr(), table_stride, table->size(0), table->size(1),
                     (const int64_t*)req, (const int64_t*)lens, (const int64_t*)prefix, (const int64_t*)ext, (int32_t)batch, (int32_t)tokens,
                     (int32_t)hq, (int32_t)hkv, (int32_t)dim, scale, code, variant, ws->data_ptr(), ws->nbytes(), &m, k.stream);
  });
}

// index, stream, req_to_token, token_weights, req_pool_indices, seq_lens, budget, recent, sinks, out_table, out_weights, evicted,
// new_lens, max_seq_len
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 14) Py_RETURN_NONE;
  Look k(a[0], a[1]);
  int64_t ts = 0, ws = 0, ots = 0, ows = 0, es = 0;
  const at::Tensor *t = k.table(a[2], at::kInt, &ts), *w = k.table(a[3], at::kFloat, &ws);
  const at::Tensor* rows = k.needed(a[4]);
  if (!k.ok || rows->dim() != 1) Py_RETURN_NONE;
  const int64_t batch = rows->size(0);
  const void* req = k.vector(a[4], at::kLong, batch, false);
  const void* lens = k.vector(a[5], at::kLong, batch, false);
  const int32_t budget = (int32_t)k.integer(a[6]), recent = (int32_t)k.integer(a[7]), sinks = (int32_t)k.integer(a[8]);
  const at::Tensor* ot = a[9] == Py_None ? t : k.table(a[9], at::kInt, &ots);
  const at::Tensor* ow = a[10] == Py_None ? w : k.table(a[10], at::kFloat, &ows);
  if (a[9] == Py_None) ots = ts;
  if (a[10] == Py_None) ows = ws;
  const at::Tensor* ev = k.table(a[11], at::kInt, &es);
  void* nl = (void*)k.vector(a[12], at::kLong, batch, false);
  const int32_t longest = (int32_t)k.integer(a[13]);
  if (!k.ok || batch < 1 || batch > INT32_MAX || t->size(0) < 1 || t->size(1) < 1 || w->sizes() != t->sizes() || ot->sizes() != t->sizes() ||
      ow->sizes() != t->sizes() || ots != ts || ows != ws || ev->size(0) != batch || ev->size(1) > INT32_MAX)
    Py_RETURN_NONE;
  if (g_evict_bytes((int32_t)batch, t->size(1), budget) != 0) Py_RETURN_NONE;  // (long rows: the wrapper sees to the workspace)
  return unlocked([&] {
    return g_evict((int32_t*)ot->data_ptr(), (float*)ow->data_ptr(), (const int32_t*)t->data_ptr(), ts, (const float*)w->data_ptr(), ws, t->size(0),
                   t->size(1), (const int64_t*)req, (const int64_t*)lens, (int64_t*)nl, ev->size(1) > 0 ? (int32_t*)ev->data_ptr() : nullptr, es,
                   (int32_t)ev->size(1), (int32_t)batch, budget, recent, sinks, longest, nullptr, 0, k.stream);
  });
}

// index, stream, logits, history, history_rows, history_lens, prompt_lens, repetition, presence, frequency, bias_ids, bias_values,
// token_mask, mask_rows, out
PyObject* logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15) Py_RETURN_NONE;
  Look k(a[0], a[1]);
  const at::Tensor* x = k.needed(a[2]);
  if (!k.ok || x->dim() != 2) Py_RETURN_NONE;
  bsgl_logit_call c{};
  const int code = dtype_code(*x);
  const at::Tensor* out = k.table(a[14], x->scalar_type(), &c.out_row_stride);
  k.table(a[2], x->scalar_type(), &c.logits_row_stride);
  const int64_t batch = x->size(0), vocab = x->size(1);
  if (!k.ok || code < 0 || batch < 1 || vocab < 1 || batch > INT32_MAX || vocab > INT32_MAX || out->sizes() != x->sizes()) Py_RETURN_NONE;
  const at::Tensor* h = k.table(a[3], at::kInt, &c.history_row_stride, true);
  if (h != nullptr) {
    if (h->size(0) < 1 || h->size(1) < 1) Py_RETURN_NONE;
    c.history = (const int32_t*)h->data_ptr();
    c.history_n_rows = h->size(0);
    c.history_cols = h->size(1);
    c.history_rows = (const int64_t*)k.vector(a[4], at::kLong, batch);
    c.history_lens = (const int64_t*)k.vector(a[5], at::kLong, batch, false);
    c.prompt_lens = (const int64_t*)k.vector(a[6], at::kLong, batch);
    c.repetition = (const float*)k.vector(a[7], at::kFloat, batch);
    c.presence = (const float*)k.vector(a[8], at::kFloat, batch);
    c.frequency = (const float*)k.vector(a[9], at::kFloat, batch);
  } else {
    for (int i = 4; i < 10; ++i) k.ok &= a[i] == Py_None;
  }
  int64_t vals_stride = 0;
  const at::Tensor *ids = k.table(a[10], at::kInt, &c.bias_row_stride, true), *vals = k.table(a[11], at::kFloat, &vals_stride, true);
  if (!k.ok || (ids == nullptr) != (vals == nullptr)) Py_RETURN_NONE;
  if (ids != nullptr) {
    if (ids->sizes() != vals->sizes() || ids->size(0) != batch || c.bias_row_stride != vals_stride || ids->size(1) > INT32_MAX) Py_RETURN_NONE;
    c.bias_ids = (const int32_t*)ids->data_ptr();
    c.bias_values = (const float*)vals->data_ptr();
    c.n_bias = (int32_t)ids->size(1);
  }
  const at::Tensor* mask = k.table(a[12], at::kInt, &c.mask_row_stride, true);
  if (mask != nullptr) {
    c.mask_rows = (const int32_t*)k.vector(a[13], at::kInt, batch);
    if (mask->size(0) < 1 || mask->size(1) < (vocab + 31) / 32 || (c.mask_rows == nullptr && mask->size(0) < batch)) Py_RETURN_NONE;
    c.token_mask = (const int32_t*)mask->data_ptr();
    c.mask_n_rows = mask->size(0);
  } else {
    k.ok &= a[13] == Py_None;
  }
  if (!k.ok) Py_RETURN_NONE;
  c.out = out->data_ptr();
  c.logits = x->data_ptr();
  c.batch = (int32_t)batch;
  c.vocab = (int32_t)vocab;
  c.dtype = code;
  c.stream = k.stream;
  return unlocked([&] { return g_logits(&c); });
}

// no C++ exception leaves a function that Python calls: whatever it was, the wrapper looks again
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    PyObject* r = F(self, a, n);
    if (PyErr_Occurred() == nullptr) return r;
    Py_XDECREF(r);
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// the library's ABI version, the sizes of its descriptors as the wrappers have them, and the addresses of the seven entry points
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const long want[4] = {BSGL_ABI_VERSION, (long)sizeof(bsgl_decode_call), (long)sizeof(bsgl_score_mods), (long)sizeof(bsgl_logit_call)};
  bool same = n == 11;
  for (int i = 0; same && i < 4; ++i) same = PyLong_AsLong(a[i]) == want[i];
  if (!same) {
    if (PyErr_Occurred() == nullptr) PyErr_SetString(PyExc_ImportError, "_fast_calls was built for another version of the library");
    return nullptr;
  }
  a += 4;
  g_decode = (decltype(g_decode))PyLong_AsVoidPtr(a[0]);
  g_decode_bytes = (decltype(g_decode_bytes))PyLong_AsVoidPtr(a[1]);
  g_evict = (decltype(g_evict))PyLong_AsVoidPtr(a[2]);
  g_evict_bytes = (decltype(g_evict_bytes))PyLong_AsVoidPtr(a[3]);
  g_logits = (decltype(g_logits))PyLong_AsVoidPtr(a[4]);
  g_prefill = (decltype(g_prefill))PyLong_AsVoidPtr(a[5]);
  g_prefill_bytes = (decltype(g_prefill_bytes))PyLong_AsVoidPtr(a[6]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {{"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
                           {"decode_scored", (PyCFunction)(void (*)())guarded<decode_scored>, METH_FASTCALL, nullptr},
                           {"prefill_scored", (PyCFunction)(void (*)())guarded<prefill_scored>, METH_FASTCALL, nullptr},
                           {"evict", (PyCFunction)(void (*)())guarded<evict>, METH_FASTCALL, nullptr},
                           {"logits", (PyCFunction)(void (*)())guarded<logits>, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fast_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast_calls() { return PyModule_Create(&g_module); }
