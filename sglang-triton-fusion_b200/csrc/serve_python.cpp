// The serving operators' direct Python binding.  A decode step calls them once
// per layer, and reading a dozen tensors' properties one by one from Python costs
// more than the kernels take; here it is done in C++.
//
// Each function takes the arguments of its namesake in fp8gq/serve.py in order
// (positional) and returns what that returns if they are all in the form that it
// expects, and None otherwise: serve.py then goes through its own checks, which
// raise or complete the call through the same C entry point.  So nothing is
// refused or accepted here that is not there.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>

#include "../../include/fp8gq.h"

namespace {

PyObject* g_workspaces = nullptr;      // fp8gq.ops' scratch: (device, stream) -> (tensor, address, bytes)

PyObject* not_here() { Py_RETURN_NONE; }

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// A CUDA tensor of the given device (or any, setting it), type and rank.
const at::Tensor* cuda_tensor(PyObject* o, at::ScalarType type, int64_t dim, int* device) {
  const at::Tensor* t = tensor(o);
  if (!t || !t->is_cuda() || t->scalar_type() != type || t->dim() != dim) return nullptr;
  const int d = t->get_device();
  if (*device < 0) *device = d;
  return d == *device ? t : nullptr;
}

// A contiguous vector of n values.
const at::Tensor* vector(PyObject* o, at::ScalarType type, int64_t n, int* device) {
  const at::Tensor* t = cuda_tensor(o, type, 1, device);
  return t && t->size(0) == n && t->is_contiguous() ? t : nullptr;
}

bool number(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *v = PyLong_AsDouble(o);
  else return false;
  return !PyErr_Occurred();
}

// Whether the C entry points' int holds them.
bool fits(std::initializer_list<int64_t> ns) {
  for (int64_t n : ns)
    if (n > INT32_MAX) return false;
  return true;
}

// The cache of two tensors [pages, page_size, heads, D].
bool paged_cache(PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso, int* device, fp8gq_paged_cache* c) {
  const at::Tensor *k = tensor(ko), *v = tensor(vo);
  if (!k || !v || !k->is_cuda() || !v->is_cuda() || k->dim() != 4 || v->dim() != 4 || k->scalar_type() != v->scalar_type() ||
      k->sizes() != v->sizes())
    return false;
  if (k->scalar_type() != at::kBFloat16 && k->scalar_type() != at::kFloat8_e4m3fn) return false;
  const int d = k->get_device();
  if (*device < 0) *device = d;
  if (d != *device || v->get_device() != d || k->stride(3) != 1 || v->stride(3) != 1 || !fits({k->size(1)})) return false;
  double ks, vs;
  if (!number(kso, &ks) || !number(vso, &vs)) return false;
  *c = {k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), k->stride(2), v->stride(0), v->stride(1), v->stride(2),
        k->size(0), static_cast<int>(k->size(1)), k->scalar_type() == at::kBFloat16 ? FP8GQ_DTYPE_BF16 : FP8GQ_DTYPE_E4M3,
        static_cast<float>(ks), static_cast<float>(vs)};
  return true;
}

// The scratch that fp8gq.ops keeps for this device and stream, if it is there.
bool workspace(int device, cudaStream_t stream, size_t bytes, void** p, size_t* n) {
  PyObject* key = Py_BuildValue("(iK)", device, reinterpret_cast<unsigned long long>(stream));
  if (!key) return false;
  PyObject* e = PyDict_GetItem(g_workspaces, key);       // borrowed
  Py_DECREF(key);
  if (!e || !PyTuple_Check(e) || PyTuple_GET_SIZE(e) != 3) return false;
  *p = PyLong_AsVoidPtr(PyTuple_GET_ITEM(e, 1));
  *n = PyLong_AsSize_t(PyTuple_GET_ITEM(e, 2));
  return !PyErr_Occurred() && *n >= bytes;
}

// A flag, True or False; anything else counts by its truth in serve.py.
bool flag(PyObject* o, bool* v) {
  *v = o == Py_True;
  return PyBool_Check(o);
}

at::Tensor empty(c10::IntArrayRef sizes, at::ScalarType type, int device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device))));
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(const at::Tensor& a, const at::Tensor& b) { return Py_BuildValue("(NN)", wrap(a), wrap(b)); }

// This device's stream; false if another device is current (the C entry points
// launch on the current one).
bool stream_of(int device, cudaStream_t* s) {
  if (c10::cuda::current_device() != device) return false;
  *s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  return true;
}

// Nothing thrown below leaves the module: a call that meets an exception goes
// back to serve.py.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    PyObject* r = f();
    if (r == Py_None) PyErr_Clear();
    return r;
  } catch (...) {
    PyErr_Clear();
    return not_here();
  }
}

PyObject* qk_norm_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  // qkv, positions, slots, cos_sin, k_cache, v_cache, q_weight, k_weight, eps, k_scale, v_scale, return_k
  return guarded([&]() -> PyObject* {
    if (n != 12) return not_here();
    int dev = -1;
    fp8gq_paged_cache c;
    const at::Tensor* qkv = cuda_tensor(a[0], at::kBFloat16, 2, &dev);
    if (!qkv || qkv->stride(1) != 1 || !paged_cache(a[4], a[5], a[9], a[10], &dev, &c)) return not_here();
    const at::Tensor& k = THPVariable_Unpack(a[4]);
    const int64_t t = qkv->size(0), d = k.size(3), hkv = k.size(2);
    if (d != 64 && d != 128) return not_here();
    const int64_t hq = qkv->size(1) / d - 2 * hkv;
    if (qkv->size(1) % d || hkv < 1 || hq < 1 || hq % hkv || !fits({t, hq, hkv})) return not_here();
    const at::Tensor *pos = vector(a[1], at::kLong, t, &dev), *slots = vector(a[2], at::kLong, t, &dev);
    const at::Tensor* cs = cuda_tensor(a[3], at::kFloat, 2, &dev);
    if (!pos || !slots || !cs || cs->size(1) != d || !cs->is_contiguous()) return not_here();
    const at::Tensor *qw = nullptr, *kw = nullptr;
    if (a[6] != Py_None && !(qw = vector(a[6], at::kBFloat16, d, &dev))) return not_here();
    if (a[7] != Py_None && !(kw = vector(a[7], at::kBFloat16, d, &dev))) return not_here();
    double eps;
    bool want_k;
    cudaStream_t stream;
    if (!number(a[8], &eps) || !flag(a[11], &want_k) || !stream_of(dev, &stream)) return not_here();
    const at::Tensor q = empty({t, hq, d}, at::kBFloat16, dev);
    const at::Tensor ko = want_k ? empty({t, hkv, d}, at::kBFloat16, dev) : at::Tensor();
    if (fp8gq_qk_norm_rope_append(qkv->data_ptr(), qkv->stride(0), pos->data_ptr<int64_t>(), slots->data_ptr<int64_t>(),
                                  cs->data_ptr<float>(), cs->size(0), qw ? qw->data_ptr() : nullptr,
                                  kw ? kw->data_ptr() : nullptr, static_cast<float>(eps), q.data_ptr(), hq * d,
                                  want_k ? ko.data_ptr() : nullptr, hkv * d, &c, static_cast<int>(t), static_cast<int>(hq),
                                  static_cast<int>(hkv), static_cast<int>(d), stream) != FP8GQ_OK)
      return not_here();
    return want_k ? pair(q, ko) : wrap(q);
  });
}

PyObject* paged_decode_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  // q, k_cache, v_cache, page_table, lens, scale, k_scale, v_scale, return_lse
  return guarded([&]() -> PyObject* {
    if (n != 9) return not_here();
    int dev = -1;
    fp8gq_paged_cache c;
    const at::Tensor* q = cuda_tensor(a[0], at::kBFloat16, 3, &dev);
    if (!q || q->stride(2) != 1 || !paged_cache(a[1], a[2], a[6], a[7], &dev, &c)) return not_here();
    const at::Tensor& k = THPVariable_Unpack(a[1]);
    const int64_t b = q->size(0), hq = q->size(1), d = q->size(2), hkv = k.size(2);
    if (k.size(3) != d || (d != 64 && d != 128) || hkv < 1 || hq < 1 || hq % hkv || !fits({b, hq, hkv})) return not_here();
    const at::Tensor *table = cuda_tensor(a[3], at::kInt, 2, &dev), *lens = vector(a[4], at::kInt, b, &dev);
    if (!table || !lens || table->size(0) != b || (table->size(1) > 1 && table->stride(1) != 1) || !fits({table->size(1)}))
      return not_here();
    double scale = 1.0 / std::sqrt(static_cast<double>(d));
    bool want_lse;
    if ((a[5] != Py_None && !number(a[5], &scale)) || !flag(a[8], &want_lse)) return not_here();
    cudaStream_t stream;
    void* ws;
    size_t ws_n;
    if (!stream_of(dev, &stream)) return not_here();
    const size_t need = fp8gq_paged_decode_workspace_bytes(static_cast<int>(hq), static_cast<int>(hkv), static_cast<int>(d));
    if (!workspace(dev, stream, need, &ws, &ws_n)) return not_here();
    const at::Tensor out = empty({b, hq, d}, at::kBFloat16, dev);
    const at::Tensor lse = want_lse ? empty({b, hq}, at::kFloat, dev) : at::Tensor();
    if (fp8gq_paged_decode_attention(q->data_ptr(), q->stride(0), q->stride(1), &c, table->data_ptr<int32_t>(),
                                     table->stride(0), static_cast<int>(table->size(1)), lens->data_ptr<int32_t>(),
                                     out.data_ptr(), hq * d, d, want_lse ? lse.data_ptr<float>() : nullptr,
                                     static_cast<int>(b), static_cast<int>(hq), static_cast<int>(hkv), static_cast<int>(d),
                                     static_cast<float>(scale), ws, ws_n, stream) != FP8GQ_OK)
      return not_here();
    return want_lse ? pair(out, lse) : wrap(out);
  });
}

PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  // q, k, v, cu_q, cu_k, causal, scale, return_lse
  return guarded([&]() -> PyObject* {
    if (n != 8) return not_here();
    int dev = -1;
    const at::Tensor *q = cuda_tensor(a[0], at::kBFloat16, 3, &dev), *k = cuda_tensor(a[1], at::kBFloat16, 3, &dev),
                     *v = cuda_tensor(a[2], at::kBFloat16, 3, &dev);
    if (!q || !k || !v || q->stride(2) != 1 || k->stride(2) != 1 || v->stride(2) != 1 || k->sizes() != v->sizes())
      return not_here();
    const int64_t tq = q->size(0), hq = q->size(1), d = q->size(2), tk = k->size(0), hkv = k->size(1);
    if (k->size(2) != d || (d != 64 && d != 128) || hkv < 1 || hq < 1 || hq % hkv || !fits({tq, tk, hq, hkv}))
      return not_here();
    const at::Tensor* cq = cuda_tensor(a[3], at::kInt, 1, &dev);
    if (!cq || cq->size(0) < 1 || !cq->is_contiguous() || !fits({cq->size(0)})) return not_here();
    const at::Tensor* ck = a[4] == Py_None ? cq : vector(a[4], at::kInt, cq->size(0), &dev);
    double scale = 1.0 / std::sqrt(static_cast<double>(d));
    bool causal, want_lse;
    if (!ck || !flag(a[5], &causal) || !flag(a[7], &want_lse) || (a[6] != Py_None && !number(a[6], &scale))) return not_here();
    cudaStream_t stream;
    void* ws;
    size_t ws_n;
    if (!stream_of(dev, &stream)) return not_here();
    // a split call's scratch is its own: another thread's launch may come between its two
    at::Tensor own;
    ws_n = fp8gq_prompt_split_bytes(static_cast<int>(cq->size(0) - 1), static_cast<int>(tq), static_cast<int>(tk),
                                    static_cast<int>(hq), static_cast<int>(hkv), static_cast<int>(d), causal);
    if (ws_n) {
      own = empty({static_cast<int64_t>(ws_n)}, at::kByte, dev);
      ws = own.data_ptr();
    } else if (!workspace(dev, stream, FP8GQ_PROMPT_COUNTER_BYTES, &ws, &ws_n)) {
      return not_here();
    }
    const at::Tensor out = empty({tq, hq, d}, at::kBFloat16, dev);
    const at::Tensor lse = want_lse ? empty({tq, hq}, at::kFloat, dev) : at::Tensor();
    if (fp8gq_prompt_attention(q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1),
                               v->data_ptr(), v->stride(0), v->stride(1), out.data_ptr(), hq * d, d,
                               want_lse ? lse.data_ptr<float>() : nullptr, cq->data_ptr<int32_t>(), ck->data_ptr<int32_t>(),
                               static_cast<int>(cq->size(0) - 1), static_cast<int>(tq), static_cast<int>(tk),
                               static_cast<int>(hq), static_cast<int>(hkv), static_cast<int>(d), static_cast<float>(scale),
                               causal, ws, ws_n, stream) != FP8GQ_OK)
      return not_here();
    return want_lse ? pair(out, lse) : wrap(out);
  });
}

PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  // logits, tokens, top_k -> (logprobs, entropy, top_ids, top_logprobs)
  return guarded([&]() -> PyObject* {
    if (n != 3) return not_here();
    const at::Tensor* x = tensor(a[0]);
    if (!x || !x->is_cuda() || x->dim() != 2 || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kFloat))
      return not_here();
    int dev = x->get_device();
    const int64_t t = x->size(0), v = x->size(1);
    if (v < 1 || (v > 1 && x->stride(1) != 1) || !fits({t, v}) || !PyLong_CheckExact(a[2])) return not_here();
    const long k = PyLong_AsLong(a[2]);
    if (k < 0 || k > 32 || k > v) return not_here();
    const at::Tensor* tok = nullptr;
    if (a[1] != Py_None && !(tok = vector(a[1], at::kLong, t, &dev))) return not_here();
    cudaStream_t stream;
    if (!stream_of(dev, &stream)) return not_here();
    const at::Tensor lp = tok ? empty({t}, at::kFloat, dev) : at::Tensor(), ent = empty({t}, at::kFloat, dev),
                     ids = empty({t, k}, at::kLong, dev), tops = empty({t, k}, at::kFloat, dev);
    if (fp8gq_token_logprobs(x->data_ptr(), x->stride(0), x->scalar_type() == at::kBFloat16 ? FP8GQ_DTYPE_BF16 : FP8GQ_DTYPE_F32,
                             tok ? tok->data_ptr<int64_t>() : nullptr, static_cast<int>(t), static_cast<int>(v),
                             tok ? lp.data_ptr<float>() : nullptr, ent.data_ptr<float>(), ids.data_ptr<int64_t>(),
                             tops.data_ptr<float>(), static_cast<int>(k), stream) != FP8GQ_OK)
      return not_here();
    PyObject* first = tok ? wrap(lp) : Py_NewRef(Py_None);
    return Py_BuildValue("(NNNN)", first, wrap(ent), wrap(ids), wrap(tops));
  });
}

PyObject* set_workspaces(PyObject*, PyObject* dict) {
  if (!PyDict_Check(dict)) {
    PyErr_SetString(PyExc_TypeError, "a dict is expected");
    return nullptr;
  }
  Py_XSETREF(g_workspaces, Py_NewRef(dict));
  Py_RETURN_NONE;
}

#define FP8GQ_FAST(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {FP8GQ_FAST(qk_norm_rope_append), FP8GQ_FAST(paged_decode_attention), FP8GQ_FAST(prompt_attention),
                         FP8GQ_FAST(token_logprobs), {"set_workspaces", set_workspaces, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve_native(void) { return PyModule_Create(&module); }
