// The serving calls of webgllm_b200.paged and webgllm_b200.speculative as one
// native step: the argument checks on torch's tensors, the outputs and
// workspaces from torch's allocator, and the C entry point on torch's current
// stream. In Python those take 9 to 11 us, several times a small launch; here
// they take one or two. A function here does what its Python namesake does for
// the arguments that are as documented, and returns None for everything else
// (and for a call that the library refused): the Python code then says what is
// wrong, or makes the copy that is needed.
//
// A context whose lock is taken (another thread is between its choice of a
// stream and its call) is left to the Python code, which waits for it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

#include "../../../include/webgllm_decoder.h"
#include "../../../include/webgllm_paged.h"

namespace {

// the library's entry points and webgllm_b200.q4's contexts, by bind()
decltype(&wg_set_stream) set_stream_;
decltype(&wg_paged_rope_kv) rope_kv_;
decltype(&wg_paged_attention) attention_;
decltype(&wg_paged_attention_workspace) attention_workspace_;
decltype(&wg_spec_sample) sample_;
decltype(&wg_spec_sample_workspace) sample_workspace_;
PyObject *contexts_, *s_handle_, *s_lock_, *s_acquire_, *s_release_;

PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long p[6];
  PyObject *contexts;
  if (!PyArg_ParseTuple(args, "O!KKKKKK", &PyDict_Type, &contexts, p, p + 1, p + 2, p + 3, p + 4, p + 5)) return nullptr;
  set_stream_ = reinterpret_cast<decltype(set_stream_)>(p[0]);
  rope_kv_ = reinterpret_cast<decltype(rope_kv_)>(p[1]);
  attention_ = reinterpret_cast<decltype(attention_)>(p[2]);
  attention_workspace_ = reinterpret_cast<decltype(attention_workspace_)>(p[3]);
  sample_ = reinterpret_cast<decltype(sample_)>(p[4]);
  sample_workspace_ = reinterpret_cast<decltype(sample_workspace_)>(p[5]);
  Py_INCREF(contexts);
  Py_XSETREF(contexts_, contexts);
  Py_RETURN_NONE;
}

const at::Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor &t, at::ScalarType type, int device) {
  return t.scalar_type() == type && t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided;
}

// A contiguous tensor of this type, device and shape.
bool is(const at::Tensor *t, at::ScalarType type, int device, at::IntArrayRef shape) {
  return t && on(*t, type, device) && t->sizes() == shape && t->is_contiguous();
}

bool integer(PyObject *o, int &v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long x = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow || x > INT_MAX || x < INT_MIN) return false;
  v = (int)x;
  return true;
}

bool real(PyObject *o, double &v) {
  int whole;
  if (PyFloat_CheckExact(o)) {
    v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!integer(o, whole)) return false;
  v = whole;
  return true;
}

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, (c10::DeviceIndex)device)));
}

// The context of a device, its lock taken; ctx is null if the call is not for
// here (no context yet, another current device, the lock is another thread's).
struct Held {
  wg_ctx *ctx = nullptr;
  PyObject *owner = nullptr, *lock = nullptr;  // kept while other threads run
  void *stream = nullptr;

  explicit Held(int device) {
    if (!contexts_ || c10::cuda::current_device() != device) return;
    const cudaStream_t s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    stream = s ? s : cudaStreamLegacy;
    PyObject *key = PyLong_FromLong(device);
    PyObject *c = key ? PyDict_GetItemWithError(contexts_, key) : nullptr;  // borrowed
    Py_XDECREF(key);
    PyObject *mine = c ? PyObject_GetAttr(c, s_lock_) : nullptr;
    PyObject *got = mine ? PyObject_CallMethodOneArg(mine, s_acquire_, Py_False) : nullptr;
    if (got == Py_True) {
      lock = mine;
      owner = Py_NewRef(c);
      PyObject *h = PyObject_GetAttr(c, s_handle_);
      if (h && h != Py_None) ctx = static_cast<wg_ctx *>(PyLong_AsVoidPtr(h));
      Py_XDECREF(h);
    } else {
      Py_XDECREF(mine);
    }
    Py_XDECREF(got);
    PyErr_Clear();
  }
  ~Held() {
    if (!lock) return;
    PyObject *r = PyObject_CallMethodNoArgs(lock, s_release_);
    Py_XDECREF(r);
    Py_DECREF(lock);
    Py_DECREF(owner);
  }
  Held(const Held &) = delete;
  Held &operator=(const Held &) = delete;

  // fn on torch's current stream, other Python threads running meanwhile
  template <typename F, typename... A>
  int call(F fn, A... args) const {
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = set_stream_(ctx, stream);
    if (!status) status = fn(ctx, args...);
    Py_END_ALLOW_THREADS;
    return status;
  }
};

// Pages and table as the C entry points take them.
bool cache(const at::Tensor *k, const at::Tensor *v, const at::Tensor *table, int64_t batch, int device,
           wg_paged_kv &kv) {
  const at::ScalarType type = k->scalar_type();
  if (k->dim() != 4 || (type != at::kHalf && type != at::kBFloat16) || !on(*k, type, device) || !v ||
      !on(*v, type, device) || v->sizes() != k->sizes() || v->strides() != k->strides())
    return false;
  if (!table || table->dim() != 2 || !is(table, at::kInt, device, {batch, table->size(1)})) return false;
  for (int i = 0; i < 3; i++)
    if (k->stride(i) <= 0 || k->stride(i) % 8 || k->size(i) > INT_MAX) return false;
  if (k->stride(3) != 1 || k->size(3) > INT_MAX || table->size(1) > INT_MAX) return false;
  kv = wg_paged_kv{k->data_ptr(), v->data_ptr(), static_cast<const int32_t *>(table->data_ptr()),
                   type == at::kHalf ? WG_F16 : WG_BF16, (int)k->size(0), (int)k->size(2), (int)table->size(1),
                   k->stride(0), k->stride(1), k->stride(2)};
  return true;
}

// attention_paged(q, pos, k, v, table, window, sinks, row_start, out, workspace)
PyObject *attention_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 10) Py_RETURN_NONE;
  try {
    const at::Tensor *q = tensor(a[0]), *pos = tensor(a[1]), *k = tensor(a[2]), *v = tensor(a[3]), *table = tensor(a[4]);
    int window, sinks;
    if (!q || !pos || !k || !k->is_cuda() || !integer(a[5], window) || !integer(a[6], sinks)) Py_RETURN_NONE;
    const int device = k->get_device();
    const int64_t batch = pos->numel();
    wg_paged_kv kv;
    if (!is(pos, at::kInt, device, {batch}) || batch > INT_MAX || !cache(k, v, table, batch, device, kv))
      Py_RETURN_NONE;
    const int64_t hkv = k->size(1), dim = k->size(3);
    if (q->dim() != 3 || q->size(2) != dim || hkv <= 0 || q->size(1) % hkv || q->size(0) > INT_MAX ||
        q->size(1) > INT_MAX || !is(q, k->scalar_type(), device, q->sizes()))
      Py_RETURN_NONE;
    const int32_t *starts = nullptr;
    if (a[7] != Py_None) {
      const at::Tensor *t = tensor(a[7]);
      if (!is(t, at::kInt, device, {batch + 1})) Py_RETURN_NONE;
      starts = static_cast<const int32_t *>(t->data_ptr());
    }
    const at::Tensor *given = nullptr, *ws_given = nullptr;
    if (a[8] != Py_None && !is(given = tensor(a[8]), q->scalar_type(), device, q->sizes())) Py_RETURN_NONE;
    if (a[9] != Py_None) {
      ws_given = tensor(a[9]);
      if (!ws_given || !ws_given->is_cuda() || ws_given->get_device() != device || !ws_given->is_contiguous())
        Py_RETURN_NONE;
    }
    const Held held(device);
    size_t bytes;
    if (!held.ctx || attention_workspace_(held.ctx, (int)dim, &bytes)) Py_RETURN_NONE;
    const at::Tensor out = given ? *given : make(q->sizes(), q->scalar_type(), device);
    const at::Tensor ws = ws_given ? *ws_given : make({(int64_t)bytes}, at::kByte, device);
    if (held.call(attention_, q->data_ptr(), (int)q->size(0), (int)batch, starts, (int)q->size(1), (int)hkv, (int)dim,
                   static_cast<const int32_t *>(pos->data_ptr()), &kv, window, sinks, out.data_ptr(), ws.data_ptr(),
                   ws.nbytes()))
      Py_RETURN_NONE;
    if (given) return Py_NewRef(a[8]);
    return THPVariable_Wrap(out);
  } catch (...) {  // (out of memory: the Python code meets it too)
    Py_RETURN_NONE;
  }
}

// rope_kv_paged(qkv, pos, k, v, table, heads, theta, q_norm, k_norm, eps, row_start, out)
PyObject *rope_kv_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 12) Py_RETURN_NONE;
  try {
    const at::Tensor *qkv = tensor(a[0]), *pos = tensor(a[1]), *k = tensor(a[2]), *v = tensor(a[3]),
                     *table = tensor(a[4]);
    int heads;
    double theta, eps;
    if (!qkv || !pos || !k || !k->is_cuda() || !integer(a[5], heads) || !real(a[6], theta) || !real(a[9], eps))
      Py_RETURN_NONE;
    const int device = k->get_device();
    const int64_t batch = pos->numel();
    wg_paged_kv kv;
    if (!is(pos, at::kInt, device, {batch}) || batch > INT_MAX || !cache(k, v, table, batch, device, kv))
      Py_RETURN_NONE;
    const int64_t hkv = k->size(1), dim = k->size(3), rows = qkv->dim() == 2 ? qkv->size(0) : 0;
    if (heads <= 0 || rows > INT_MAX || !is(qkv, at::kFloat, device, {rows, (heads + 2 * hkv) * dim})) Py_RETURN_NONE;
    const float *norm[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; i++)
      if (a[7 + i] != Py_None) {
        const at::Tensor *t = tensor(a[7 + i]);
        if (!is(t, at::kFloat, device, {dim})) Py_RETURN_NONE;
        norm[i] = static_cast<const float *>(t->data_ptr());
      }
    const int32_t *starts = nullptr;
    if (a[10] != Py_None) {
      const at::Tensor *t = tensor(a[10]);
      if (!is(t, at::kInt, device, {batch + 1})) Py_RETURN_NONE;
      starts = static_cast<const int32_t *>(t->data_ptr());
    }
    const at::Tensor *given = nullptr;
    if (a[11] != Py_None && !is(given = tensor(a[11]), k->scalar_type(), device, {rows, heads, dim})) Py_RETURN_NONE;
    const Held held(device);
    if (!held.ctx) Py_RETURN_NONE;
    const at::Tensor out = given ? *given : make({rows, heads, dim}, k->scalar_type(), device);
    if (held.call(rope_kv_, static_cast<const float *>(qkv->data_ptr()), (int)rows, (int)batch, starts, heads, (int)hkv,
                 (int)dim, static_cast<const int32_t *>(pos->data_ptr()), theta, norm[0], norm[1], (float)eps,
                 out.data_ptr(), &kv))
      Py_RETURN_NONE;
    if (given) return Py_NewRef(a[11]);
    return THPVariable_Wrap(out);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// spec_sample(target, draft, drafts, u, temperature, out)
PyObject *spec_sample(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 6) Py_RETURN_NONE;
  try {
    const at::Tensor *target = tensor(a[0]), *u = tensor(a[3]);
    double temperature;
    if (!target || !target->is_cuda() || !real(a[4], temperature)) Py_RETURN_NONE;
    const int device = target->get_device();
    const bool flat = target->dim() == 2 && a[1] == Py_None;
    if ((!flat && target->dim() != 3) || !is(target, at::kFloat, device, target->sizes())) Py_RETURN_NONE;
    const int64_t rows = flat ? 1 : target->size(0), batch = target->size(flat ? 0 : 1), V = target->size(flat ? 1 : 2);
    const int64_t k = rows - 1;
    if (k < 0 || rows > INT_MAX || batch > INT_MAX || V > INT_MAX || (a[1] == Py_None) != (k == 0) ||
        (a[2] == Py_None) != (k == 0) || !is(u, at::kFloat, device, {batch, rows}))
      Py_RETURN_NONE;
    const float *draft = nullptr;
    const int32_t *drafts = nullptr;
    if (k) {
      const at::Tensor *x = tensor(a[1]), *d = tensor(a[2]);
      if (!is(x, at::kFloat, device, {k, batch, V}) || !is(d, at::kInt, device, {batch, k})) Py_RETURN_NONE;
      draft = static_cast<const float *>(x->data_ptr());
      drafts = static_cast<const int32_t *>(d->data_ptr());
    }
    const at::Tensor *given = nullptr;
    if (a[5] != Py_None && !is(given = tensor(a[5]), at::kInt, device, {rows, batch})) Py_RETURN_NONE;
    const Held held(device);
    size_t bytes;
    if (!held.ctx || sample_workspace_(held.ctx, (int)batch, (int)k, (int)V, &bytes)) Py_RETURN_NONE;
    const at::Tensor out = given ? *given : make({rows, batch}, at::kInt, device);
    const at::Tensor ws = make({(int64_t)(bytes > 8 ? bytes : 8)}, at::kByte, device);
    if (held.call(sample_, static_cast<const float *>(target->data_ptr()), draft, drafts, (int)batch, (int)k, (int)V,
                temperature, static_cast<const float *>(u->data_ptr()), static_cast<int32_t *>(out.data_ptr()),
                ws.data_ptr(), ws.nbytes()))
      Py_RETURN_NONE;
    if (given) return Py_NewRef(a[5]);
    return THPVariable_Wrap(out);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"attention_paged", (PyCFunction)(void (*)(void))attention_paged, METH_FASTCALL, nullptr},
    {"rope_kv_paged", (PyCFunction)(void (*)(void))rope_kv_paged, METH_FASTCALL, nullptr},
    {"spec_sample", (PyCFunction)(void (*)(void))spec_sample, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  s_handle_ = PyUnicode_InternFromString("handle");
  s_lock_ = PyUnicode_InternFromString("lock");
  s_acquire_ = PyUnicode_InternFromString("acquire");
  s_release_ = PyUnicode_InternFromString("release");
  if (!s_handle_ || !s_lock_ || !s_acquire_ || !s_release_) return nullptr;
  PyObject *m = PyModule_Create(&module);
  // read before bind() by whoever imports this: another torch lays tensors out otherwise
  if (m && PyModule_AddStringConstant(m, "built_for", WG_HOST_TARGET) < 0) Py_CLEAR(m);
  return m;
}
