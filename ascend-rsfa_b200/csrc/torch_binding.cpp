// The ordinary calls of attention() and of the operators around it (rotary.py, kv_cache.py) from PyTorch in native code:
// check the tensors, allocate the results and the scratch, find the current stream, call the library.  attention():
// the same steps in Python (flash_attention_forward.py, _forward) take 10 us of the host's time per call, three times what
// the launch itself takes, which is what a call of a few heads or of a short sequence costs its caller; here they take
// about 1.5 us.
//
// A function here answers only for the ordinary case and returns None for everything else - tensors to copy first,
// empty ones, another device than the current one, subclasses, dispatch or function modes, transforms,
// tracing, argument types other than the plain ones, anything to refuse - and the Python code decides then.
// So nothing is accepted, refused or seen by a mode differently than without this file.
#include <Python.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <string>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/rsfa.h"

namespace {

// rsfa_fwd of the library that the Python side has loaded (bind() hands its address over).
using FwdFn = decltype(&rsfa_fwd);
FwdFn g_fwd = nullptr;

bool plain_mode() {
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerBackMode) &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Functionalize) &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer) &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::VmapMode);
}

// A dense CUDA tensor that rsfa_fwd can take as it is: unit innermost stride, the others multiples of eight
// elements, a 16-byte aligned base.
bool plain_tensor(PyObject* obj) {
  if (!THPVariable_CheckExact(obj)) return false;
  const at::Tensor& t = THPVariable_Unpack(obj);
  const c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                     c10::DispatchKey::Batched, c10::DispatchKey::Functionalize, c10::DispatchKey::Negative,
                                     c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor, c10::DispatchKey::Python});
  if (!t.defined() || t.key_set().has_any(wrapped) || t.layout() != c10::kStrided || !t.is_cuda() || t.dim() != 4 ||
      !t.has_storage())
    return false;
  if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16) return false;
  const int64_t D = t.size(3);
  if (t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) % 8 != 0 || t.stride(i) < D)) return false;
  return true;
}

bool plain_int(PyObject* obj, int* out) {
  if (!PyLong_CheckExact(obj)) return false;
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(obj, &overflow);
  if (overflow != 0 || v < INT32_MIN || v > INT32_MAX) return false;
  *out = static_cast<int>(v);
  return true;
}

// forward(q, k, v, causal, sm_scale, block_m, block_n, want_lse) -> (o, lse or None), an error code of
// rsfa_fwd (int), or None where this is not the ordinary case.
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int block_m = 0, block_n = 0;
  if (g_fwd == nullptr || n != 8 || !plain_mode() || !plain_tensor(args[0]) || !plain_tensor(args[1]) ||
      !plain_tensor(args[2]) || !PyBool_Check(args[3]) || !PyFloat_CheckExact(args[4]) || !plain_int(args[5], &block_m) ||
      !plain_int(args[6], &block_n) || !PyBool_Check(args[7]))
    Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  const int64_t D = q.size(3);
  if (!(D == 16 || D == 32 || D == 64 || D == 128 || D == 256) || q.sizes() != k.sizes() || q.sizes() != v.sizes() ||
      q.numel() == 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.device() != q.device() || v.device() != q.device() || q.device().index() != c10::cuda::current_device() ||
      q.size(0) > INT32_MAX || q.size(1) > INT32_MAX || q.size(2) > INT32_MAX)
    Py_RETURN_NONE;

  at::Tensor o = at::empty_like(q);
  bool fits = o.stride(3) == 1;
  for (int i = 0; i < 3; ++i) fits = fits && (o.size(i) == 1 || o.stride(i) % 8 == 0);
  if (!fits) o = at::empty(q.sizes(), q.options());
  at::Tensor lse;
  if (args[7] == Py_True) lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));

  int64_t strides[16];
  const at::Tensor* all[4] = {&q, &k, &v, &o};
  for (int t = 0; t < 4; ++t)
    for (int i = 0; i < 4; ++i) strides[4 * t + i] = all[t]->stride(i);
  const void* qp = q.const_data_ptr();
  const void* kp = k.const_data_ptr();
  const void* vp = v.const_data_ptr();
  void* op = o.mutable_data_ptr();
  float* lp = lse.defined() ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr;
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const float scale = static_cast<float>(PyFloat_AS_DOUBLE(args[4]));
  const int dtype = q.scalar_type() == at::kBFloat16 ? RSFA_DTYPE_BF16 : RSFA_DTYPE_F16;
  const int B = static_cast<int>(q.size(0)), H = static_cast<int>(q.size(1)), S = static_cast<int>(q.size(2));
  const int causal = args[3] == Py_True ? 1 : 0;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS   // as ctypes does: a launch can block while the device's queue is full
  rc = g_fwd(qp, kp, vp, op, lp, B, H, S, static_cast<int>(D), strides, causal, scale, block_m, block_n, dtype, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject* po = THPVariable_Wrap(std::move(o));
  if (po == nullptr) return nullptr;
  PyObject* pl = Py_None;
  if (lse.defined()) {
    pl = THPVariable_Wrap(std::move(lse));
    if (pl == nullptr) {
      Py_DECREF(po);
      return nullptr;
    }
  } else {
    Py_INCREF(pl);
  }
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) {
    Py_DECREF(po);
    Py_DECREF(pl);
    return nullptr;
  }
  PyTuple_SET_ITEM(pair, 0, po);
  PyTuple_SET_ITEM(pair, 1, pl);
  return pair;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- the operators around attention
// The same bargain: None for whatever is not the ordinary call, and rotary.py and kv_cache.py decide.
struct Ops {
  decltype(&rsfa_rotary) rotary = nullptr;
  decltype(&rsfa_cache4_append) append = nullptr;
  decltype(&rsfa_cache4_read) read = nullptr;
  decltype(&rsfa_cache4_attention_workspace) attention_workspace = nullptr;
  decltype(&rsfa_cache4_attention) attention = nullptr;
  decltype(&rsfa_cache4_evict_workspace) evict_workspace = nullptr;
  decltype(&rsfa_cache4_evict) evict = nullptr;
  decltype(&rsfa_strerror) strerror = nullptr;
} g_ops;

// Raises what _capi.check() raises for a code of the library, where there is no Python caller to hand it to.
void check_code(int rc, const char* what) {
  if (rc == RSFA_OK) return;
  const std::string message = std::string(what) + " failed: " + g_ops.strerror(rc) + " (code " + std::to_string(rc) + ")";
  TORCH_CHECK_VALUE(rc != RSFA_ERR_INVALID_ARGUMENT && rc != RSFA_ERR_TOO_LARGE, message);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != RSFA_ERR_UNSUPPORTED, message);
  TORCH_CHECK(false, message);
}

// The current device, if the tensor lives on it; -1: it does not (there may be no device at all).
int device_of(PyObject* obj) {
  if (!THPVariable_CheckExact(obj)) return -1;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.defined() || !t.is_cuda()) return -1;
  const int device = c10::cuda::current_device();
  return t.device().index() == device ? device : -1;
}
// A plain CUDA tensor of `type` with `dims` dimensions on the current device; null: something else.
const at::Tensor* plain_cuda(PyObject* obj, at::ScalarType type, int64_t dims, int device) {
  if (!THPVariable_CheckExact(obj)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  const c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                     c10::DispatchKey::Batched, c10::DispatchKey::Functionalize, c10::DispatchKey::Negative,
                                     c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor, c10::DispatchKey::Python});
  if (!t.defined() || t.key_set().has_any(wrapped) || t.layout() != c10::kStrided || !t.is_cuda() || t.dim() != dims ||
      !t.has_storage() || t.scalar_type() != type || t.device().index() != device)
    return nullptr;
  return &t;
}
// The tangent that a tensor has in forward-mode differentiation; undefined: none.
at::Tensor tangent_of(const at::Tensor& t) { return t.defined() && t.unsafeGetTensorImpl()->autograd_meta() != nullptr ? t._fw_grad(0) : at::Tensor(); }
// The same for [B, H, S, D] rows that the library reads as they are (plain_tensor) and that are not empty.
const at::Tensor* plain_rows(PyObject* obj, int device) {
  if (!plain_tensor(obj)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (tangent_of(t).defined()) return nullptr;
  if (t.device().index() != device || t.numel() == 0 || t.size(0) > INT32_MAX || t.size(1) > INT32_MAX || t.size(2) > INT32_MAX) return nullptr;
  return &t;
}
bool records_grad(const at::Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }
// An output like t whose rows the library can write.
at::Tensor rows_like(const at::Tensor& t) {
  at::Tensor o = at::empty_like(t);
  bool fits = o.stride(3) == 1;
  for (int i = 0; i < 3; ++i) fits = fits && (o.size(i) == 1 || o.stride(i) % 8 == 0);
  return fits ? o : at::empty(t.sizes(), t.options());
}
void copy_strides(int64_t* to, const at::Tensor& t) {
  for (int i = 0; i < 4; ++i) to[i] = t.stride(i);
}
int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RSFA_DTYPE_BF16 : RSFA_DTYPE_F16; }
// (a, b or None) of two new tensors.
PyObject* tensor_pair(at::Tensor a, at::Tensor b) {
  PyObject* pa = THPVariable_Wrap(std::move(a));
  if (pa == nullptr) return nullptr;
  PyObject* pb = Py_None;
  if (b.defined())
    pb = THPVariable_Wrap(std::move(b));
  else
    Py_INCREF(pb);
  PyObject* pair = pb == nullptr ? nullptr : PyTuple_New(2);
  if (pair == nullptr) {
    Py_DECREF(pa);
    Py_XDECREF(pb);
    return nullptr;
  }
  PyTuple_SET_ITEM(pair, 0, pa);
  PyTuple_SET_ITEM(pair, 1, pb);
  return pair;
}

// The GIL is released while a launch may block; what is thrown in between comes out with it held again.
template <typename F>
void without_gil(F f) {
  PyThreadState* state = PyEval_SaveThread();
  try {
    f();
  } catch (...) {
    PyEval_RestoreThread(state);
    throw;
  }
  PyEval_RestoreThread(state);
}

// rsfa_rotary on tensors that it can read; k and pos may be undefined.
int turn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& table, const at::Tensor& pos, bool interleaved, bool inverse, at::Tensor* qo,
         at::Tensor* ko) {
  *qo = rows_like(q);
  if (k.defined()) *ko = rows_like(k);
  int64_t strides[16] = {}, pos_strides[2] = {0, 0};
  copy_strides(strides, q);
  copy_strides(strides + 8, *qo);
  if (k.defined()) {
    copy_strides(strides + 4, k);
    copy_strides(strides + 12, *ko);
  }
  if (pos.defined()) {
    pos_strides[0] = pos.dim() == 1 || pos.size(0) == 1 ? 0 : pos.stride(0);
    pos_strides[1] = pos.stride(-1);
  }
  return g_ops.rotary(q.const_data_ptr(), k.defined() ? k.const_data_ptr() : nullptr, qo->mutable_data_ptr(),
                      k.defined() ? ko->mutable_data_ptr() : nullptr, static_cast<int>(q.size(0)), static_cast<int>(q.size(1)),
                      k.defined() ? static_cast<int>(k.size(1)) : 0, static_cast<int>(q.size(2)), static_cast<int>(q.size(3)), strides,
                      static_cast<const float*>(table.const_data_ptr()), static_cast<int>(table.size(0)), static_cast<int>(2 * table.size(1)),
                      pos.defined() ? pos.const_data_ptr() : nullptr, pos.defined() && pos.scalar_type() == at::kLong ? 1 : 0,
                      pos.defined() ? pos_strides : nullptr, interleaved, inverse, dtype_of(q),
                      c10::cuda::getCurrentCUDAStream(q.device().index()).stream());
}

// The same as an operation that autograd records: its gradient is the transposed rotation, which can be recorded again.
// (As a Python function the two calls of a training step took 40 us more of the host's time.)
struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const std::optional<at::Tensor>& k_or,
                                                const at::Tensor& table, const std::optional<at::Tensor>& pos_or, bool interleaved, bool inverse) {
    const at::Tensor k = k_or.value_or(at::Tensor()), pos = pos_or.value_or(at::Tensor());
    at::Tensor qo, ko;
    check_code(turn(q, k, table, pos, interleaved, inverse, &qo, &ko), "rsfa_rotary");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({table, pos});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    if (!k.defined()) return {qo};
    return {qo, ko};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
    at::Tensor of_q = readable(grads[0]), of_k = grads.size() > 1 ? readable(grads[1]) : at::Tensor();
    torch::autograd::variable_list out(6);
    if (!of_q.defined() && !of_k.defined()) return out;
    const bool q_first = of_q.defined();                       // the library wants the first of its two tensors
    const at::Tensor first = q_first ? of_q : of_k, second = q_first ? of_k : at::Tensor();
    at::Tensor a, b;
    const at::Tensor of_first = readable(tangent_of(first)), of_second = readable(tangent_of(second));
    turn_again(primal(first), primal(second), saved, interleaved, inverse, &a, &b);
    if (of_first.defined() || of_second.defined()) {           // a gradient's tangent turns like the gradient
      at::Tensor ta, tb;
      if (of_first.defined())
        turn_again(of_first, of_second, saved, interleaved, inverse, &ta, &tb);
      else
        turn_again(of_second, of_first, saved, interleaved, inverse, &tb, &ta);
      if (ta.defined()) a._set_fw_grad(ta, 0, false);
      if (tb.defined()) b._set_fw_grad(tb, 0, false);
    }
    out[q_first ? 0 : 1] = a;
    if (q_first) out[1] = b;
    return out;
  }
  // Recorded in its turn, where that is asked for.
  static void turn_again(const at::Tensor& first, const at::Tensor& second, const torch::autograd::variable_list& saved, bool interleaved, bool inverse,
                         at::Tensor* a, at::Tensor* b) {
    if (c10::GradMode::is_enabled() && (first.requires_grad() || (second.defined() && second.requires_grad()))) {
      const auto again = RotaryFunction::apply(first, given(second), saved[0], given(saved[1]), interleaved, inverse);
      *a = again[0];
      if (second.defined()) *b = again[1];
      return;
    }
    check_code(turn(first, second, saved[0], saved[1], interleaved, inverse, a, b), "rsfa_rotary");
  }
  static at::Tensor primal(const at::Tensor& t) { return tangent_of(t).defined() ? t._fw_primal(0) : t; }
  static std::optional<at::Tensor> given(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }
  // Rows as the library reads them, copied once if need be.
  static at::Tensor readable(const at::Tensor& t) {
    if (!t.defined()) return t;
    bool ok = t.stride(3) == 1;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= t.size(3)));
    at::Tensor r = ok ? t : t.contiguous();
    return (reinterpret_cast<uintptr_t>(r.const_data_ptr()) & 15u) == 0 ? r : r.clone(at::MemoryFormat::Contiguous);
  }
};

// rotary(q, k or None, table, positions or None, interleaved, inverse) -> (q', k' or None), an error code, or None.
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (g_ops.rotary == nullptr || n != 6 || !plain_mode() || !PyBool_Check(args[4]) || !PyBool_Check(args[5])) Py_RETURN_NONE;
  const int device = device_of(args[0]);
  if (device < 0) Py_RETURN_NONE;
  const at::Tensor* q = plain_rows(args[0], device);
  const at::Tensor* k = args[1] == Py_None ? nullptr : plain_rows(args[1], device);
  const at::Tensor* table = plain_cuda(args[2], at::kFloat, 3, device);
  if (q == nullptr || (k == nullptr && args[1] != Py_None) || table == nullptr) Py_RETURN_NONE;
  const int64_t B = q->size(0), S = q->size(2), D = q->size(3), R = 2 * table->size(1);
  if (!(D == 16 || D == 32 || D == 64 || D == 128 || D == 256) || R > D || R < 2 || table->size(2) != 2 || !table->is_contiguous() ||
      table->size(0) < 1 || table->size(0) > INT32_MAX || table->requires_grad())
    Py_RETURN_NONE;
  if (k != nullptr && (k->size(0) != B || k->size(2) != S || k->size(3) != D || k->scalar_type() != q->scalar_type())) Py_RETURN_NONE;
  const at::Tensor* pos = nullptr;
  if (args[3] != Py_None) {
    if (!THPVariable_CheckExact(args[3])) Py_RETURN_NONE;
    const at::Tensor& p = THPVariable_Unpack(args[3]);
    if (!p.defined() || (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)) Py_RETURN_NONE;
    pos = plain_cuda(args[3], p.scalar_type(), p.dim(), device);
    if (pos == nullptr || (p.dim() != 1 && p.dim() != 2) || p.size(-1) != S || (p.dim() == 2 && p.size(0) != 1 && p.size(0) != B)) Py_RETURN_NONE;
  }
  const at::Tensor none;
  if (records_grad(*q) || (k != nullptr && records_grad(*k))) {
    torch::autograd::variable_list out;
    without_gil([&] {
      out = RotaryFunction::apply(*q, RotaryFunction::given(k != nullptr ? *k : none), *table, RotaryFunction::given(pos != nullptr ? *pos : none), args[4] == Py_True, args[5] == Py_True);
    });
    return tensor_pair(out[0], k != nullptr ? out[1] : none);
  }
  at::Tensor qo, ko;
  int rc = 0;
  without_gil([&] {
    rc = turn(*q, k != nullptr ? *k : none, *table, pos != nullptr ? *pos : none, args[4] == Py_True, args[5] == Py_True, &qo, &ko);
  });
  if (rc != 0) return PyLong_FromLong(rc);
  return tensor_pair(std::move(qo), std::move(ko));
  END_HANDLE_TH_ERRORS
}

// int32 [n] or None; false: something else.
bool plain_ints(PyObject* obj, int64_t n, int device, const int** out) {
  *out = nullptr;
  if (obj == Py_None) return true;
  const at::Tensor* t = plain_cuda(obj, at::kInt, 1, device);
  if (t == nullptr || t->size(0) != n || (n > 1 && t->stride(0) != 1)) return false;
  *out = static_cast<const int*>(t->const_data_ptr());
  return true;
}

// The cache of kv, table, lengths, weight or None and position or None; false: something else.
bool plain_cache(PyObject* kv_obj, PyObject* table_obj, PyObject* lengths_obj, PyObject* weight_obj, PyObject* position_obj, int dtype, int device,
                 rsfa_cache4* c) {
  const at::Tensor* kv = plain_cuda(kv_obj, at::kByte, 4, device);
  const at::Tensor* table = plain_cuda(table_obj, at::kInt, 2, device);
  if (kv == nullptr || table == nullptr) return false;
  const int64_t rec = kv->size(3), page = kv->size(2);
  if (!(rec == 80 || rec == 160 || rec == 320) || kv->size(0) < 1 || kv->size(1) < 1 || kv->stride(3) != 1 || kv->stride(2) != rec ||
      kv->stride(0) % 16 != 0 || kv->stride(1) % 16 != 0 || (reinterpret_cast<uintptr_t>(kv->const_data_ptr()) & 15u) != 0)
    return false;
  if (table->size(0) < 1 || table->size(1) < 1 || table->stride(1) != 1 || kv->size(0) > INT32_MAX || kv->size(1) > INT32_MAX || page > 1024 ||
      table->size(0) > INT32_MAX || table->size(1) > INT32_MAX)
    return false;
  std::memset(c, 0, sizeof(*c));
  if (lengths_obj == Py_None || !plain_ints(lengths_obj, table->size(0), device, &c->lengths)) return false;
  PyObject* extra[2] = {weight_obj, position_obj};
  for (int i = 0; i < 2; ++i) {
    if (extra[i] == Py_None) continue;
    const at::Tensor* t = plain_cuda(extra[i], i == 0 ? at::kFloat : at::kInt, 3, device);
    if (t == nullptr || t->size(0) != kv->size(0) || t->size(1) != kv->size(1) || t->size(2) != page || t->stride(2) != 1) return false;
    int64_t* st = i == 0 ? c->weight_stride : c->position_stride;
    st[0] = t->stride(0);
    st[1] = t->stride(1);
    if (i == 0)
      c->weight = static_cast<float*>(t->mutable_data_ptr());
    else
      c->position = static_cast<int*>(t->mutable_data_ptr());
  }
  c->kv = kv->mutable_data_ptr();
  c->kv_stride[0] = kv->stride(0);
  c->kv_stride[1] = kv->stride(1);
  c->table = static_cast<const int*>(table->const_data_ptr());
  c->table_stride = table->stride(0);
  c->batch = static_cast<int>(table->size(0));
  c->heads = static_cast<int>(kv->size(1));
  c->head_dim = static_cast<int>(rec / 5 * 4);
  c->page_size = static_cast<int>(page);
  c->pages = static_cast<int>(kv->size(0));
  c->max_pages = static_cast<int>(table->size(1));
  c->dtype = dtype;
  return true;
}

// append(k, v, kv, table, lengths, counts, weight, position, positions) -> True, an error code, or None.
PyObject* cache4_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (g_ops.append == nullptr || n != 9 || !plain_mode()) Py_RETURN_NONE;
  const int device = device_of(args[0]);
  if (device < 0) Py_RETURN_NONE;
  const at::Tensor* k = plain_rows(args[0], device);
  const at::Tensor* v = plain_rows(args[1], device);
  rsfa_cache4 c;
  if (k == nullptr || v == nullptr || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() ||
      !plain_cache(args[2], args[3], args[4], args[6], args[7], dtype_of(*k), device, &c))
    Py_RETURN_NONE;
  const int64_t S = k->size(2);
  const int* counts = nullptr;
  if (k->size(0) != c.batch || k->size(1) != c.heads || k->size(3) != c.head_dim || !plain_ints(args[5], c.batch, device, &counts) ||
      (args[7] == Py_None) != (args[8] == Py_None))
    Py_RETURN_NONE;
  int64_t pos_strides[2] = {0, 0};
  const int* positions = nullptr;
  if (args[8] != Py_None) {
    const at::Tensor* p = plain_cuda(args[8], at::kInt, 2, device);
    if (p == nullptr || p->size(0) != c.batch || p->size(1) != S) Py_RETURN_NONE;
    pos_strides[0] = p->stride(0);
    pos_strides[1] = p->stride(1);
    positions = static_cast<const int*>(p->const_data_ptr());
  }
  int64_t strides[8];
  copy_strides(strides, *k);
  copy_strides(strides + 4, *v);
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ops.append(&c, k->const_data_ptr(), v->const_data_ptr(), static_cast<int>(S), strides, counts, positions,
                    positions != nullptr ? pos_strides : nullptr, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// read(kv, table, lengths, n, bf16, starts) -> (k, v), an error code, or None.
PyObject* cache4_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int rows = 0;
  if (g_ops.read == nullptr || n != 6 || !plain_mode() || !plain_int(args[3], &rows) || rows < 1 || !PyBool_Check(args[4])) Py_RETURN_NONE;
  const int device = device_of(args[0]);
  if (device < 0) Py_RETURN_NONE;
  rsfa_cache4 c;
  const int* starts = nullptr;
  if (!plain_cache(args[0], args[1], args[2], Py_None, Py_None, args[4] == Py_True ? RSFA_DTYPE_BF16 : RSFA_DTYPE_F16, device, &c) ||
      !plain_ints(args[5], c.batch, device, &starts))
    Py_RETURN_NONE;
  const at::TensorOptions options = THPVariable_Unpack(args[0]).options().dtype(args[4] == Py_True ? at::kBFloat16 : at::kHalf);
  at::Tensor k = at::empty({c.batch, c.heads, rows, c.head_dim}, options), v = at::empty({c.batch, c.heads, rows, c.head_dim}, options);
  int64_t strides[8];
  copy_strides(strides, k);
  copy_strides(strides + 4, v);
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ops.read(&c, k.mutable_data_ptr(), v.mutable_data_ptr(), rows, strides, starts, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  return tensor_pair(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// attention(q, kv, table, lengths, sm_scale, counts, weight, want_lse) -> (o, lse or None), an error code, or None.
PyObject* cache4_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (g_ops.attention == nullptr || n != 8 || !plain_mode() || !PyFloat_CheckExact(args[4]) || !PyBool_Check(args[7])) Py_RETURN_NONE;
  const int device = device_of(args[0]);
  if (device < 0) Py_RETURN_NONE;
  const at::Tensor* q = plain_rows(args[0], device);
  rsfa_cache4 c;
  if (q == nullptr || !plain_cache(args[1], args[2], args[3], args[6], Py_None, dtype_of(*q), device, &c)) Py_RETURN_NONE;
  const int64_t Hq = q->size(1), S = q->size(2);
  const int* counts = nullptr;
  if (q->size(0) != c.batch || q->size(3) != c.head_dim || Hq % c.heads != 0 || !plain_ints(args[5], c.batch, device, &counts)) Py_RETURN_NONE;
  const long long bytes = g_ops.attention_workspace(&c, static_cast<int>(Hq), static_cast<int>(S));
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor o = rows_like(*q), lse;
  if (args[7] == Py_True || c.weight != nullptr) lse = at::empty({q->size(0), Hq, S}, q->options().dtype(at::kFloat));
  // the call's own scratch, from the pool of the current stream or of the graph that is being captured
  at::Tensor scratch = at::empty({bytes}, q->options().dtype(at::kByte));
  int64_t strides[8];
  copy_strides(strides, *q);
  copy_strides(strides + 4, o);
  float* lp = lse.defined() ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr;
  const float scale = static_cast<float>(PyFloat_AS_DOUBLE(args[4]));
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ops.attention(&c, q->const_data_ptr(), o.mutable_data_ptr(), lp, static_cast<int>(Hq), static_cast<int>(S), strides, counts, scale,
                       scratch.mutable_data_ptr(), bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  if (args[7] != Py_True) lse.reset();
  return tensor_pair(std::move(o), std::move(lse));
  END_HANDLE_TH_ERRORS
}

// evict(kv, weight, position, table, lengths, budget, recent) -> new lengths, an error code, or None.
PyObject* cache4_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int budget = 0, recent = 0;
  if (g_ops.evict == nullptr || n != 7 || !plain_mode() || !plain_int(args[5], &budget) || !plain_int(args[6], &recent) || budget < 1 ||
      recent < 0 || recent > budget || args[1] == Py_None || args[2] == Py_None)
    Py_RETURN_NONE;
  const int device = device_of(args[0]);
  if (device < 0) Py_RETURN_NONE;
  rsfa_cache4 c;
  if (!plain_cache(args[0], args[3], args[4], args[1], args[2], RSFA_DTYPE_F16, device, &c)) Py_RETURN_NONE;
  const at::Tensor& lengths = THPVariable_Unpack(args[4]);
  // as many records can move as there are slots within the budget, or beyond it
  const int64_t beyond = std::max<int64_t>(static_cast<int64_t>(c.max_pages) * c.page_size - budget, 0);
  const long long bytes = g_ops.evict_workspace(c.batch, c.heads, static_cast<int>(std::min<int64_t>(budget, beyond)));
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor out = at::empty({c.batch}, lengths.options());
  at::Tensor scratch = at::empty({bytes}, lengths.options().dtype(at::kByte));
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ops.evict(&c, budget, recent, static_cast<int*>(out.mutable_data_ptr()), scratch.mutable_data_ptr(), bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind_ops(addresses of the functions of Ops, in its order)
PyObject* bind_ops(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bind_ops takes eight addresses");
    return nullptr;
  }
  void* p[8];
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  g_ops.rotary = reinterpret_cast<decltype(g_ops.rotary)>(p[0]);
  g_ops.append = reinterpret_cast<decltype(g_ops.append)>(p[1]);
  g_ops.read = reinterpret_cast<decltype(g_ops.read)>(p[2]);
  g_ops.attention_workspace = reinterpret_cast<decltype(g_ops.attention_workspace)>(p[3]);
  g_ops.attention = reinterpret_cast<decltype(g_ops.attention)>(p[4]);
  g_ops.evict_workspace = reinterpret_cast<decltype(g_ops.evict_workspace)>(p[5]);
  g_ops.evict = reinterpret_cast<decltype(g_ops.evict)>(p[6]);
  g_ops.strerror = reinterpret_cast<decltype(g_ops.strerror)>(p[7]);
  Py_RETURN_NONE;
}

// bind(address of rsfa_fwd)
PyObject* bind(PyObject*, PyObject* arg) {
  void* p = PyLong_AsVoidPtr(arg);
  if (p == nullptr && PyErr_Occurred()) return nullptr;
  g_fwd = reinterpret_cast<FwdFn>(p);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(forward)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_O, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rotary)), METH_FASTCALL, nullptr},
    {"cache4_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache4_append)), METH_FASTCALL, nullptr},
    {"cache4_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache4_read)), METH_FASTCALL, nullptr},
    {"cache4_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache4_attention)), METH_FASTCALL, nullptr},
    {"cache4_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache4_evict)), METH_FASTCALL, nullptr},
    {"bind_ops", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind_ops)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rsfa_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rsfa_torch() {
  PyObject* m = PyModule_Create(&module);
  // the torch whose tensor layout this file was compiled for: the Python side uses it with no other
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", RSFA_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
