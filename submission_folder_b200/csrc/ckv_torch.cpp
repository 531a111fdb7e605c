// The paged cache's calls on torch tensors, as a CPython module: the arguments are checked, the
// outputs allocated and the C ABI (include/ckv.h) called on torch's current stream.  A decode step
// in eager mode makes these calls once per layer while its kernels take a few microseconds; in Python
// the checks and the packing of the structures cost more than the launch.
//
// Every function returns its result, or None when an argument is not what the call takes (ops.py
// then says which), or the C ABI's negative status as an int.
#include <Python.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/types.h>

#include "../../include/ckv.h"

namespace {

using at::Tensor;

// A new tensor on a device, not filled.
Tensor fresh_tensor(at::IntArrayRef size, at::ScalarType type, at::Device device) {
  return Tensor(at::detail::empty_cuda(size, type, device, std::nullopt));
}

// The tensor behind a Python argument, or null.
const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? CKV_BF16 : t == at::kHalf ? CKV_FP16 : t == at::kFloat ? CKV_FP32 : -1;
}

bool on(const Tensor* t, int device) { return t && t->is_cuda() && t->get_device() == device; }
bool vec(const Tensor* t, int device, at::ScalarType type, int64_t n) {
  return on(t, device) && t->scalar_type() == type && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}
bool rows(const Tensor* t, int device) {
  return on(t, device) && t->dim() == 3 && (t->stride(2) == 1 || t->size(2) == 1) && dtype_code(t->scalar_type()) >= 0;
}
// Whether autograd, of either mode, would follow this tensor.
bool grad(const Tensor* t) {
  return t && ((t->requires_grad() && at::GradMode::is_enabled()) ||
               (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined()));
}
// Tells autograd that the tensor's values have changed.
void wrote(const Tensor* t) {
  if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
bool table(const Tensor* t, int device) {
  return on(t, device) && t->scalar_type() == at::kInt && t->dim() == 2 && t->stride(1) == 1;
}
// Of the rows of a table; of a single row, whatever it is, at least the row.
int64_t table_stride(const Tensor* t) { return t->size(0) > 1 ? t->stride(0) : std::max(t->stride(0), t->size(1)); }
bool fits(int64_t x) { return x >= 0 && x <= INT32_MAX; }
template <typename T> T* ptr(const Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

// One call of the library: the device current, the tensor's current stream.
template <typename F> int call(int device, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device) guard.set_index(device);
  return f(reinterpret_cast<ckv_stream_t>(c10::cuda::getCurrentCUDAStream(device).stream()));
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* status(int rc) { return PyLong_FromLong(rc); }

bool cache_of(const Tensor* kc, const Tensor* vc, const Tensor* ks, const Tensor* vs, int device, ckv_cache* c) {
  if (!on(kc, device) || !on(vc, device) || !on(ks, device) || !on(vs, device)) return false;
  const auto type = kc->scalar_type();
  if ((type != at::kFloat8_e4m3fn && type != at::kChar) || vc->scalar_type() != type) return false;
  if (kc->dim() != 4 || vc->sizes() != kc->sizes() || kc->stride(3) != 1 || vc->stride(3) != 1) return false;
  for (const Tensor* s : {ks, vs})
    if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != kc->size(0) || s->size(1) != kc->size(1) ||
        !s->is_contiguous())
      return false;
  for (int i = 0; i < 4; ++i)
    if (!fits(kc->size(i))) return false;
  *c = {kc->data_ptr(), vc->data_ptr(), ptr<float>(ks), ptr<float>(vs), kc->stride(0), kc->stride(1), kc->stride(2),
        vc->stride(0), vc->stride(1), vc->stride(2), (int32_t)kc->size(0), (int32_t)kc->size(1), (int32_t)kc->size(2),
        (int32_t)kc->size(3), type == at::kChar ? CKV_CACHE_INT8 : CKV_CACHE_E4M3};
  return true;
}

#define CKV_FN(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)
#define CKV_ARGS(count) \
  if (n != (count)) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }

// lens, new, tables, free_list, free_count, block_size, total, shift, lens_out, free_count_out
CKV_FN(block_tables) {
  HANDLE_TH_ERRORS
  CKV_ARGS(10)
  const Tensor *lens = tensor(a[0]), *fresh = tensor(a[1]), *tables = tensor(a[2]), *list = tensor(a[3]), *count = tensor(a[4]);
  const Tensor *shift = a[7] == Py_None ? nullptr : tensor(a[7]);
  const Tensor *lens_out = a[8] == Py_None ? lens : tensor(a[8]), *count_out = a[9] == Py_None ? count : tensor(a[9]);
  const int64_t block = PyLong_AsLongLong(a[5]), total = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (!lens || !lens->is_cuda() || lens->dim() != 1) return none();
  const int dev = lens->get_device();
  const int64_t R = lens->size(0);
  if (!vec(lens, dev, at::kInt, R) || !vec(fresh, dev, at::kInt, R) || !vec(lens_out, dev, at::kInt, R) ||
      !vec(count, dev, at::kInt, 1) || !vec(count_out, dev, at::kInt, 1) || !list || !vec(list, dev, at::kInt, list->numel()) ||
      !table(tables, dev) || tables->size(0) != R || (a[7] != Py_None && !vec(shift, dev, at::kInt, R)) || !fits(total) ||
      !fits(block) || !fits(R) || !fits(tables->size(1)) || !fits(list->numel()))
    return none();
  const at::Device at = lens->device();
  Tensor cu = fresh_tensor({R + 1}, at::kInt, at), granted = fresh_tensor({R}, at::kInt, at), seen = fresh_tensor({R}, at::kInt, at);
  Tensor slots = fresh_tensor({total}, at::kLong, at), positions = fresh_tensor({total}, at::kLong, at);
  Tensor work;
  if (R + total > CKV_TABLES_SMALL) work = fresh_tensor({3 * R + 4}, at::kInt, at);
  const int64_t width = tables->size(1);
  const ckv_table_step s = {ptr<int32_t>(lens), ptr<int32_t>(fresh), ptr<int32_t>(shift), ptr<int32_t>(tables),
                            table_stride(tables), (int32_t)width, ptr<int32_t>(list), (int32_t)list->numel(),
                            ptr<int32_t>(count), (int32_t)block, (int32_t)R, (int32_t)total, ptr<int32_t>(lens_out),
                            ptr<int32_t>(count_out), ptr<int32_t>(&cu), ptr<int64_t>(&slots), ptr<int64_t>(&positions),
                            ptr<int32_t>(&granted), work.defined() ? ptr<int32_t>(&work) : nullptr, ptr<int32_t>(&seen)};
  const int rc = call(dev, [&](ckv_stream_t st) { return ckv_block_tables(&s, st); });
  if (rc) return status(rc);
  for (const Tensor* t : {lens_out, count_out, tables, list}) wrote(t);
  return Py_BuildValue("(NNNNNNN)", THPVariable_Wrap(*lens_out), THPVariable_Wrap(*count_out), THPVariable_Wrap(cu),
                       THPVariable_Wrap(slots), THPVariable_Wrap(positions), THPVariable_Wrap(granted), THPVariable_Wrap(seen));
  END_HANDLE_TH_ERRORS
}

// q, k, positions, inv_freq, interleaved, factor, inverse, out_q, out_k
CKV_FN(rotary) {
  HANDLE_TH_ERRORS
  CKV_ARGS(9)
  const Tensor *q = tensor(a[0]), *k = a[1] == Py_None ? nullptr : tensor(a[1]), *pos = tensor(a[2]), *freq = tensor(a[3]);
  const bool has_k = a[1] != Py_None;
  const int inter = PyObject_IsTrue(a[4]), inverse = PyObject_IsTrue(a[6]);
  const double factor = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!q || !q->is_cuda()) return none();
  const int dev = q->get_device();
  if (!rows(q, dev) || (has_k && !rows(k, dev)) || grad(q) || grad(k)) return none();
  const int64_t T = q->size(0), H = q->size(1), D = q->size(2), Hk = has_k ? k->size(1) : 0;
  if ((has_k && (k->scalar_type() != q->scalar_type() || k->size(0) != T || k->size(2) != D)) || !vec(pos, dev, at::kLong, T) ||
      !freq || !vec(freq, dev, at::kDouble, freq->numel()) || !fits(T) || !fits(H) || !fits(Hk) || !fits(D) ||
      !fits(2 * freq->numel()))
    return none();
  Tensor qo, ko;
  if (a[7] == Py_None && a[8] != Py_None) return none();
  if (a[7] == Py_None) {
    qo = fresh_tensor({T, H, D}, q->scalar_type(), q->device());
    if (has_k) ko = fresh_tensor({T, Hk, D}, q->scalar_type(), q->device());
  } else {
    const Tensor *x = tensor(a[7]), *y = a[8] == Py_None ? nullptr : tensor(a[8]);
    if (!rows(x, dev) || x->sizes() != q->sizes() || x->scalar_type() != q->scalar_type() || grad(x)) return none();
    if (has_k != (a[8] != Py_None)) return none();
    if (has_k && (!rows(y, dev) || y->sizes() != k->sizes() || y->scalar_type() != q->scalar_type() || grad(y))) return none();
    qo = *x;
    if (has_k) ko = *y;
  }
  ckv_rotary_args r = {};
  r.q = q->data_ptr(); r.q_tok_stride = q->stride(0); r.q_head_stride = q->stride(1);
  r.out_q = qo.data_ptr(); r.out_q_tok_stride = qo.stride(0); r.out_q_head_stride = qo.stride(1);
  if (has_k) {
    r.k = k->data_ptr(); r.k_tok_stride = k->stride(0); r.k_head_stride = k->stride(1);
    r.out_k = ko.data_ptr(); r.out_k_tok_stride = ko.stride(0); r.out_k_head_stride = ko.stride(1);
  }
  r.positions = ptr<int64_t>(pos); r.inv_freq = ptr<double>(freq);
  r.factor = (float)factor;
  r.tokens = (int32_t)T; r.q_heads = (int32_t)H; r.k_heads = (int32_t)Hk; r.head_dim = (int32_t)D;
  r.rotary_dim = (int32_t)(2 * freq->numel());
  r.dtype = dtype_code(q->scalar_type()); r.interleaved = inter; r.inverse = inverse;
  const int rc = call(dev, [&](ckv_stream_t st) { return ckv_rotary(&r, st); });
  if (rc) return status(rc);
  if (a[7] != Py_None) wrote(&qo);
  if (a[8] != Py_None) wrote(&ko);
  if (has_k) return Py_BuildValue("(NN)", THPVariable_Wrap(qo), THPVariable_Wrap(ko));
  return Py_BuildValue("(NO)", THPVariable_Wrap(qo), Py_None);
  END_HANDLE_TH_ERRORS
}

// k, v, k_cache, v_cache, k_scale, v_scale, slots
CKV_FN(cache_write) {
  HANDLE_TH_ERRORS
  CKV_ARGS(7)
  const Tensor *k = tensor(a[0]), *v = tensor(a[1]), *slots = tensor(a[6]);
  if (!k || !k->is_cuda()) return none();
  const int dev = k->get_device();
  ckv_cache c;
  if (!rows(k, dev) || !rows(v, dev) || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || grad(k) || grad(v) ||
      !vec(slots, dev, at::kLong, k->size(0)) || !fits(k->size(0)) ||
      !cache_of(tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5]), dev, &c) || k->size(1) != c.num_kv_heads ||
      k->size(2) != c.head_dim)
    return none();
  const int rc = call(dev, [&](ckv_stream_t st) {
    return ckv_cache_write(&c, k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1),
                           dtype_code(k->scalar_type()), ptr<int64_t>(slots), (int32_t)k->size(0), st);
  });
  if (rc) return status(rc);
  for (int i = 2; i < 6; ++i) wrote(tensor(a[i]));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// k_cache, v_cache, k_scale, v_scale, slots, dtype
CKV_FN(cache_read) {
  HANDLE_TH_ERRORS
  CKV_ARGS(6)
  const Tensor* slots = tensor(a[4]);
  if (!slots || !slots->is_cuda() || !THPDtype_Check(a[5])) return none();
  const int dev = slots->get_device();
  const auto type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  ckv_cache c;
  if (dtype_code(type) < 0 || !vec(slots, dev, at::kLong, slots->numel()) || !fits(slots->numel()) ||
      !cache_of(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), dev, &c))
    return none();
  const int64_t shape[] = {slots->numel(), c.num_kv_heads, c.head_dim};
  Tensor k = fresh_tensor(shape, type, slots->device()), v = fresh_tensor(shape, type, slots->device());
  const int rc = call(dev, [&](ckv_stream_t st) {
    return ckv_cache_read(&c, k.data_ptr(), v.data_ptr(), dtype_code(type), ptr<int64_t>(slots), (int32_t)slots->numel(), st);
  });
  if (rc) return status(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  END_HANDLE_TH_ERRORS
}

// q, k_cache, v_cache, k_scale, v_scale, tables, lens, cu, max_q, scale, causal, want_lse, out
CKV_FN(cache_attention) {
  HANDLE_TH_ERRORS
  CKV_ARGS(13)
  const Tensor *q = tensor(a[0]), *tables = tensor(a[5]), *lens = tensor(a[6]), *cu = a[7] == Py_None ? nullptr : tensor(a[7]);
  int64_t max_q = PyLong_AsLongLong(a[8]);
  const double scale = a[9] == Py_None ? 0.0 : PyFloat_AsDouble(a[9]);
  const int causal = PyObject_IsTrue(a[10]), want_lse = PyObject_IsTrue(a[11]);
  if (PyErr_Occurred()) return nullptr;
  if (!q || !q->is_cuda()) return none();
  const int dev = q->get_device();
  ckv_cache c;
  if (!rows(q, dev) || grad(q) || !table(tables, dev) || !vec(lens, dev, at::kInt, tables->size(0)) ||
      !cache_of(tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), dev, &c))
    return none();
  const int64_t T = q->size(0), H = q->size(1), D = q->size(2), R = tables->size(0);
  if (D != c.head_dim || c.num_kv_heads < 1 || H % c.num_kv_heads || !fits(T) || !fits(H) || !fits(tables->size(1))) return none();
  if (a[7] == Py_None) {
    if (R != T) return none();
    max_q = 1;
  } else if (!vec(cu, dev, at::kInt, R + 1)) {
    return none();
  }
  if (max_q > INT32_MAX || max_q < INT32_MIN) return none();
  Tensor out;
  if (a[12] == Py_None) {
    out = fresh_tensor({T, H, D}, q->scalar_type(), q->device());
  } else {
    const Tensor* o = tensor(a[12]);
    if (!rows(o, dev) || o->sizes() != q->sizes() || o->scalar_type() != q->scalar_type() || grad(o)) return none();
    out = *o;
  }
  size_t bytes = 0;
  int rc = ckv_cache_attention_workspace((int32_t)D, (int32_t)max_q, (int32_t)H, c.num_kv_heads, &bytes);
  if (rc) return status(rc);
  Tensor lse;
  if (want_lse) lse = fresh_tensor({T, H}, at::kFloat, q->device());
  // from the allocator for each call: two streams, or two captured graphs, never share it
  Tensor ws = fresh_tensor({(int64_t)bytes}, at::kByte, q->device());
  ckv_attention_args r = {};
  r.q = q->data_ptr(); r.q_tok_stride = q->stride(0); r.q_head_stride = q->stride(1);
  r.out = out.data_ptr(); r.out_tok_stride = out.stride(0); r.out_head_stride = out.stride(1);
  r.lse = want_lse ? ptr<float>(&lse) : nullptr;
  r.tables = ptr<int32_t>(tables); r.table_stride = table_stride(tables);
  r.table_width = (int32_t)tables->size(1);
  r.lens = ptr<int32_t>(lens); r.cu = ptr<int32_t>(cu);
  r.requests = (int32_t)R; r.tokens = (int32_t)T; r.max_q = (int32_t)max_q; r.q_heads = (int32_t)H;
  r.causal = causal;
  r.scale = (float)(a[9] == Py_None ? 1.0 / std::sqrt((double)D) : scale);
  r.dtype = dtype_code(q->scalar_type());
  rc = call(dev, [&](ckv_stream_t st) { return ckv_cache_attention(&c, &r, ws.data_ptr(), bytes, st); });
  if (rc) return status(rc);
  if (a[12] != Py_None) wrote(&out);
  if (want_lse) return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define CKV_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CKV_METHOD(block_tables), CKV_METHOD(rotary), CKV_METHOD(cache_write), CKV_METHOD(cache_read),
                         CKV_METHOD(cache_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ckv_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__ckv_torch(void) { return PyModule_Create(&module); }
