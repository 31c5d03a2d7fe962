// The plain form of the decode path's operators as one native call each: tensors in, tensors out.
//
// A decode step is a chain of kernels of 3 to 25 us, and what a call of ops.py costs on the host (argument checks,
// allocations and a ctypes call, each through Python) is about as much.  These functions do the same checks, allocate the
// results and enter the C ABI of libinferop_b200.so without coming back to Python in between.  Quantiser and GEMM of
// 32 x 1024 x 1024, called one after the other: 21.8 -> 9.2 us; of 64 x 24576 x 1536, where the kernels are about as long: 22.1 ->
// 18.4; an attention step of a few short sequences 72 -> 41.
//
// Each takes the arguments of its namesake in ops.py that a plain call has and returns
//   the result(s)   the call was made,
//   an int          the C ABI refused it (status; nothing was launched),
//   None            not the plain case (another device, a view that is not contiguous, a subclass, a wrong type or shape):
//                   ops.py makes the call, or refuses it with its own message.
// Tensors are allocated through torch's dispatcher as torch.empty does; its errors come out as the Python exceptions they
// are there.  The interpreter lock is released from the first allocation to the end of the call, as ctypes does.
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "inferop_b200.h"

namespace {

const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}
// Whether `t` is a contiguous tensor on the current CUDA device, which it names.  (A CPU tensor asks CUDA nothing.)
bool leads(const at::Tensor* t, c10::DeviceIndex* dev) {
  if (!t || !t->is_cuda() || !t->is_contiguous()) return false;
  *dev = c10::cuda::current_device();
  return t->device().index() == *dev;
}
// the other tensors of the call
bool plain(const at::Tensor* t, c10::DeviceIndex dev) {
  return t && t->is_cuda() && t->device().index() == dev && t->is_contiguous();
}
int code_of(at::ScalarType t) {   // element type codes of the C ABI, -1: none
  return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}
int out_code(PyObject* o, at::ScalarType* t) {
  if (!THPDtype_Check(o)) return -1;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return code_of(*t);
}
bool number(PyObject* o, float* v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *v = static_cast<float>(d);
  return true;
}
void* stream_of(c10::DeviceIndex dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
at::Tensor make(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType t) {
  return at::empty(sizes, like.options().dtype(t).requires_grad(false).memory_format(std::nullopt));
}
// b_q uint8 [n, k], b_scales fp32 [ceil(n / 128), k / 128]
bool weights_ok(const at::Tensor& bq, const at::Tensor& bs, int64_t k) {
  return bq.dim() == 2 && bq.scalar_type() == at::kByte && bq.size(1) == k && bs.dim() == 2 &&
         bs.scalar_type() == at::kFloat && bs.size(0) == (bq.size(0) + 127) / 128 && bs.size(1) == k / 128;
}
PyObject* pair(at::Tensor&& a, at::Tensor&& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = THPVariable_Wrap(std::move(b));
  if (!x || !y) {
    Py_XDECREF(x);
    Py_XDECREF(y);
    Py_DECREF(t);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}

// quant(x)
PyObject* quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1) Py_RETURN_NONE;
  const at::Tensor* x = tensor(a[0]);
  c10::DeviceIndex dev;
  if (!leads(x, &dev) || x->dim() != 2) Py_RETURN_NONE;
  const int dt = code_of(x->scalar_type());
  const int64_t rows = x->size(0), cols = x->size(1);
  if (dt < 0 || rows == 0 || cols % 128 != 0) Py_RETURN_NONE;
  at::Tensor q, s;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    q = make({rows, cols}, *x, at::kByte);
    s = make({rows, cols / 128}, *x, at::kFloat);
    rc = inferop_quant_fp8_per_token_group(q.data_ptr(), s.data_ptr(), x->data_ptr(), dt, rows, cols, 128, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return pair(std::move(q), std::move(s));
  END_HANDLE_TH_ERRORS
}

// gemm(a_q, a_scales, b_q, b_scales, out_dtype)
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *aq = tensor(a[0]), *as = tensor(a[1]), *bq = tensor(a[2]), *bs = tensor(a[3]);
  at::ScalarType ot;
  const int od = out_code(a[4], &ot);
  c10::DeviceIndex dev;
  if (od < 0 || !leads(aq, &dev) || !plain(as, dev) || !plain(bq, dev) || !plain(bs, dev)) Py_RETURN_NONE;
  if (aq->dim() != 2 || aq->scalar_type() != at::kByte || as->dim() != 2 || as->scalar_type() != at::kFloat) Py_RETURN_NONE;
  const int64_t m = aq->size(0), k = aq->size(1);
  if (k % 128 != 0 || as->size(0) != m || as->size(1) != k / 128 || !weights_ok(*bq, *bs, k)) Py_RETURN_NONE;
  const int64_t nn = bq->size(0);
  at::Tensor c;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    c = make({m, nn}, *aq, ot);
    rc = inferop_w8a8_block_fp8_gemm(c.data_ptr(), aq->data_ptr(), as->data_ptr(), bq->data_ptr(), bs->data_ptr(), m, nn, k,
                                     128, 128, od, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(c));
  END_HANDLE_TH_ERRORS
}

// gemm_fused_quant(a, b_q, b_scales, out_dtype)
PyObject* gemm_fused_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor *x = tensor(a[0]), *bq = tensor(a[1]), *bs = tensor(a[2]);
  at::ScalarType ot;
  const int od = out_code(a[3], &ot);
  c10::DeviceIndex dev;
  if (od < 0 || !leads(x, &dev) || !plain(bq, dev) || !plain(bs, dev) || x->dim() != 2) Py_RETURN_NONE;
  const int dt = code_of(x->scalar_type());
  const int64_t m = x->size(0), k = x->size(1);
  if (dt < 1 || k % 128 != 0 || !weights_ok(*bq, *bs, k)) Py_RETURN_NONE;
  const int64_t nn = bq->size(0);
  at::Tensor c;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    c = make({m, nn}, *x, ot);
    rc = inferop_w8a8_block_fp8_gemm_fused_quant(c.data_ptr(), x->data_ptr(), dt, bq->data_ptr(), bs->data_ptr(), m, nn, k, 128,
                                                 128, od, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(c));
  END_HANDLE_TH_ERRORS
}

// rmsnorm_quant(x, weight, eps, residual or None)
PyObject* rmsnorm_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float eps;
  if (n != 4 || !number(a[2], &eps)) Py_RETURN_NONE;
  const bool add = a[3] != Py_None;
  const at::Tensor *x = tensor(a[0]), *w = tensor(a[1]), *r = add ? tensor(a[3]) : nullptr;
  c10::DeviceIndex dev;
  if (!leads(x, &dev) || !plain(w, dev) || (add && !plain(r, dev)) || x->dim() != 2) Py_RETURN_NONE;
  const int dt = code_of(x->scalar_type());
  const int64_t rows = x->size(0), cols = x->size(1);
  if (dt < 1 || cols % 128 != 0 || w->scalar_type() != x->scalar_type() || w->dim() != 1 || w->size(0) != cols) Py_RETURN_NONE;
  if (add && (r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes())) Py_RETURN_NONE;
  at::Tensor q, s;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    q = make({rows, cols}, *x, at::kByte);
    s = make({rows, cols / 128}, *x, at::kFloat);
    rc = inferop_rmsnorm_quant(q.data_ptr(), s.data_ptr(), add ? r->data_ptr() : nullptr, x->data_ptr(), w->data_ptr(), dt, rows,
                               cols, 128, eps, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return pair(std::move(q), std::move(s));
  END_HANDLE_TH_ERRORS
}

// rope_neox(qkv, positions, rotary_dim, base, yarn_factor): in place; True when done
PyObject* rope_neox(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float base, yarn;
  if (n != 5 || !PyLong_CheckExact(a[2]) || !number(a[3], &base) || !number(a[4], &yarn)) Py_RETURN_NONE;
  int overflow = 0;
  const long rotary = PyLong_AsLongAndOverflow(a[2], &overflow);
  const at::Tensor *x = tensor(a[0]), *pos = tensor(a[1]);
  c10::DeviceIndex dev;
  if (overflow || rotary < 0 || rotary > 0x7FFFFFFF || !leads(x, &dev) || !plain(pos, dev) || x->dim() != 3) Py_RETURN_NONE;
  const int dt = code_of(x->scalar_type());
  if (dt < 0 || pos->scalar_type() != at::kLong || pos->numel() != x->size(0) || x->size(1) > 0x7FFFFFFF ||
      x->size(2) > 0x7FFFFFFF) {
    Py_RETURN_NONE;
  }
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    rc = inferop_rope_neox(x->data_ptr(), static_cast<const int64_t*>(pos->data_ptr()), dt, x->size(0),
                           static_cast<int32_t>(x->size(1)), static_cast<int32_t>(x->size(2)), static_cast<int32_t>(rotary), base,
                           yarn, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_attn_decode(q, k_cache, v_cache, block_tables, seq_lens, scale)
PyObject* paged_attn_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float scale;
  if (n != 6 || !number(a[5], &scale)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *kc = tensor(a[1]), *vc = tensor(a[2]), *bt = tensor(a[3]), *sl = tensor(a[4]);
  c10::DeviceIndex dev;
  if (!leads(q, &dev) || !plain(kc, dev) || !plain(vc, dev) || !plain(bt, dev) || !plain(sl, dev)) Py_RETURN_NONE;
  const at::ScalarType t = q->scalar_type();
  const int dt = code_of(t);
  if (dt < 0 || q->dim() != 3 || kc->dim() != 4 || vc->sizes() != kc->sizes() || kc->scalar_type() != t ||
      vc->scalar_type() != t || kc->size(3) != q->size(2)) {
    Py_RETURN_NONE;
  }
  if (bt->scalar_type() != at::kInt || sl->scalar_type() != at::kInt || bt->dim() != 2 || bt->size(0) != q->size(0) ||
      sl->numel() != q->size(0)) {
    Py_RETURN_NONE;
  }
  for (const int64_t v : {q->size(0), q->size(1), kc->size(1), kc->size(2), q->size(2), bt->size(1)})
    if (v > 0x7FFFFFFF) Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    out = make(q->sizes(), *q, t);
    rc = inferop_paged_attn_decode(out.data_ptr(), q->data_ptr(), kc->data_ptr(), vc->data_ptr(),
                                   static_cast<const int32_t*>(bt->data_ptr()), static_cast<const int32_t*>(sl->data_ptr()), dt,
                                   static_cast<int32_t>(q->size(0)), static_cast<int32_t>(q->size(1)),
                                   static_cast<int32_t>(kc->size(2)), static_cast<int32_t>(q->size(2)),
                                   static_cast<int32_t>(kc->size(1)), static_cast<int32_t>(bt->size(1)), scale, stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

bool integer(PyObject* o, long* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongAndOverflow(o, &overflow);
  return overflow == 0;
}
bool real(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) {
    long l;
    if (!integer(o, &l)) return false;
    *v = static_cast<double>(l);
    return true;
  }
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}
// an argument that may be None: true where it is, or where it is a plain tensor of this type and shape
bool optional(PyObject* o, c10::DeviceIndex dev, at::ScalarType type, at::IntArrayRef sizes, const void** ptr) {
  *ptr = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!plain(t, dev) || t->scalar_type() != type || t->sizes() != sizes) return false;
  *ptr = t->data_ptr();
  return true;
}
bool is(const at::Tensor* t, c10::DeviceIndex dev, at::ScalarType type, at::IntArrayRef sizes) {
  return plain(t, dev) && t->scalar_type() == type && t->sizes() == sizes;
}
// [tokens, rows, dim] whose rows of a token are contiguous: the stride of a token, or -1
int64_t token_stride(const at::Tensor* t, c10::DeviceIndex dev, at::ScalarType type, at::IntArrayRef sizes) {
  if (!t || !t->is_cuda() || t->device().index() != dev || t->scalar_type() != type || t->sizes() != sizes || t->size(0) == 0 ||
      t->stride(2) != 1 || (t->size(1) > 1 && t->stride(1) != t->size(2))) {
    return -1;
  }
  return t->size(0) > 1 ? t->stride(0) : t->size(1) * t->size(2);
}
bool fits(std::initializer_list<int64_t> sizes) {
  for (const int64_t v : sizes)
    if (v > 0x7FFFFFFF) return false;
  return true;
}
const int32_t* ints(const at::Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); }

// rope_append(q, k, v, k_cache, v_cache, k_scales, v_scales, block_tables, seq_lens, rotary_dim, base, yarn_factor, cu_seqlens or
// None, k_out or None); k_scales None: caches of q's type
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  long rotary;
  double base, yarn;
  if (n != 14 || !integer(a[9], &rotary) || rotary < 0 || rotary > 0x7FFFFFFF || !real(a[10], &base) || !real(a[11], &yarn)) Py_RETURN_NONE;
  const bool fp8 = a[5] != Py_None;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *kc = tensor(a[3]), *vc = tensor(a[4]);
  const at::Tensor *bt = tensor(a[7]), *sl = tensor(a[8]), *ko = a[13] == Py_None ? nullptr : tensor(a[13]);
  if (!q || !k || !kc || !q->is_cuda() || q->dim() != 3 || k->dim() != 3 || !bt || bt->dim() != 2 || kc->dim() != 4) Py_RETURN_NONE;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  const at::ScalarType t = q->scalar_type();
  const int dt = code_of(t);
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), kv = k->size(1);
  const int64_t batch = bt->size(0), per = bt->size(1), blocks = kc->size(0), block = kc->size(1);
  if (dt < 0 || !fits({heads, kv, dim, batch, per, blocks, block})) Py_RETURN_NONE;
  const int64_t qs = token_stride(q, dev, t, {tokens, heads, dim}), ks = token_stride(k, dev, t, {tokens, kv, dim});
  const int64_t vs = token_stride(v, dev, t, {tokens, kv, dim}), kos = ko ? token_stride(ko, dev, t, {tokens, kv, dim}) : 0;
  const at::ScalarType ct = fp8 ? at::kByte : t;
  if (qs < 0 || ks < 0 || vs < 0 || kos < 0 || (a[13] != Py_None && !ko) || !is(kc, dev, ct, {blocks, block, kv, dim}) ||
      !is(vc, dev, ct, {blocks, block, kv, dim}) || !is(bt, dev, at::kInt, {batch, per}) || !is(sl, dev, at::kInt, {batch})) {
    Py_RETURN_NONE;
  }
  const void *kss, *vss, *cu;
  if (!optional(a[5], dev, at::kFloat, {blocks, kv}, &kss) || !optional(a[6], dev, at::kFloat, {blocks, kv}, &vss) ||
      !optional(a[12], dev, at::kInt, {batch + 1}, &cu)) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    out = make({tokens, heads, dim}, *q, t);
    void* const ko_ptr = ko ? ko->data_ptr() : nullptr;
    const auto i32 = [](int64_t x) { return static_cast<int32_t>(x); };
    if (fp8) {
      rc = inferop_rope_append_kv_fp8(out.data_ptr(), heads * dim, ko_ptr, kos, kc->data_ptr(), vc->data_ptr(), const_cast<void*>(kss),
                                      const_cast<void*>(vss), q->data_ptr(), qs, k->data_ptr(), ks, v->data_ptr(), vs, ints(bt), ints(sl),
                                      static_cast<const int32_t*>(cu), dt, tokens, i32(batch), i32(heads), i32(kv), i32(dim), i32(rotary),
                                      i32(block), i32(blocks), i32(per), base, yarn, stream_of(dev));
    } else {
      rc = inferop_rope_append_kv(out.data_ptr(), heads * dim, ko_ptr, kos, kc->data_ptr(), vc->data_ptr(), q->data_ptr(), qs,
                                  k->data_ptr(), ks, v->data_ptr(), vs, ints(bt), ints(sl), static_cast<const int32_t*>(cu), dt, tokens,
                                  i32(batch), i32(heads), i32(kv), i32(dim), i32(rotary), i32(block), i32(blocks), i32(per), base, yarn,
                                  stream_of(dev));
    }
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_attn_decode_scored(q, k_cache, v_cache, k_scales, v_scales, block_tables, seq_lens, scale, softcap, alibi_slopes or None);
// k_scales None: caches of q's type
PyObject* paged_attn_decode_scored(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float scale, cap;
  if (n != 10 || !number(a[7], &scale) || !number(a[8], &cap)) Py_RETURN_NONE;
  const bool fp8 = a[3] != Py_None;
  const at::Tensor *q = tensor(a[0]), *kc = tensor(a[1]), *vc = tensor(a[2]), *bt = tensor(a[5]), *sl = tensor(a[6]);
  c10::DeviceIndex dev;
  if (!leads(q, &dev) || q->dim() != 3 || !kc || kc->dim() != 4 || !bt || bt->dim() != 2) Py_RETURN_NONE;
  const at::ScalarType t = q->scalar_type(), ct = fp8 ? at::kByte : t;
  const int dt = code_of(t);
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2), per = bt->size(1);
  const int64_t blocks = kc->size(0), block = kc->size(1), kv = kc->size(2);
  if (dt < (fp8 ? 1 : 0) || !fits({batch, heads, dim, per, blocks, block, kv})) Py_RETURN_NONE;
  const void *kss, *vss, *slopes;
  if (!is(kc, dev, ct, {blocks, block, kv, dim}) || !is(vc, dev, ct, {blocks, block, kv, dim}) || !is(bt, dev, at::kInt, {batch, per}) ||
      !is(sl, dev, at::kInt, {batch}) || !optional(a[3], dev, at::kFloat, {blocks, kv}, &kss) ||
      !optional(a[4], dev, at::kFloat, {blocks, kv}, &vss) || !optional(a[9], dev, at::kFloat, {heads}, &slopes)) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    out = make(q->sizes(), *q, t);
    const auto i32 = [](int64_t x) { return static_cast<int32_t>(x); };
    const float* sl_ptr = static_cast<const float*>(slopes);
    if (fp8) {
      rc = inferop_paged_attn_decode_fp8(out.data_ptr(), q->data_ptr(), kc->data_ptr(), vc->data_ptr(), kss, vss, ints(bt), ints(sl), dt,
                                         i32(batch), i32(heads), i32(kv), i32(dim), i32(block), i32(blocks), i32(per), scale, cap, sl_ptr,
                                         stream_of(dev));
    } else {
      rc = inferop_paged_attn_decode_scored(out.data_ptr(), q->data_ptr(), kc->data_ptr(), vc->data_ptr(), ints(bt), ints(sl), dt,
                                            i32(batch), i32(heads), i32(kv), i32(dim), i32(block), i32(per), scale, cap, sl_ptr, stream_of(dev));
    }
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// prefill_attn(q, k, v, cu_seqlens, scale, softcap, alibi_slopes or None, prefix_lens or None)
PyObject* prefill_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float scale, cap;
  if (n != 8 || !number(a[4], &scale) || !number(a[5], &cap)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *cu = tensor(a[3]);
  if (!q || !q->is_cuda() || q->dim() != 3 || !k || k->dim() != 3 || !cu || cu->dim() != 1 || cu->size(0) < 2) Py_RETURN_NONE;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  const at::ScalarType t = q->scalar_type();
  const int dt = code_of(t);
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), kv = k->size(1), batch = cu->size(0) - 1;
  if (dt < 1 || !fits({heads, kv, dim, batch})) Py_RETURN_NONE;
  const int64_t qs = token_stride(q, dev, t, {tokens, heads, dim}), ks = token_stride(k, dev, t, {tokens, kv, dim});
  const int64_t vs = token_stride(v, dev, t, {tokens, kv, dim});
  const void *slopes, *prefix;
  if (qs < 0 || ks < 0 || vs < 0 || !is(cu, dev, at::kInt, {batch + 1}) || !optional(a[6], dev, at::kFloat, {heads}, &slopes) ||
      !optional(a[7], dev, at::kInt, {batch}, &prefix)) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    out = make({tokens, heads, dim}, *q, t);
    rc = inferop_prefill_attn(out.data_ptr(), heads * dim, q->data_ptr(), qs, k->data_ptr(), ks, v->data_ptr(), vs, ints(cu),
                              static_cast<const int32_t*>(prefix), dt, tokens, static_cast<int32_t>(batch), static_cast<int32_t>(heads),
                              static_cast<int32_t>(kv), static_cast<int32_t>(dim), scale, cap, static_cast<const float*>(slopes),
                              stream_of(dev));
  }
  if (rc != INFEROP_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(quant), FAST(gemm), FAST(gemm_fused_quant), FAST(rmsnorm_quant), FAST(rope_neox),
                         FAST(paged_attn_decode), FAST(rope_append), FAST(paged_attn_decode_scored), FAST(prefill_attn),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall() { return PyModule_Create(&module); }
