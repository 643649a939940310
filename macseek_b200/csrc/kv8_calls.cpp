// Calls of the 8-bit cache's entry points with PyTorch tensors: their checks and addresses, read from the tensors themselves.  In the
// interpreter these took 10 to 20 us of a call whose kernel takes 2 to 10.  A call that is not plainly right is not made (kNotTaken): the
// caller's own checks then say what is wrong with it; tensors without strides or memory throw here, which ends the same way.  Nothing is
// kept between calls.
#include <torch/csrc/autograd/python_variable.h>
#include <cstdint>
#include "../../include/macseek_b200.h"

namespace {
constexpr int kNotTaken = 1;

const at::Tensor* tensor(PyObject* o, int device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device ? &t : nullptr;
}
int type_of(const at::Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kFloat ? MSB_F32 : s == at::kHalf ? MSB_F16 : s == at::kBFloat16 ? MSB_BF16 : -1;
}
struct Rows { void* p; int64_t n, heads, dim, stride; int type; };
// rows [n][heads][dim] with dense heads
bool rows(PyObject* o, int device, Rows& r) {
  const at::Tensor* t = tensor(o, device);
  if (!t || t->dim() != 3) return false;
  r.n = t->size(0); r.heads = t->size(1); r.dim = t->size(2); r.type = type_of(*t);
  if (r.type < 0 || t->stride(2) != 1 || (t->stride(1) != r.dim && r.heads != 1)) return false;
  r.stride = r.n > 1 ? t->stride(0) : r.heads * r.dim;
  r.p = t->data_ptr();
  return true;
}
bool same(const Rows& a, int64_t n, int64_t heads, int64_t dim, int type) { return a.n == n && a.heads == heads && a.dim == dim && a.type == type; }
// contiguous F32 (int32) of n elements, or None where that is allowed
bool vector(PyObject* o, int device, at::ScalarType type, int64_t n, void** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o, device);
  if (!t || t->scalar_type() != type || t->numel() != n || !t->is_contiguous()) return false;
  *p = t->data_ptr();
  return true;
}
typedef int (*RowsFn)(const msb_kv8_cache*, const msb_kv8_batch*, int, void*, void*, int64_t, int64_t, void*);
typedef int (*AttnFn)(const msb_kv8_cache*, const msb_kv8_batch*, int, const void*, int64_t, int, float, int, const float*, void*, int64_t, void*,
                      size_t, void*);
typedef int (*NormRopeFn)(int, const void*, int, int64_t, const float*, const void*, int, int64_t, const float*, int, int, float, const float*,
                          const int*, int, int, int, int, void*, int64_t, void*, int64_t, void*);
}  // namespace

extern "C" int msb_host_kv8_rows(PyObject* k, PyObject* v, const msb_kv8_cache* c, const msb_kv8_batch* b, int device, RowsFn call, void* stream) {
  try {
    Rows x, y;
    if (!rows(k, device, x) || !rows(v, device, y) || !same(x, b->n_tokens, c->kv_heads, c->head_dim, y.type) || !same(y, x.n, x.heads, x.dim, x.type))
      return kNotTaken;
    return call(c, b, x.type, x.p, y.p, x.stride, y.stride, stream);
  } catch (...) {
    return kNotTaken;
  }
}

extern "C" int msb_host_kv8_attn(PyObject* q, PyObject* out, PyObject* scratch, PyObject* sinks, const msb_kv8_cache* c, const msb_kv8_batch* b,
                                 int device, double scale, int window, AttnFn call, void* stream) {
  try {
    Rows x, y;
    void* s;
    const at::Tensor* w = tensor(scratch, device);
    if (!w || !w->is_contiguous() || !rows(q, device, x) || !rows(out, device, y) || !same(x, b->n_tokens, x.heads, c->head_dim, y.type) ||
        !same(y, x.n, x.heads, x.dim, x.type) || !vector(sinks, device, at::kFloat, x.heads, &s) || (s && THPVariable_Unpack(sinks).dim() != 1))
      return kNotTaken;
    return call(c, b, x.type, x.p, x.stride, (int)x.heads, (float)scale, window, static_cast<const float*>(s), y.p, y.stride, w->data_ptr(),
                w->nbytes(), stream);
  } catch (...) {
    return kNotTaken;
  }
}

extern "C" int msb_host_head_norm_rope(PyObject* q, PyObject* k, PyObject* q_w, PyObject* k_w, double eps, PyObject* cs, PyObject* pos,
                                       PyObject* q_out, PyObject* k_out, int device, int first, int halves, NormRopeFn call, void* stream) {
  try {
    Rows a{}, b{}, ao{}, bo{};
    if (q != Py_None && (!rows(q, device, a) || !rows(q_out, device, ao) || !same(ao, a.n, a.heads, a.dim, a.type))) return kNotTaken;
    if (k != Py_None && (!rows(k, device, b) || !rows(k_out, device, bo) || !same(bo, b.n, b.heads, b.dim, b.type))) return kNotTaken;
    if (q == Py_None) { if (k == Py_None) return kNotTaken; a = Rows{nullptr, b.n, 0, b.dim, 0, b.type}; }
    if (k == Py_None) b = Rows{nullptr, a.n, 0, a.dim, 0, a.type};
    void *qw, *kw, *p;
    const at::Tensor* f = tensor(cs, device);
    if (a.n != b.n || a.dim != b.dim || a.type != b.type || !vector(q_w, device, at::kFloat, a.dim, &qw) || !vector(k_w, device, at::kFloat, a.dim, &kw) ||
        pos == Py_None || !vector(pos, device, at::kInt, a.n, &p) || !f || f->scalar_type() != at::kFloat || f->dim() != 3 || f->size(2) != 2 ||
        !f->is_contiguous() || f->size(0) > 0x7fffffff || f->size(1) > 0x3fffffff || a.n > 0x7fffffff)
      return kNotTaken;
    return call(a.type, a.p, (int)a.heads, a.stride, static_cast<const float*>(qw), b.p, (int)b.heads, b.stride, static_cast<const float*>(kw), (int)a.n,
                (int)a.dim, (float)eps, static_cast<const float*>(f->data_ptr()), static_cast<const int*>(p), (int)f->size(0), (int)(2 * f->size(1)),
                first, halves, ao.p, ao.stride, bo.p, bo.stride, stream);
  } catch (...) {
    return kNotTaken;
  }
}
