// Calls of the 8-bit cache's operators without Python's share: the argument checks of ops.append_kv8, read_kv8, paged_attn8 and paged_prefill8 on the tensors
// themselves, then the native entry point on the current stream.  A small call is bound by the host: 25 attribute lookups and 20 ctypes
// conversions take 6 to 9 us, this 0.5, the launch 3.  Each function returns 1 (launched), -1 (the entry point refused) or 0: not a plain call on the current
// device's tensors, for which ops.* does the rest (the CPU, fp32 rows, and the error message of what is wrong).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

using I = int;
using AppendFn = I (*)(const void*, I, void*, I, I, const void*, const void*, const void*, I, I, I, I, I, I, void*);
using ReadFn = I (*)(const void*, I, I, void*, void*, I, I, const void*, const void*, const void*, I, I, I, I, I, I, void*);
using AttnFn = I (*)(const void*, I, void*, I, I, void*, I, const void*, const void*, const void*, I, I, I, I, I, float, I, I, I, void*);
using RunsFn = I (*)(const void*, I, const void*, I, I, void*, I, const void*, const void*, const void*, I, I, I, I, I, float, I, const void*, const void*, I, void*);
AppendFn g_append;
ReadFn g_read;
AttnFn g_attn;
RunsFn g_runs;

constexpr int64_t INT_TOP = 0x7fffffff;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
// an int that fits 32 bits (larger ones: the largest), or false
bool number(PyObject* o, int& x) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over < 0 || v < -INT_TOP) return false;
  x = (int)(over || v > INT_TOP ? INT_TOP : v);
  return true;
}
bool rows(const at::Tensor& t, c10::ScalarType type, int64_t width, int64_t n) {
  return t.scalar_type() == type && t.dim() == 2 && t.stride(1) == 1 && t.size(1) >= width && t.size(0) >= n && t.stride(0) <= INT_TOP && t.size(0) <= INT_TOP;
}

// What the operators share: cache, positions, sequences, table, bs, H, hd.
struct Cache {
  void *kv, *pos, *slot, *btab, *stream;
  int n_blocks, rec, n_slots, max_lb, bs, H, hd;
  int64_t listed;                                  // positions and sequences that are given
  c10::DeviceIndex dev;
  bool on(const at::Tensor& t) const { return t.is_cuda() && t.device().index() == dev; }
  // a: kv, pos, slot, btab, bs, H, hd
  bool take(PyObject* const* a, PyObject* kv_obj) {
    const at::Tensor *c = tensor(kv_obj), *p = tensor(a[0]), *s = tensor(a[1]), *b = tensor(a[2]);
    if (!c || !p || !s || !b || !number(a[3], bs) || !number(a[4], H) || !number(a[5], hd)) return false;
    if ((hd != 16 && hd != 32 && hd != 64 && hd != 128) || bs < 1 || bs > 65535 || H < 1 || !c->is_cuda()) return false;
    dev = c->device().index();
    if (dev != c10::cuda::current_device() || !on(*p) || !on(*s) || !on(*b)) return false;
    if (c->scalar_type() != at::kByte || c->dim() != 3 || c->size(1) != H || c->size(2) != (2LL * bs * hd + 2 * bs + 31) / 32 * 32 || c->size(0) > INT_TOP || !c->is_contiguous()) return false;
    if (p->scalar_type() != at::kInt || s->scalar_type() != at::kInt || b->scalar_type() != at::kInt) return false;
    if (b->dim() != 2 || !b->is_contiguous() || b->size(0) > INT_TOP || b->size(1) > INT_TOP || !p->is_contiguous() || !s->is_contiguous()) return false;
    listed = std::min(p->numel(), s->numel());
    kv = c->data_ptr(); pos = p->data_ptr(); slot = s->data_ptr(); btab = b->data_ptr();
    n_blocks = (int)c->size(0); rec = (int)c->size(2); n_slots = (int)b->size(0); max_lb = (int)b->size(1);
    stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    return true;
  }
};
// No C++ exception leaves for Python (a tensor without memory of its own throws when it is asked for an address).
using Call = PyObject* (*)(PyObject* const*, Py_ssize_t);
template <Call F>
PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(a, n);
  } catch (...) {
    return PyLong_FromLong(0);
  }
}
PyObject* result(int rc) { return PyLong_FromLong(rc == 0 ? 1 : -1); }
PyObject* not_mine() { return PyLong_FromLong(0); }

// (qkv, kv, pos, slot, btab, bs, H, hd, ntok)
PyObject* append_kv8(PyObject* const* a, Py_ssize_t n) {
  Cache c;
  int ntok;
  const at::Tensor* x;
  if (n != 9 || !g_append || !c.take(a + 2, a[1]) || !(x = tensor(a[0])) || !number(a[8], ntok)) return not_mine();
  if (ntok < 0 || ntok > c.listed || !c.on(*x) || !rows(*x, at::kBFloat16, 3LL * c.H * c.hd, ntok)) return not_mine();
  return result(g_append(x->data_ptr(), (int)x->stride(0), c.kv, c.n_blocks, c.rec, c.pos, c.slot, c.btab, c.n_slots, c.max_lb, c.bs, c.H, c.hd, ntok, c.stream));
}
// (kv, k, v, pos, slot, btab, bs, H, hd, ntok)
PyObject* read_kv8(PyObject* const* a, Py_ssize_t n) {
  Cache c;
  int ntok;
  const at::Tensor *k, *v;
  if (n != 10 || !g_read || !c.take(a + 3, a[0]) || !(k = tensor(a[1])) || !(v = tensor(a[2])) || !number(a[9], ntok)) return not_mine();
  const c10::ScalarType t = k->scalar_type();
  if ((t != at::kBFloat16 && t != at::kFloat) || ntok < 0 || ntok > c.listed || !c.on(*k) || !c.on(*v)) return not_mine();
  if (!rows(*k, t, (int64_t)c.H * c.hd, ntok) || !rows(*v, t, (int64_t)c.H * c.hd, ntok) || k->stride(0) != v->stride(0)) return not_mine();
  return result(g_read(c.kv, c.n_blocks, c.rec, k->data_ptr(), v->data_ptr(), (int)k->stride(0), t == at::kFloat, c.pos, c.slot, c.btab, c.n_slots, c.max_lb, c.bs, c.H, c.hd, ntok, c.stream));
}
// (qkv, kv, out, pos, slot, btab, bs, H, hd, ntok, max_ctx, append)
PyObject* paged_attn8(PyObject* const* a, Py_ssize_t n) {
  Cache c;
  int ntok, max_ctx, append;
  const at::Tensor *x, *y;
  if (n != 12 || !g_attn || !c.take(a + 3, a[1]) || !(x = tensor(a[0])) || !(y = tensor(a[2])) || !number(a[9], ntok) || !number(a[10], max_ctx)) return not_mine();
  if ((append = PyObject_IsTrue(a[11])) < 0) return nullptr;
  if (ntok < 0 || ntok > c.listed || !c.on(*x) || !c.on(*y) || !rows(*x, at::kBFloat16, 3LL * c.H * c.hd, ntok) || !rows(*y, at::kBFloat16, (int64_t)c.H * c.hd, ntok)) return not_mine();
  return result(g_attn(x->data_ptr(), (int)x->stride(0), c.kv, c.n_blocks, c.rec, y->data_ptr(), (int)y->stride(0), c.pos, c.slot, c.btab, c.n_slots, c.max_lb, c.bs, c.H, c.hd,
                       (float)(1.0 / std::sqrt((double)c.hd)), ntok, max_ctx, append, c.stream));
}
// (qkv, kv, out, pos, slot, btab, bs, H, hd, runs, max_ctx)
PyObject* paged_prefill8(PyObject* const* a, Py_ssize_t n) {
  Cache c;
  int max_ctx;
  const at::Tensor *x, *y;
  if (n != 11 || !g_runs || !c.take(a + 3, a[1]) || c.hd == 16 || !(x = tensor(a[0])) || !(y = tensor(a[2])) || !PyList_Check(a[9]) || !number(a[10], max_ctx)) return not_mine();
  if (!c.on(*x) || !c.on(*y) || !rows(*x, at::kBFloat16, 3LL * c.H * c.hd, 0) || !rows(*y, at::kBFloat16, (int64_t)c.H * c.hd, 0)) return not_mine();
  const int64_t limit = std::min({x->size(0), y->size(0), c.listed});
  const Py_ssize_t k = PyList_GET_SIZE(a[9]);
  if (k > 1 << 24) return not_mine();
  std::vector<int> lists(2 * k);
  for (Py_ssize_t i = 0; i < k; i++) {
    PyObject* run = PyList_GET_ITEM(a[9], i);
    int r, len;
    if (!PyTuple_Check(run) || PyTuple_GET_SIZE(run) != 2 || !number(PyTuple_GET_ITEM(run, 0), r) || !number(PyTuple_GET_ITEM(run, 1), len)) return not_mine();
    if (r < 0 || len < 1 || (int64_t)r + len > limit) return not_mine();
    lists[i] = r;
    lists[k + i] = len;
  }
  return result(g_runs(x->data_ptr(), (int)x->stride(0), c.kv, c.n_blocks, c.rec, y->data_ptr(), (int)y->stride(0), c.pos, c.slot, c.btab, c.n_slots, c.max_lb, c.bs, c.H, c.hd,
                       (float)(1.0 / std::sqrt((double)c.hd)), max_ctx, lists.data(), lists.data() + k, (int)k, c.stream));
}
// addresses of the four entry points in libkharon_cuda
PyObject* set_entries(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[4];
  if (n != 4) { PyErr_SetString(PyExc_TypeError, "four addresses"); return nullptr; }
  for (int i = 0; i < 4; i++) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address"); return nullptr; }
  }
  g_append = (AppendFn)p[0];
  g_read = (ReadFn)p[1];
  g_attn = (AttnFn)p[2];
  g_runs = (RunsFn)p[3];
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"append_kv8", FAST(guarded<append_kv8>), nullptr}, {"read_kv8", FAST(guarded<read_kv8>), nullptr}, {"paged_attn8", FAST(guarded<paged_attn8>), nullptr},
                         {"paged_prefill8", FAST(guarded<paged_prefill8>), nullptr}, {"set_entries", FAST(set_entries), nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kharon_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kharon_bind() { return PyModule_Create(&module); }
