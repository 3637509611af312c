// The host's side of calls that are shorter than Python's checks of their arguments: a
// layer's tree or branch attention, the verification, the beams' selection, the moves in a
// model's caches (128 tensors).
// Python reads a tensor's device, dtype, shape, contiguity and address in about 0.3 us
// each, and ctypes a call of 30 arguments in 4.  Here a call in its plain form (every
// tensor of the type and layout that the kernels read, on the current device) is checked
// and made in one go; any other form is answered with None, and the caller's Python
// converts or refuses it.
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <climits>
#include <cstring>
#include <vector>

#include "kf_attn.h"

namespace {

// same(list, out: writable buffer of 8 bytes an element, at: first element) -> the
// tensors' device index (-1: not on a GPU); raises ValueError where an element is
// no tensor, differs from the first in device, dtype or shape, or is not
// contiguous.  The data pointers go to out[at], out[at + 1], ...
PyObject* same(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  // (fake and symbolic tensors throw where they are asked for sizes or an address)
  HANDLE_TH_ERRORS
  if (nargs != 3 || !PyList_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "same(list, buffer, first)");
    return nullptr;
  }
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const Py_ssize_t at = PyLong_AsSsize_t(args[2]);
  if (at == -1 && PyErr_Occurred()) return nullptr;
  struct Buffer {
    Py_buffer b;
    bool held;
    ~Buffer() {
      if (held) PyBuffer_Release(&b);
    }
  } buf = {};
  buf.held = PyObject_GetBuffer(args[1], &buf.b, PyBUF_WRITABLE) == 0;
  if (!buf.held) return nullptr;
  const char* wrong = nullptr;
  long device = -1;
  if (at < 0 || n < 1 || (at + n) * 8 > buf.b.len) wrong = "no room for the pointers";
  const at::Tensor* first = nullptr;
  for (Py_ssize_t i = 0; !wrong && i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_Check(o)) {
      wrong = "tensors are needed";
      break;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.has_storage() || t.layout() != at::kStrided)
      wrong = "strided tensors are needed";
    else if (!t.is_contiguous())
      wrong = "contiguous tensors are needed";
    else if (first && t.device() != first->device())
      wrong = "the tensors must lie on one device";
    else if (first && t.scalar_type() != first->scalar_type())
      wrong = "the tensors must share a dtype";
    else if (first && t.sizes() != first->sizes())
      wrong = "the tensors must share a shape";
    if (!first) {
      first = &t;
      device = t.is_cuda() ? (long)t.get_device() : -1;
    }
    const uint64_t p = wrong ? 0 : (uint64_t)(uintptr_t)t.data_ptr();
    std::memcpy((char*)buf.b.buf + (at + i) * 8, &p, 8);
  }
  if (wrong) {
    PyErr_SetString(PyExc_ValueError, wrong);
    return nullptr;
  }
  return PyLong_FromLong(device);
  END_HANDLE_TH_ERRORS
}

// The library's entry points, by bind() (the library is opened by Python).
struct Entries {
  decltype(&kf_attn_tree_workspace_size) tree_size;
  decltype(&kf_attn_tree) tree;
  decltype(&kf_verify_drafts_workspace_size) verify_size;
  decltype(&kf_verify_drafts) verify;
  decltype(&kf_kv_cache_keep) keep;
} lib = {};
// Those of several continuations of one prompt, by bind_branches().
struct BranchEntries {
  decltype(&kf_attn_branch_workspace_size) branch_size;
  decltype(&kf_attn_branch) branch;
  decltype(&kf_beam_select_workspace_size) select_size;
  decltype(&kf_beam_select) select;
  decltype(&kf_kv_cache_reorder) reorder;
} branches = {};

PyObject* bind_to(void* entries, PyObject* const* args, Py_ssize_t nargs) {
  void* p[5];
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "bind(five addresses)");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i)
    if (!(p[i] = PyLong_AsVoidPtr(args[i]))) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  std::memcpy(entries, p, sizeof(p));
  Py_RETURN_NONE;
}
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  static_assert(sizeof(lib) == 5 * sizeof(void*), "an address each");
  return bind_to(&lib, args, nargs);
}
PyObject* bind_branches(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  static_assert(sizeof(branches) == 5 * sizeof(void*), "an address each");
  return bind_to(&branches, args, nargs);
}

// An argument's tensor if it is one of the plain type on the device, else null.
const at::Tensor* tensor(PyObject* o, long device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided ? &t : nullptr;
}
const at::Tensor* tensor(PyObject* o, long device, at::ScalarType type, at::IntArrayRef sizes) {
  const at::Tensor* t = tensor(o, device);
  return t && t->scalar_type() == type && t->sizes() == sizes && t->is_contiguous() ? t : nullptr;
}
// The same, None being allowed (*t is then null).
bool optional(PyObject* o, long device, at::ScalarType type, at::IntArrayRef sizes,
              const at::Tensor** t) {
  *t = o == Py_None ? nullptr : tensor(o, device, type, sizes);
  return *t || o == Py_None;
}
template <typename T>
T* data(const at::Tensor* t) {
  return t ? (T*)t->data_ptr() : nullptr;
}
int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KF_DTYPE_F32;
    case at::kBFloat16: return KF_DTYPE_BF16;
    case at::kHalf: return KF_DTYPE_F16;
    default: return -1;
  }
}
bool integer(PyObject* o, int64_t* x) {
  int overflow = 0;
  if (!PyLong_CheckExact(o)) return false;
  *x = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow;
}
bool fits(int64_t x) { return x >= INT_MIN && x <= INT_MAX; }
bool number(PyObject* o, double* x) {
  int64_t i = 0;
  if (!PyFloat_CheckExact(o) && !(integer(o, &i) && fits(i))) return false;
  *x = PyFloat_CheckExact(o) ? PyFloat_AS_DOUBLE(o) : (double)i;
  return true;
}
at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)(n > 0 ? n : 1)}, like.options().dtype(at::kByte));
}
// parents: [N] or [B, N]; their row stride
bool tree_shape(PyObject* parents, PyObject* counts, long device, int64_t B, int64_t N,
                const at::Tensor** par, int64_t* stride, const at::Tensor** cnt) {
  *stride = 0;
  if (!optional(parents, device, at::kInt, {N}, par)) {
    if (!(*par = tensor(parents, device, at::kInt, {B, N}))) return false;
    *stride = N;
  }
  return optional(counts, device, at::kInt, {B}, cnt);
}

// tree(q, k, v, k_cache, v_cache, lens, cos, sin, parents, counts, q_norm_weight,
//      k_norm_weight, norm_eps, rope_row_offset, max_len, device, stream)
//   -> out, an error code, or None
PyObject* tree(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t offset, max_len, device, stream, stride;
  double eps;
  if (nargs != 17 || !lib.tree || !number(args[12], &eps) || !integer(args[13], &offset) ||
      !integer(args[14], &max_len) || !fits(max_len) || !integer(args[15], &device) ||
      !integer(args[16], &stream))
    Py_RETURN_NONE;
  const at::Tensor *q = tensor(args[0], device), *kc = tensor(args[3], device);
  if (!q || !kc || q->dim() != 4 || kc->dim() != 4 || !q->is_contiguous()) Py_RETURN_NONE;
  const int64_t B = q->size(0), N = q->size(1), Hq = q->size(2), D = q->size(3);
  const int64_t Hkv = kc->size(1), Smax = kc->size(2);
  const auto type = q->scalar_type();
  const int dt = dtype_of(*q);
  const at::Tensor *k = tensor(args[1], device, type, {B, N, Hkv, D}),
                   *v = tensor(args[2], device, type, {B, N, Hkv, D}),
                   *vc = tensor(args[4], device, type, {B, Hkv, Smax, D}),
                   *lens = tensor(args[5], device, at::kInt, {B}),
                   *cos = tensor(args[6], device), *parents, *counts, *qnw, *knw;
  if (dt < 0 || !k || !v || !vc || !lens || !cos || cos->dim() != 2 ||
      !tensor(args[3], device, type, {B, Hkv, Smax, D}) ||
      !tensor(args[6], device, at::kFloat, {cos->size(0), D / 2}) || !fits(B) || !fits(N) ||
      !fits(Hq) || !fits(Hkv) || !fits(Smax) || !fits(D))
    Py_RETURN_NONE;
  const at::Tensor* sin = tensor(args[7], device, at::kFloat, cos->sizes());
  if (!sin || !tree_shape(args[8], args[9], device, B, N, &parents, &stride, &counts) ||
      !optional(args[10], device, at::kFloat, {D}, &qnw) ||
      !optional(args[11], device, at::kFloat, {D}, &knw) || !qnw != !knw)
    Py_RETURN_NONE;
  size_t need = 0;
  int rc = lib.tree_size((int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)max_len, dt, &need);
  if (rc) return PyLong_FromLong(rc);
  at::Tensor out = at::empty(q->sizes(), q->options()), ws = bytes(need, *q);
  rc = lib.tree(q->data_ptr(), k->data_ptr(), v->data_ptr(), kc->data_ptr(), vc->data_ptr(),
                data<int32_t>(lens), data<int32_t>(parents), stride, data<int32_t>(counts),
                data<float>(cos), data<float>(sin), offset, cos->size(0), out.data_ptr(),
                ws.data_ptr(), ws.numel(), (int)B, (int)N, (int)Smax, (int)Hq, (int)Hkv, (int)D,
                (int)max_len, data<float>(qnw), data<float>(knw), (float)eps, dt, (void*)stream);
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// verify(logits, tokens, uniforms, parents, counts, draft_logits, temperature, device, stream)
//   -> (path, kept, token), an error code, or None
PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t device, stream, stride;
  double temperature;
  if (nargs != 9 || !lib.verify || !number(args[6], &temperature) ||
      !integer(args[7], &device) || !integer(args[8], &stream))
    Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[0], device);
  if (!x || x->dim() != 3 || x->stride(2) != 1) Py_RETURN_NONE;
  const int64_t B = x->size(0), N = x->size(1), V = x->size(2);
  const int dt = dtype_of(*x);
  const at::Tensor *tokens = tensor(args[1], device, at::kLong, {B, N}),
                   *uniforms = tensor(args[2], device, at::kFloat, {B, N}), *parents, *counts,
                   *draft = nullptr;
  if (dt < 0 || !tokens || !uniforms || !fits(B) || !fits(N) || !fits(V) ||
      !tree_shape(args[3], args[4], device, B, N, &parents, &stride, &counts))
    Py_RETURN_NONE;
  if (args[5] != Py_None) {
    draft = tensor(args[5], device);
    if (!draft || parents || !(temperature > 0.0) || N < 2 || draft->dim() != 3 ||
        draft->scalar_type() != x->scalar_type() || draft->stride(2) != 1 ||
        draft->sizes() != at::IntArrayRef({B, N - 1, V}))
      Py_RETURN_NONE;
  }
  size_t need = 0;
  int rc = lib.verify_size((int)B, (int)N, (int)V, draft != nullptr, dt, &need);
  if (rc) return PyLong_FromLong(rc);
  const auto options = x->options();
  at::Tensor path = at::empty({B, N}, options.dtype(at::kInt)),
             kept = at::empty({B}, options.dtype(at::kInt)),
             next = at::empty({B}, options.dtype(at::kLong)), ws = bytes(need, *x);
  rc = lib.verify(x->data_ptr(), x->stride(0), x->stride(1), data<int64_t>(tokens),
                  data<int32_t>(parents), stride, data<int32_t>(counts), data<void>(draft),
                  draft ? draft->stride(0) : 0, draft ? draft->stride(1) : 0,
                  data<float>(uniforms), temperature, data<int32_t>(&path), data<int32_t>(&kept),
                  data<int64_t>(&next), ws.data_ptr(), ws.numel(), (int)B, (int)N, (int)V, dt,
                  (void*)stream);
  if (rc) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(path));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(kept));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(next));
  return r;
  END_HANDLE_TH_ERRORS
}

// The pointers of a list of n tensors of one type and shape; false if it is none.
bool pointers(PyObject* list, Py_ssize_t n, long device, at::ScalarType type,
              at::IntArrayRef sizes, std::vector<void*>& out) {
  if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) != n) return false;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = tensor(PyList_GET_ITEM(list, i), device, type, sizes);
    if (!t) return false;
    out.push_back(t->data_ptr());
  }
  return true;
}

// keep(k_caches, v_caches, lens, lens_out, path, kept, device, stream) -> error code or None
PyObject* keep(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t device, stream;
  if (nargs != 8 || !lib.keep || !integer(args[6], &device) || !integer(args[7], &stream) ||
      !PyList_CheckExact(args[0]) || PyList_GET_SIZE(args[0]) < 1)
    Py_RETURN_NONE;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const at::Tensor *k0 = tensor(PyList_GET_ITEM(args[0], 0), device),
                   *path = tensor(args[4], device);
  if (!k0 || k0->dim() != 4 || !path || path->dim() != 2 || !fits(n)) Py_RETURN_NONE;
  const int64_t B = k0->size(0), N = path->size(1);
  const int dt = dtype_of(*k0);
  const auto type = k0->scalar_type();
  const at::Tensor* kept = tensor(args[5], device, at::kInt, {B});
  std::vector<void*> p;
  p.reserve(4 * n);
  if (dt < 0 || !kept || !tensor(args[4], device, at::kInt, {B, N}) || !fits(B) || !fits(N) ||
      !fits(k0->size(1)) || !fits(k0->size(2)) || !fits(k0->size(3)) ||
      !pointers(args[0], n, device, type, k0->sizes(), p) ||
      !pointers(args[1], n, device, type, k0->sizes(), p) ||
      !pointers(args[2], n, device, at::kInt, {B}, p) ||
      !pointers(args[3], n, device, at::kInt, {B}, p))
    Py_RETURN_NONE;
  return PyLong_FromLong(lib.keep(p.data(), p.data() + n, (const int32_t* const*)(p.data() + 2 * n),
                                  (int32_t* const*)(p.data() + 3 * n), (int)n,
                                  data<int32_t>(path), data<int32_t>(kept), (int)N, (int)B,
                                  (int)k0->size(1), (int)k0->size(2), (int)k0->size(3), dt,
                                  (void*)stream));
  END_HANDLE_TH_ERRORS
}

// branch(q, k, v, k_prefix, v_prefix, prefix_lens, k_cache, v_cache, lens, cos, sin, counts,
//        q_norm_weight, k_norm_weight, norm_eps, rope_row_offset, max_prefix, max_len,
//        device, stream) -> out, an error code, or None
PyObject* branch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t offset, max_prefix, max_len, device, stream;
  double eps;
  if (nargs != 20 || !branches.branch || !number(args[14], &eps) || !integer(args[15], &offset) ||
      !integer(args[16], &max_prefix) || !fits(max_prefix) || !integer(args[17], &max_len) ||
      !fits(max_len) || !integer(args[18], &device) || !integer(args[19], &stream))
    Py_RETURN_NONE;
  const at::Tensor *q = tensor(args[0], device), *kp = tensor(args[3], device),
                   *kc = tensor(args[6], device);
  if (!q || !kp || !kc || q->dim() != 4 || kp->dim() != 4 || kc->dim() != 4 ||
      !q->is_contiguous())
    Py_RETURN_NONE;
  const int64_t B = q->size(0), N = q->size(1), Hq = q->size(2), D = q->size(3);
  const int64_t G = kp->size(0), Pmax = kp->size(2), Hkv = kc->size(1), Smax = kc->size(2);
  const auto type = q->scalar_type();
  const int dt = dtype_of(*q);
  const at::Tensor *k = tensor(args[1], device, type, {B, N, Hkv, D}),
                   *v = tensor(args[2], device, type, {B, N, Hkv, D}),
                   *vp = tensor(args[4], device, type, {G, Hkv, Pmax, D}),
                   *plens = tensor(args[5], device, at::kInt, {G}),
                   *vc = tensor(args[7], device, type, {B, Hkv, Smax, D}),
                   *lens = tensor(args[8], device, at::kInt, {B}),
                   *cos = tensor(args[9], device), *counts, *qnw, *knw;
  if (dt < 0 || !k || !v || !vp || !plens || !vc || !lens || !cos || cos->dim() != 2 ||
      !tensor(args[3], device, type, {G, Hkv, Pmax, D}) ||
      !tensor(args[6], device, type, {B, Hkv, Smax, D}) ||
      !tensor(args[9], device, at::kFloat, {cos->size(0), D / 2}) || G < 1 || B % G || !fits(B) ||
      !fits(N) || !fits(Hq) || !fits(Hkv) || !fits(Pmax) || !fits(Smax) || !fits(D))
    Py_RETURN_NONE;
  const at::Tensor* sin = tensor(args[10], device, at::kFloat, cos->sizes());
  if (!sin || !optional(args[11], device, at::kInt, {B}, &counts) ||
      !optional(args[12], device, at::kFloat, {D}, &qnw) ||
      !optional(args[13], device, at::kFloat, {D}, &knw) || !qnw != !knw)
    Py_RETURN_NONE;
  size_t need = 0;
  int rc = branches.branch_size((int)G, (int)B, (int)N, (int)Hq, (int)Hkv, (int)D, (int)max_prefix,
                           (int)max_len, dt, &need);
  if (rc) return PyLong_FromLong(rc);
  at::Tensor out = at::empty(q->sizes(), q->options()), ws = bytes(need, *q);
  rc = branches.branch(q->data_ptr(), k->data_ptr(), v->data_ptr(), kp->data_ptr(), vp->data_ptr(),
                  data<int32_t>(plens), kc->data_ptr(), vc->data_ptr(), data<int32_t>(lens),
                  data<int32_t>(counts), data<float>(cos), data<float>(sin), offset, cos->size(0),
                  out.data_ptr(), ws.data_ptr(), ws.numel(), (int)G, (int)B, (int)N, (int)Pmax,
                  (int)Smax, (int)Hq, (int)Hkv, (int)D, (int)max_prefix, (int)max_len,
                  data<float>(qnw), data<float>(knw), (float)eps, dt, (void*)stream);
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// select(logits, scores, K, device, stream) -> (scores, parents, tokens), an error code, or None
PyObject* select(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t K, device, stream;
  if (nargs != 5 || !branches.select || !integer(args[2], &K) || !integer(args[3], &device) ||
      !integer(args[4], &stream))
    Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[0], device);
  if (!x || x->dim() != 3 || x->stride(2) != 1) Py_RETURN_NONE;
  const int64_t G = x->size(0), W = x->size(1), V = x->size(2);
  const int dt = dtype_of(*x);
  const at::Tensor* scores = tensor(args[1], device, at::kFloat, {G, W});
  // (what Python refuses is left to it, so that a mistake raises one exception)
  if (dt < 0 || !scores || !fits(G) || !fits(V) || W < 1 || W > KF_BEAM_MAX || K < 1 ||
      K > KF_BEAM_MAX_SELECT)
    Py_RETURN_NONE;
  size_t need = 0;
  int rc = branches.select_size((int)G, (int)W, (int)V, (int)K, dt, &need);
  if (rc) return PyLong_FromLong(rc);
  const auto options = x->options();
  at::Tensor best = at::empty({G, K}, options.dtype(at::kFloat)),
             parents = at::empty({G, K}, options.dtype(at::kInt)),
             tokens = at::empty({G, K}, options.dtype(at::kLong)), ws = bytes(need, *x);
  rc = branches.select(x->data_ptr(), x->stride(0), x->stride(1), data<float>(scores),
                  data<float>(&best), data<int32_t>(&parents), data<int64_t>(&tokens),
                  ws.data_ptr(), ws.numel(), (int)G, (int)W, (int)V, (int)K, dt, (void*)stream);
  if (rc) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(best));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(parents));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(tokens));
  return r;
  END_HANDLE_TH_ERRORS
}

// reorder(k_caches, v_caches, lens, parents, device, stream) -> error code or None
PyObject* reorder(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t device, stream;
  if (nargs != 6 || !branches.reorder || !integer(args[4], &device) || !integer(args[5], &stream) ||
      !PyList_CheckExact(args[0]) || PyList_GET_SIZE(args[0]) < 1)
    Py_RETURN_NONE;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const at::Tensor *k0 = tensor(PyList_GET_ITEM(args[0], 0), device),
                   *parents = tensor(args[3], device);
  if (!k0 || k0->dim() != 4 || !parents || parents->dim() != 2 || !fits(n)) Py_RETURN_NONE;
  const int64_t B = k0->size(0), G = parents->size(0), W = parents->size(1);
  const int dt = dtype_of(*k0);
  const auto type = k0->scalar_type();
  const at::Tensor* lens = tensor(args[2], device, at::kInt, {B});
  std::vector<void*> p;
  p.reserve(2 * n);
  if (dt < 0 || !lens || !tensor(args[3], device, at::kInt, {G, W}) || !fits(B) || !fits(G) ||
      W > KF_BEAM_MAX || G * W != B || !fits(k0->size(1)) || !fits(k0->size(2)) ||
      !fits(k0->size(3)) ||
      !pointers(args[0], n, device, type, k0->sizes(), p) ||
      !pointers(args[1], n, device, type, k0->sizes(), p))
    Py_RETURN_NONE;
  return PyLong_FromLong(branches.reorder(p.data(), p.data() + n, (int)n, data<int32_t>(lens),
                                     data<int32_t>(parents), (int)W, (int)B, (int)k0->size(1),
                                     (int)k0->size(2), (int)k0->size(3), dt, (void*)stream));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"same", (PyCFunction)(void (*)())same, METH_FASTCALL,
     "same(list, buffer, first) -> device index (-1: not on a GPU)"},
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, "bind(addresses of the entry points)"},
    {"bind_branches", (PyCFunction)(void (*)())bind_branches, METH_FASTCALL,
     "bind_branches(addresses of the entry points)"},
    {"tree", (PyCFunction)(void (*)())tree, METH_FASTCALL, "tree attention, if in plain form"},
    {"verify", (PyCFunction)(void (*)())verify, METH_FASTCALL, "verification, if in plain form"},
    {"keep", (PyCFunction)(void (*)())keep, METH_FASTCALL, "the caches' move, if in plain form"},
    {"branch", (PyCFunction)(void (*)())branch, METH_FASTCALL,
     "attention behind shared prefixes, if in plain form"},
    {"select", (PyCFunction)(void (*)())select, METH_FASTCALL,
     "the beams' selection, if in plain form"},
    {"reorder", (PyCFunction)(void (*)())reorder, METH_FASTCALL,
     "the caches' reordering, if in plain form"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kf_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kf_torch(void) {
  PyObject* m = PyModule_Create(&module);
  // what it was built for, by the headers
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
