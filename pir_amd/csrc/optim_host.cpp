// Host half of pir_amd.optim: reads lists of tensors into the arrays that pir_adamw_step and pir_grad_norm take, and
// calls them.  One step of the reference's networks has some hundred tensors in each of four lists; reading their types,
// strides and addresses through Python takes 3 us a tensor, here 0.1 us; whether they overlap is found out here too.
//
// Every function answers NotImplemented where the tensors are not as the kernels want them.  The Python side then says
// what is wrong, or brings them into order and calls again.
#include <Python.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>
#include <algorithm>
#include <vector>
#include "../../include/pir_hip.h"

namespace {

using StepFn = decltype(&pir_adamw_step);
using StepBytesFn = decltype(&pir_adamw_workspace_bytes);
using NormFn = decltype(&pir_grad_norm);
using NormBytesFn = decltype(&pir_grad_norm_workspace_bytes);
using DecodeFn = decltype(&pir_moments8_decode);

// borrowed items of a list
struct Items {
  PyObject** at = nullptr;
  Py_ssize_t n = -1;
  explicit Items(PyObject* list) {
    if (!PyList_Check(list)) return;
    at = PySequence_Fast_ITEMS(list);
    n = PyList_GET_SIZE(list);
  }
};

// a plain dense tensor of this device, or null
const at::Tensor* tensor_of(PyObject* o, c10::Device dev) {
  if (!PyType_IsSubtype(Py_TYPE(o), (PyTypeObject*)THPVariableClass)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || t.device() != dev || t.is_neg() ||
      t.unsafeGetTensorImpl()->is_python_dispatch())
    return nullptr;
  return &t;
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PIR_F32;
    case at::kBFloat16: return PIR_BF16;
    case at::kHalf: return PIR_F16;
    default: return -1;
  }
}

bool same_layout(const at::Tensor& p, const at::Tensor& t) {
  if (p.sizes() != t.sizes()) return false;
  return p.is_contiguous() ? t.is_contiguous() : p.strides() == t.strides();
}

bool dense(const at::Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

char* address(const at::Tensor& t) { return (char*)t.unsafeGetTensorImpl()->mutable_data(); }

// whether these are the 8-bit moments of nb blocks as the kernels read them
bool coded(const at::Tensor& q, const at::Tensor& c, const at::Tensor& s, long nb) {
  return q.scalar_type() == at::kChar && c.scalar_type() == at::kByte && s.scalar_type() == at::kFloat && q.is_contiguous() &&
         c.is_contiguous() && s.is_contiguous() && q.dim() == 2 && q.size(0) == nb && q.size(1) == 256 && c.sizes() == q.sizes() &&
         s.dim() == 2 && s.size(0) == nb && s.size(1) == 2 && !(((size_t)address(q) | (size_t)address(c)) & 15) &&
         !((size_t)address(s) & 7);
}

// whether p's elements lie in the order that the state of its codes records, if it does
bool same_order(const at::Tensor& p, PyObject* state) {
  static PyObject* const key = PyUnicode_InternFromString("strides");
  PyObject* strides = PyDict_Check(state) ? PyDict_GetItem(state, key) : nullptr;
  if (!strides) return true;
  if (!PyTuple_Check(strides) || PyTuple_GET_SIZE(strides) != p.dim()) return false;
  for (int64_t k = 0; k < p.dim(); ++k) {
    const long x = PyLong_AsLong(PyTuple_GET_ITEM(strides, k));
    if (x == -1 && PyErr_Occurred()) PyErr_Clear();
    if (p.size(k) != 1 && p.stride(k) != x) return false;
  }
  return true;
}

// The memory of a step's tensors, in lists that are written (parameters, both moments, scales, step counts) or only read
// (gradients).  No byte that is written may belong to two tensors; those that are only read may share theirs.
class Memory {
  static constexpr size_t kWritten = (size_t)1 << 63;
  struct Span {
    size_t at, end;                              // kWritten in end
  };
  struct List {
    Span *from, *to;
    bool ascending, written;
    size_t lo, hi;
  };
  std::vector<Span> spans;
  std::vector<List> lists;

  static Span* merge(const Span* a, const Span* a_end, const Span* b, const Span* b_end, Span* out) {
    while (a != a_end && b != b_end) {           // without a branch on which comes first: lists lie among each other
      const bool second = b->at < a->at;
      *out++ = second ? *b : *a;
      b += second;
      a += !second;
    }
    out = std::copy(a, a_end, out);
    return std::copy(b, b_end, out);
  }

 public:
  enum { kParams, kGrads, kFirst, kSecond, kScales, kSteps, kLists };

  explicit Memory(Py_ssize_t n) : spans(kLists * n), lists(kLists) {
    for (int i = 0; i < kLists; ++i) lists[i] = {&spans[i * n], &spans[i * n], true, i != kGrads, ~(size_t)0, 0};
  }

  void add(int list, const void* at, long bytes) {
    if (!bytes) return;
    List& l = lists[list];
    const size_t start = (size_t)at, end = start + (size_t)bytes;
    l.ascending &= start >= l.hi;
    l.lo = std::min(l.lo, start);
    l.hi = std::max(l.hi, end);
    *l.to++ = {start, l.written ? end | kWritten : end};
  }

  // Lists that are in the order of memory and apart from all others (views of a buffer each) need no more than their
  // ends.  Others, as a model's parameters and their states lie, are merged in that order: 4 us for the 500 of a training iteration.
  bool disjoint() {
    std::vector<std::pair<Span*, Span*>> runs;
    for (const List& l : lists) {
      bool among = l.written && !l.ascending;
      for (const List& o : lists) among |= &o != &l && l.lo < o.hi && o.lo < l.hi;
      if (!among) continue;
      if (!l.ascending) std::sort(l.from, l.to, [](const Span& x, const Span& y) { return x.at < y.at; });
      runs.emplace_back(l.from, l.to);
    }
    if (runs.empty()) return true;
    std::vector<Span> other(spans.size());
    Span* to = other.data();
    while (runs.size() > 1) {                    // pairs of runs, from one buffer to the other and back
      Span* out = to;
      size_t k = 0;
      for (size_t i = 0; i < runs.size(); i += 2) {
        const auto a = runs[i], b = i + 1 < runs.size() ? runs[i + 1] : std::make_pair(a.second, a.second);
        Span* const end = merge(a.first, a.second, b.first, b.second, out);
        runs[k++] = {out, end};
        out = end;
      }
      runs.resize(k);
      to = to == other.data() ? spans.data() : other.data();
    }
    size_t written = 0, read = 0;                // where what came so far ends
    for (const Span* s = runs[0].first; s != runs[0].second; ++s) {
      const bool w = s->end & kWritten;
      if (s->at < written || (w && s->at < read)) return false;
      size_t& end = w ? written : read;
      end = std::max(end, s->end & ~kWritten);
    }
    return true;
  }
};

struct Lists {
  std::vector<void*> p, g, m, v, s, t;
  std::vector<long> numels;
  std::vector<int> dtypes;
};

PyObject* fail(const char* what, int code) {
  return PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", what, code);
}

// adamw_step(fn, bytes_fn, params, grads, exp_avgs, exp_avg_sqs, scales | None, steps: tensor or list, groups: address of
// an int for each tensor | 0, list of (lr, beta1, beta2, eps, weight decay, address of the lr on the device | 0),
// max_norm, skip_nonfinite, want_norm, device index, stream, states: list of dictionaries | None) -> norm | None
PyObject* step(PyObject*, PyObject* args) {
  unsigned long long fn, bytes_fn, groups_at, stream;
  PyObject *params, *grads, *ms, *vs, *ss, *ts, *hypers, *states;
  int skip, want, index;
  double max_norm;
  if (!PyArg_ParseTuple(args, "KKOOOOOOKO!dppiKO", &fn, &bytes_fn, &params, &grads, &ms, &vs, &ss, &ts, &groups_at,
                        &PyList_Type, &hypers, &max_norm, &skip, &want, &index, &stream, &states))
    return nullptr;
  try {
    const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)index);
    const Items P(params), G(grads), M(ms), V(vs), S(ss), T(ts), D(states);
    const Py_ssize_t n = P.n;
    if (n < 1 || G.n != n || M.n != n || V.n != n || (ss != Py_None && S.n != n) || (D.n >= 0 && D.n != n))
      Py_RETURN_NOTIMPLEMENTED;
    Lists a;
    for (auto* x : {&a.p, &a.g, &a.m, &a.v, &a.s, &a.t}) x->resize(n);
    a.numels.resize(n);
    a.dtypes.resize(n);
    Memory memory(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor *p = tensor_of(P.at[i], dev), *g = tensor_of(G.at[i], dev), *m = tensor_of(M.at[i], dev),
                       *v = tensor_of(V.at[i], dev);
      if (!p || !g || !m || !v) Py_RETURN_NOTIMPLEMENTED;
      const long numel = p->numel();
      const int type = dtype_of(*p);
      if (type < 0 || g->scalar_type() != p->scalar_type() || !dense(*p) || !same_layout(*p, *g)) Py_RETURN_NOTIMPLEMENTED;
      if (((size_t)address(*p) | (size_t)address(*g)) & (p->element_size() - 1)) Py_RETURN_NOTIMPLEMENTED;
      char *am = address(*m), *av = address(*v), *as = nullptr;
      PyObject* so = ss == Py_None ? Py_None : S.at[i];
      if (so == Py_None) {
        if (m->scalar_type() != at::kFloat || v->scalar_type() != at::kFloat || !same_layout(*p, *m) || !same_layout(*p, *v))
          Py_RETURN_NOTIMPLEMENTED;
        memory.add(Memory::kFirst, am, 4 * numel);
        memory.add(Memory::kSecond, av, 4 * numel);
      } else {
        const at::Tensor* s = tensor_of(so, dev);
        const long nb = (numel + 255) / 256;
        if (!s || !coded(*m, *v, *s, nb) || (D.n >= 0 && !same_order(*p, D.at[i]))) Py_RETURN_NOTIMPLEMENTED;
        as = address(*s);
        if (!as) as = (char*)16;                 // no blocks: 8-bit all the same
        memory.add(Memory::kFirst, am, 256 * nb);
        memory.add(Memory::kSecond, av, 256 * nb);
        memory.add(Memory::kScales, as, 8 * nb);
      }
      a.p[i] = address(*p);
      a.g[i] = address(*g);
      a.m[i] = am;
      a.v[i] = av;
      a.s[i] = as;
      a.numels[i] = numel;
      memory.add(Memory::kParams, a.p[i], numel * (long)p->element_size());
      memory.add(Memory::kGrads, a.g[i], numel * (long)p->element_size());
      a.dtypes[i] = type;
    }
    if (T.n >= 0) {
      if (T.n != n) Py_RETURN_NOTIMPLEMENTED;
      for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor* t = tensor_of(T.at[i], dev);
        if (!t || t->scalar_type() != at::kFloat || t->numel() != 1) Py_RETURN_NOTIMPLEMENTED;
        a.t[i] = address(*t);
        memory.add(Memory::kSteps, a.t[i], 4);
      }
    } else {
      const at::Tensor* t = tensor_of(ts, dev);
      if (!t || t->scalar_type() != at::kFloat || t->numel() != n || !t->is_contiguous()) Py_RETURN_NOTIMPLEMENTED;
      for (Py_ssize_t i = 0; i < n; ++i) a.t[i] = address(*t) + 4 * i;
      memory.add(Memory::kSteps, a.t[0], 4 * n);
    }
    if (!memory.disjoint()) Py_RETURN_NOTIMPLEMENTED;
    std::vector<PirAdamwGroup> table(PyList_GET_SIZE(hypers));
    for (size_t k = 0; k < table.size(); ++k) {
      unsigned long long lr = 0;
      PirAdamwGroup& h = table[k];
      if (!PyArg_ParseTuple(PyList_GET_ITEM(hypers, k), "dddddK", &h.lr, &h.beta1, &h.beta2, &h.eps, &h.weight_decay, &lr))
        return nullptr;
      h.lr_device = (const float*)lr;
    }
    std::vector<int> zeros;
    if (!groups_at) zeros.resize(n, 0);
    const int with_norm = want || skip || max_norm > 0.0;
    const c10::OptionalDeviceGuard guard(dev);
    const size_t size = ((StepBytesFn)bytes_fn)((int)n, a.numels.data(), with_norm);
    const at::Tensor work = at::empty({(long)size}, at::TensorOptions().dtype(at::kByte).device(dev));
    at::Tensor norm;
    if (with_norm) norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    const int code = ((StepFn)fn)((int)n, a.p.data(), (const void* const*)a.g.data(), a.m.data(), a.v.data(),
                                  ss == Py_None ? nullptr : (float* const*)a.s.data(), (float* const*)a.t.data(),
                                  a.numels.data(), a.dtypes.data(), groups_at ? (const int*)groups_at : zeros.data(),
                                  table.data(), (int)table.size(), max_norm, skip,
                                  with_norm ? norm.data_ptr<float>() : nullptr, work.data_ptr(), size, (void*)stream);
    if (code != PIR_OK) return fail("pir_adamw_step", code);
    for (Py_ssize_t i = 0; i < n; ++i) {         // autograd and the networks' packed weights go by the version
      const at::Tensor& p = THPVariable_Unpack(P.at[i]);
      if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
    }
    if (!with_norm) Py_RETURN_NONE;
    return THPVariable_Wrap(norm);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// grad_norm(fn, bytes_fn, tensors, device index, stream) -> [total, norm of each]
PyObject* norm(PyObject*, PyObject* args) {
  unsigned long long fn, bytes_fn, stream;
  PyObject* tensors;
  int index;
  if (!PyArg_ParseTuple(args, "KKOiK", &fn, &bytes_fn, &tensors, &index, &stream)) return nullptr;
  try {
    const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)index);
    const Items G(tensors);
    if (G.n < 1) Py_RETURN_NOTIMPLEMENTED;
    std::vector<void*> g(G.n);
    std::vector<long> numels(G.n);
    std::vector<int> dtypes(G.n);
    for (Py_ssize_t i = 0; i < G.n; ++i) {
      const at::Tensor* t = tensor_of(G.at[i], dev);
      if (!t || (dtypes[i] = dtype_of(*t)) < 0 || !dense(*t) || ((size_t)address(*t) & (t->element_size() - 1)))
        Py_RETURN_NOTIMPLEMENTED;
      g[i] = address(*t);
      numels[i] = t->numel();
    }
    const c10::OptionalDeviceGuard guard(dev);
    const size_t size = ((NormBytesFn)bytes_fn)((int)G.n, numels.data());
    const at::Tensor work = at::empty({(long)size}, at::TensorOptions().dtype(at::kByte).device(dev));
    const at::Tensor out = at::empty({G.n + 1}, at::TensorOptions().dtype(at::kFloat).device(dev));
    float* o = out.data_ptr<float>();
    const int code = ((NormFn)fn)((int)G.n, (const void* const*)g.data(), numels.data(), dtypes.data(), o, o + 1,
                                  work.data_ptr(), size, (void*)stream);
    if (code != PIR_OK) return fail("pir_grad_norm", code);
    return THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// moments8_decode(fn, exp_avg, exp_avg_sq, scales, type, device index, stream) -> (m, v)
PyObject* decode(PyObject*, PyObject* args) {
  unsigned long long fn, stream;
  PyObject *qo, *co, *so;
  int type, index;
  if (!PyArg_ParseTuple(args, "KOOOiiK", &fn, &qo, &co, &so, &type, &index, &stream)) return nullptr;
  try {
    const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)index);
    const at::Tensor *q = tensor_of(qo, dev), *c = tensor_of(co, dev), *s = tensor_of(so, dev);
    if (!q || !c || !s || !coded(*q, *c, *s, q->dim() ? q->size(0) : 0)) Py_RETURN_NOTIMPLEMENTED;
    const c10::OptionalDeviceGuard guard(dev);
    const auto as = at::TensorOptions().dtype(type == PIR_F32 ? at::kFloat : type == PIR_BF16 ? at::kBFloat16 : at::kHalf).device(dev);
    const at::Tensor m = at::empty(q->sizes(), as), v = at::empty(q->sizes(), as);
    const int code = ((DecodeFn)fn)(q->size(0), (const signed char*)address(*q), (const unsigned char*)address(*c),
                                    (const float*)address(*s), type, m.data_ptr(), v.data_ptr(), (void*)stream);
    if (code != PIR_OK) return fail("pir_moments8_decode", code);
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(m));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
    return pair;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {{"adamw_step", step, METH_VARARGS, nullptr},
                         {"grad_norm", norm, METH_VARARGS, nullptr},
                         {"moments8_decode", decode, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_optim_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__optim_host() { return PyModule_Create(&module); }
