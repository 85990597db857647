// Lists of tensors as the C ABI takes them: an optimizer step has hundreds of tensors
// in five lists, and a look at each from Python costs more than the step (320 adapter
// factors: 550 us of checks and addresses, 17 here).  Everything that the kernels rely
// on is checked: types, devices, sizes, layouts, memory that meets.

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <vector>

#include "compact_amd.h"

namespace {

// A violated condition: AssertionError, as the wrappers' other checks.
struct Refused {
  std::string why;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused{why}; }

std::string describe(const at::Tensor& t) {
  std::string s = std::string(c10::toString(t.scalar_type())) + " [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  s += "] strides [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
  return s + "] on " + t.device().str();
}

// A list or tuple of tensors (borrowed).
class List {
 public:
  List(PyObject* o, const char* name) : name_(name) {
    if (o == Py_None) return;
    fast_ = PySequence_Fast(o, "a sequence of tensors expected");
    if (!fast_) throw python_error();
    n_ = PySequence_Fast_GET_SIZE(fast_);
    items_ = PySequence_Fast_ITEMS(fast_);
  }
  List(const List&) = delete;
  ~List() { Py_XDECREF(fast_); }
  explicit operator bool() const { return fast_ != nullptr; }
  int64_t size() const { return n_; }
  const char* name() const { return name_; }
  PyObject* object(int64_t i) const { return items_[i]; }
  const at::Tensor& operator[](int64_t i) const {
    if (!THPVariable_CheckExact(items_[i]) && !THPVariable_Check(items_[i]))
      refuse(std::string(name_) + ": tensors expected");
    const at::Tensor& t = THPVariable_Unpack(items_[i]);
    if (t.layout() != at::kStrided) refuse(std::string(name_) + ": strided tensors expected");
    return t;
  }

 private:
  const char* name_;
  PyObject* fast_ = nullptr;
  Py_ssize_t n_ = 0;
  PyObject** items_ = nullptr;
};

// Whether a tensor's elements fill its memory once, in whatever order of its axes.
bool dense(const at::Tensor& t) {
  return t.is_contiguous() || t.unsafeGetTensorImpl()->is_non_overlapping_and_dense_default();
}
// Whether dense tensors of one shape lie alike.
bool alike(const at::Tensor& a, const at::Tensor& b) {
  return (a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides();
}

int code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}

void expect(const at::Tensor& t, const at::Tensor& p, at::ScalarType type, const char* name) {
  if (t.scalar_type() != type || t.device() != p.device() || t.sizes() != p.sizes() || !alike(p, t))
    refuse(std::string(name) + ": " + c10::toString(type) + " that lies as " + describe(p) +
           " expected, got " + describe(t));
}
void expect_bytes(const at::Tensor& t, const at::Tensor& p, int64_t n, const char* name) {
  if (t.scalar_type() != at::kByte || t.device() != p.device() || t.numel() != n ||
      !t.is_contiguous())
    refuse(std::string(name) + ": contiguous Byte of " + std::to_string(n) + " on " +
           p.device().str() + " expected, got " + describe(t));
}

// Addresses met so far; a hash table in place of a set of the library's, which allocates
// for each.
class Addresses {
 public:
  explicit Addresses(int64_t most) {
    size_t n = 16;
    while (n < static_cast<size_t>(2 * most)) n *= 2;
    table_.resize(n);
  }
  // Whether p is new.
  bool add(const void* p) {
    const size_t mask = table_.size() - 1;
    size_t at = (reinterpret_cast<uintptr_t>(p) >> 4) * 0x9E3779B97F4A7C15ull >> 32 & mask;
    while (table_[at]) {
      if (table_[at] == p) return false;
      at = (at + 1) & mask;
    }
    table_[at] = p;
    return true;
  }
  bool has(const void* p) const {
    const size_t mask = table_.size() - 1;
    size_t at = (reinterpret_cast<uintptr_t>(p) >> 4) * 0x9E3779B97F4A7C15ull >> 32 & mask;
    while (table_[at] && table_[at] != p) at = (at + 1) & mask;
    return table_[at];
  }

 private:
  std::vector<const void*> table_;
};

constexpr int64_t kBlock = 128;   // elements of an 8-bit moment that share a scale

// One of a step's lists: where its tensors' addresses stand, and the bytes of `block` elements.
struct Written {
  void* cpt_adamw_tensor::*address;
  int64_t unit, block;
};
struct Range {
  uintptr_t at, end;
  int64_t tensor;
};
bool before(const Range& a, const Range& b) { return a.at < b.at; }
Range range(const void* p, int64_t bytes, int64_t i) {
  const auto at = reinterpret_cast<uintptr_t>(p);
  return Range{at, at + (at ? bytes : 0), i};
}
// Refuses a step whose tensors' memory meets: what is written lies apart from all else, or its
// elements depend on which thread comes first.  A gradient may be its parameter or moment
// itself, whose elements are each read before they are written.
void check_apart(const List& p, const std::vector<cpt_adamw_tensor>& rows, int64_t size,
                 int64_t grad_size, bool bits8, bool grads) {
  const int64_t moment = bits8 ? 1 : 4;
  const Written lists[] = {{&cpt_adamw_tensor::p, size, 1},
                           {&cpt_adamw_tensor::m, moment, 1},
                           {&cpt_adamw_tensor::v, moment, 1},
                           {&cpt_adamw_tensor::m_scale, 1, kBlock},
                           {&cpt_adamw_tensor::v_scale, 1, kBlock},
                           {&cpt_adamw_tensor::master, 4, 1}};
  const auto at = [&](const Written& l, int64_t i) {
    return range(rows[i].*l.address, (rows[i].n + l.block - 1) / l.block * l.unit, i);
  };
  const int64_t count = rows.size();
  // lists cut from a buffer each lie in order, one list behind the other: nothing to sort
  bool apart = !grads;
  Range spans[6];
  int n = 0;
  for (const Written& l : lists) {
    Range span{0, 0, 0};
    for (int64_t i = 0; i < count && apart; ++i) {
      const Range r = at(l, i);
      if (r.at == r.end) continue;
      apart = r.at >= span.end;
      span = Range{span.at ? span.at : r.at, r.end, 0};
    }
    for (int k = 0; k < n; ++k) apart &= span.end <= spans[k].at || span.at >= spans[k].end;
    if (span.end) spans[n++] = span;
  }
  if (apart) return;
  std::vector<Range> all;
  all.reserve(count * 6);
  for (const Written& l : lists)
    for (int64_t i = 0; i < count; ++i)
      if (const Range r = at(l, i); r.at != r.end) all.push_back(r);
  std::sort(all.begin(), all.end(), before);
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].at < all[i - 1].end)
      refuse("two of a step's tensors share memory: " + describe(p[all[i].tensor]));
  for (int64_t i = 0; grads && i < count; ++i) {
    const Range r = range(rows[i].g, rows[i].n * grad_size, i);
    if (r.at == r.end) continue;        // one that will be copied has no address
    auto w = std::upper_bound(all.begin(), all.end(), r, before);
    if (w != all.begin()) --w;
    for (; w != all.end() && w->at < r.end; ++w)
      if (w->end > r.at && (w->at != r.at || w->end != r.end || w->tensor != r.tensor))
        refuse("grads: a step writes to the memory of that for " + describe(p[i]));
  }
}

template <class F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_AssertionError, r.why.c_str());
  } catch (python_error& e) {
    e.persist();
    e.restore();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// {table, its address, elements, more...}
PyObject* result(const std::vector<cpt_adamw_tensor>& rows, int64_t elements, int dtype,
                 int grad_dtype, PyObject* more) {
  PyObject* table = PyBytes_FromStringAndSize(reinterpret_cast<const char*>(rows.data()),
                                              rows.size() * sizeof(cpt_adamw_tensor));
  if (!table) throw python_error();
  return Py_BuildValue("(NLLiiN)", table,
                       static_cast<long long>(reinterpret_cast<intptr_t>(PyBytes_AS_STRING(table))),
                       static_cast<long long>(elements), dtype, grad_dtype, more);
}

// The steps' numbers, or addresses of counts on the device.
void steps(PyObject* step, std::vector<cpt_adamw_tensor>& rows, const at::Device& device) {
  const int64_t n = rows.size();
  auto number = [](PyObject* o) {
    if (!PyLong_Check(o)) refuse("step: whole numbers expected");
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < 1) refuse("step=" + std::to_string(v) + ": the first is 1");
    return v;
  };
  auto counts = [&](PyObject* o, int64_t m) -> int64_t* {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kLong || t.numel() != m || !t.is_contiguous() ||
        t.device() != device)
      refuse("step: " + std::to_string(m) + " contiguous Long on " + device.str() +
             " expected, got " + describe(t));
    return static_cast<int64_t*>(t.data_ptr());
  };
  if (THPVariable_Check(step)) {
    int64_t* at = counts(step, n);
    for (int64_t i = 0; i < n; ++i) rows[i].step_device = at + i;
    return;
  }
  if (PyLong_Check(step)) {
    const long long v = number(step);
    for (auto& r : rows) r.step = v;
    return;
  }
  const List list(step, "step");
  if (list.size() != n) refuse("step: " + std::to_string(n) + " expected");
  const bool on_device = n && THPVariable_Check(list.object(0));
  Addresses seen(n);
  for (int64_t i = 0; i < n; ++i) {
    if (!on_device) {
      rows[i].step = number(list.object(i));
      continue;
    }
    if (!THPVariable_Check(list.object(i))) refuse("step: a count each expected");
    rows[i].step_device = counts(list.object(i), 1);
    if (!seen.add(rows[i].step_device))
      refuse("step: a count of its own for each parameter expected");
  }
}

// adamw_table(params, grads, exp_avgs, exp_avg_sqs, m_scales, v_scales, masters, step,
// written): (table, address, elements, dtype, grads' dtype, [indices of gradients that lie
// otherwise than their parameters]).  written: the moments are, and lie apart.
PyObject* adamw_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 9) refuse("nine arguments expected");
    const List p(a[0], "params"), g(a[1], "grads"), m(a[2], "exp_avgs"), v(a[3], "exp_avg_sqs"),
        ms(a[4], "m_scales"), vs(a[5], "v_scales"), w(a[6], "masters");
    for (const List* l : {&g, &m, &v, &ms, &vs, &w})
      if (*l && l->size() != p.size())
        refuse(std::string(l->name()) + ": " + std::to_string(p.size()) +
               " tensors expected, got " + std::to_string(l->size()));
    const int64_t count = p.size();
    if (count == 0 || !g || !m || !v) refuse("adamw_table: tensors expected");
    if (static_cast<bool>(ms) != static_cast<bool>(vs))
      refuse("m_scales and v_scales belong together");
    std::vector<cpt_adamw_tensor> rows(count);
    const bool written = PyObject_IsTrue(a[8]) == 1;
    // tensors in storages of their own are apart
    Addresses storages(6 * count);
    bool shared = false;
    const auto write = [&](const at::Tensor& t) {
      if (t.numel()) shared |= !storages.add(t.storage().data());
    };
    const at::ScalarType type = p[0].scalar_type(), grad_type = g[0].scalar_type();
    const at::Device device = p[0].device();
    if (code(type) < 0) refuse("params: unsupported " + describe(p[0]));
    if (grad_type != type && grad_type != at::kFloat)
      refuse("grads: the parameters' type or Float expected, got " + describe(g[0]));
    if (w && type == at::kFloat) refuse("masters: of 16-bit parameters");
    THPObjectPtr otherwise(PyList_New(0));
    if (!otherwise) throw python_error();
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
      const at::Tensor &pi = p[i], &gi = g[i], &mi = m[i], &vi = v[i];
      cpt_adamw_tensor& r = rows[i];
      if (pi.scalar_type() != type || pi.device() != device)
        refuse("params: " + describe(p[0]) + " and " + describe(pi));
      if (gi.scalar_type() != grad_type || gi.device() != device)
        refuse("grads: " + describe(g[0]) + " and " + describe(gi));
      if (gi.sizes() != pi.sizes())
        refuse("grads: " + describe(gi) + " for " + describe(pi));
      if (!dense(pi)) refuse("params: dense memory expected, got " + describe(pi));
      r.n = pi.numel();
      total += r.n;
      r.p = pi.data_ptr();
      write(pi);
      if (alike(pi, gi)) {
        r.g = gi.data_ptr();
      } else {
        THPObjectPtr at(PyLong_FromLongLong(i));
        if (!at || PyList_Append(otherwise.get(), at.get())) throw python_error();
      }
      if (ms) {
        const int64_t blocks = (r.n + kBlock - 1) / kBlock;
        const at::Tensor &msi = ms[i], &vsi = vs[i];
        expect_bytes(mi, pi, r.n, m.name());
        expect_bytes(vi, pi, r.n, v.name());
        expect_bytes(msi, pi, blocks, ms.name());
        expect_bytes(vsi, pi, blocks, vs.name());
        r.m_scale = msi.data_ptr();
        r.v_scale = vsi.data_ptr();
        if (written) write(msi), write(vsi);
      } else {
        expect(mi, pi, at::kFloat, m.name());
        expect(vi, pi, at::kFloat, v.name());
      }
      r.m = mi.data_ptr();
      r.v = vi.data_ptr();
      if (w) {
        const at::Tensor& wi = w[i];
        expect(wi, pi, at::kFloat, w.name());
        r.master = wi.data_ptr();
        write(wi);
      }
      if (written) write(mi), write(vi);
    }
    bool grads = false;
    for (int64_t i = 0; i < count && !grads; ++i)
      grads = rows[i].g && rows[i].n && storages.has(g[i].storage().data());
    if (written && (shared || grads))
      check_apart(p, rows, p[0].element_size(), g[0].element_size(), static_cast<bool>(ms), grads);
    steps(a[7], rows, device);
    return result(rows, total, code(type), code(grad_type), otherwise.release());
  });
}

// grads_table(grads): (table, address, elements, dtype, dtype, [indices of gradients that
// do not fill their memory once])
PyObject* grads_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1) refuse("one argument expected");
    const List g(a[0], "grads");
    if (g.size() == 0) refuse("grads_table: tensors expected");
    std::vector<cpt_adamw_tensor> rows(g.size());
    const at::ScalarType type = g[0].scalar_type();
    const at::Device device = g[0].device();
    if (code(type) < 0) refuse("grads: unsupported " + describe(g[0]));
    THPObjectPtr otherwise(PyList_New(0));
    if (!otherwise) throw python_error();
    int64_t total = 0;
    for (int64_t i = 0; i < g.size(); ++i) {
      const at::Tensor& t = g[i];
      if (t.scalar_type() != type || t.device() != device)
        refuse("grads: " + describe(g[0]) + " and " + describe(t));
      rows[i].n = t.numel();
      rows[i].g = t.data_ptr();
      total += rows[i].n;
      if (!dense(t)) {
        THPObjectPtr at(PyLong_FromLongLong(i));
        if (!at || PyList_Append(otherwise.get(), at.get())) throw python_error();
      }
    }
    return result(rows, total, code(type), code(type), otherwise.release());
  });
}

// one_kind(tensors): whether they share type and device
PyObject* one_kind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1) refuse("one argument expected");
    const List l(a[0], "tensors");
    for (int64_t i = 1; i < l.size(); ++i)
      if (l[i].scalar_type() != l[0].scalar_type() || l[i].device() != l[0].device())
        Py_RETURN_FALSE;
    Py_RETURN_TRUE;
  });
}

// state_forms(states): (whether one is empty, all states' form or -1, what their counts are or
// -1).  A form is 1 where moments are in 8 bits and 2 where there is an fp32 copy; counts are
// 0 numbers and 1 tensors.
PyObject* state_forms(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    static PyObject* const scale = PyUnicode_InternFromString("m_scale");
    static PyObject* const master = PyUnicode_InternFromString("master");
    static PyObject* const step = PyUnicode_InternFromString("step");
    if (n != 1 || !PyList_Check(a[0])) refuse("a list expected");
    int form = -2, counts = -2, empty = 0;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) {
      PyObject* s = PyList_GET_ITEM(a[0], i);
      if (!PyDict_Check(s)) refuse("dicts of a state expected");
      empty |= PyDict_GET_SIZE(s) == 0;
      const int f = PyDict_Contains(s, scale) | PyDict_Contains(s, master) << 1;
      PyObject* at = PyDict_GetItemWithError(s, step);
      if (f < 0 || PyErr_Occurred()) throw python_error();
      const int c = at && PyLong_Check(at) ? 0 : 1;
      form = form == -2 || form == f ? f : -1;
      counts = counts == -2 || counts == c ? c : -1;
    }
    return Py_BuildValue("(iii)", empty, form, counts);
  });
}

// bump_versions(tensors): they were written to
PyObject* bump_versions(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1) refuse("one argument expected");
    const List l(a[0], "tensors");
    for (int64_t i = 0; i < l.size(); ++i)
      if (!l[i].is_inference()) l[i].unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
  });
}

#define ENTRY(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(adamw_table), ENTRY(grads_table), ENTRY(one_kind),
                         ENTRY(state_forms), ENTRY(bump_versions), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lists", "lists of tensors for the C ABI", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lists(void) { return PyModule_Create(&module); }
