// Reads lists of tensors at once: addresses and sizes, with the checks that allow a launch on them.
// From Python each attribute of each tensor costs 0.07 us, 20 of them a parameter; here all of
// a parameter's take 0.05 us.  Only this module knows torch's types: what it returns are the rows
// of structures that the C ABI of include/tidegs_amd.h takes.
//
// Both functions return None where a tensor is not what most are (contiguous, on one GPU, of
// fitting types and sizes): the caller then checks them one by one, which names the fault.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/tidegs_amd.h"

namespace {

struct List {  // a list or tuple of tensors
  PyObject* fast;
  explicit List(PyObject* o) : fast(PySequence_Fast(o, "lists of tensors are needed")) {}
  ~List() { Py_XDECREF(fast); }
  List(const List&) = delete;
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
  // The tensor, or null for another object.
  const at::Tensor* operator[](Py_ssize_t i) const {
    PyObject* o = PySequence_Fast_GET_ITEM(fast, i);
    return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
  }
};

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TGS_F32;
    case at::kBFloat16: return TGS_BF16;
    case at::kHalf: return TGS_F16;
    default: return -1;
  }
}

bool plain(const at::Tensor* t, c10::Device device) {
  return t && t->layout() == at::kStrided && t->device() == device && t->is_contiguous();
}

// The device of all tensors, from the first; false if that is no GPU.
bool device_of(const at::Tensor* t, c10::Device& device) {
  if (!t) return false;
  device = t->device();
  return device.is_cuda();
}

PyObject* answer(c10::Device device, const void* rows, size_t bytes) {
  return Py_BuildValue("(iy#)", (int)device.index(), (const char*)rows, (Py_ssize_t)bytes);
}

// spans(tensors) -> (device index, rows of tgs_span) or None
PyObject* spans(PyObject*, PyObject* arg) try {
  const List list(arg);
  if (!list.fast) return nullptr;
  const Py_ssize_t n = list.size();
  c10::Device device(c10::kCPU);
  if (n == 0 || !device_of(list[0], device)) Py_RETURN_NONE;
  std::vector<tgs_span> rows(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = list[i];
    if (!plain(t, device) || dtype_of(*t) < 0) Py_RETURN_NONE;
    rows[i] = {t->const_data_ptr(), (uint64_t)t->numel(), dtype_of(*t)};
  }
  return answer(device, rows.data(), n * sizeof(tgs_span));
} catch (const std::exception&) {  // (a tensor without memory, as a traced one)
  Py_RETURN_NONE;
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, scales, scales, block, numbers, groups)
// -> (device index, rows of tgs_adamw_tensor) or None.  scales: lists, or None for 32-bit states;
// numbers and groups: sequences of integers.
PyObject* adamw(PyObject*, PyObject* const* args, Py_ssize_t count) try {
  if (count != 9) {
    PyErr_SetString(PyExc_TypeError, "adamw takes nine arguments");
    return nullptr;
  }
  const bool eight = args[4] != Py_None;
  const uint64_t block = PyLong_AsUnsignedLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  const List p_(args[0]), g_(args[1]), m_(args[2]), v_(args[3]), ms_(eight ? args[4] : args[2]),
      vs_(eight ? args[5] : args[3]), numbers(args[7]), groups(args[8]);
  const List* all[] = {&p_, &g_, &m_, &v_, &ms_, &vs_, &numbers, &groups};
  for (const List* l : all)
    if (!l->fast) return nullptr;
  const Py_ssize_t n = p_.size();
  for (const List* l : all)
    if (l->size() != n) {
      PyErr_SetString(PyExc_ValueError, "lists of one length are needed");
      return nullptr;
    }
  c10::Device device(c10::kCPU);
  if (n == 0 || !device_of(p_[0], device)) Py_RETURN_NONE;
  std::vector<tgs_adamw_tensor> rows(n);
  std::vector<const void*> written;
  written.reserve((eight ? 5 : 3) * n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor *p = p_[i], *g = g_[i], *m = m_[i], *v = v_[i];
    if (!plain(p, device) || !plain(g, device) || !plain(m, device) || !plain(v, device))
      Py_RETURN_NONE;
    if (dtype_of(*p) < 0 || g->scalar_type() != p->scalar_type() || g->sizes() != p->sizes() ||
        m->sizes() != p->sizes() || v->sizes() != p->sizes() ||
        m->scalar_type() != (eight ? at::kFloat8_e4m3fn : at::kFloat) ||
        v->scalar_type() != (eight ? at::kFloat8_e5m2 : at::kFloat))
      Py_RETURN_NONE;
    tgs_adamw_tensor& r = rows[i];
    r = {};
    r.n = (uint64_t)p->numel();
    r.param = p->mutable_data_ptr();
    r.grad = g->const_data_ptr();
    r.exp_avg = m->mutable_data_ptr();
    r.exp_avg_sq = v->mutable_data_ptr();
    r.dtype = dtype_of(*p);
    if (eight) {
      const at::Tensor *ms = ms_[i], *vs = vs_[i];
      const int64_t blocks = (int64_t)((r.n + block - 1) / block);
      for (const at::Tensor* s : {ms, vs})
        if (!plain(s, device) || s->dim() != 1 || s->numel() != blocks ||
            s->scalar_type() != at::kFloat)
          Py_RETURN_NONE;
      r.exp_avg_scale = (float*)ms->mutable_data_ptr();
      r.exp_avg_sq_scale = (float*)vs->mutable_data_ptr();
    }
    r.number = (uint32_t)PyLong_AsUnsignedLong(PySequence_Fast_GET_ITEM(numbers.fast, i));
    r.group = (uint32_t)PyLong_AsUnsignedLong(PySequence_Fast_GET_ITEM(groups.fast, i));
    if (PyErr_Occurred()) return nullptr;
    if (r.n) {
      written.insert(written.end(), {r.param, r.exp_avg, r.exp_avg_sq});
      if (eight) written.insert(written.end(), {r.exp_avg_scale, r.exp_avg_sq_scale});
    }
  }
  std::sort(written.begin(), written.end());
  if (std::adjacent_find(written.begin(), written.end()) != written.end()) Py_RETURN_NONE;
  return answer(device, rows.data(), n * sizeof(tgs_adamw_tensor));
} catch (const std::exception&) {
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"spans", spans, METH_O, "(device index, rows of tgs_span) of a list of tensors, or None"},
    {"adamw", (PyCFunction)(void (*)(void))adamw, METH_FASTCALL,
     "(device index, rows of tgs_adamw_tensor) of lists of tensors, or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists(void) { return PyModule_Create(&module); }
