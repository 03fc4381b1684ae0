// Group norm as a node of torch's autograd graph.  Both directions of few values take 65 us, most
// of them torch's engine; with a Function in Python, whose backward the engine's thread has to take
// the interpreter for, they took 107 (3 x 241x137x48 float32: 77 and 125).  The launches are
// those of the C ABI (include/tidegs_amd.h), whose addresses `bind` is given; arguments have been
// checked by tidegs_amd.decoder_ops.group_norm.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/tidegs_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
  decltype(&tgs_last_error) last_error;
  decltype(&tgs_group_norm_stats_size) stats_size;
  decltype(&tgs_group_norm_fwd_workspace_size) fwd_workspace_size;
  decltype(&tgs_group_norm_fwd) fwd;
  decltype(&tgs_group_norm_bwd_workspace_size) bwd_workspace_size;
  decltype(&tgs_group_norm_bwd) bwd;
} abi;

void check(int status, const char* name) {
  TORCH_CHECK(status == 0, name, " failed (code ", status, "): ", abi.last_error());
}

int32_t dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? TGS_F32
                                       : t.scalar_type() == at::kBFloat16 ? TGS_BF16 : TGS_F16;
}

// x [samples, ..., width] as samples of pixels, in place where its pixels lie at one pitch.
struct Pixels {
  Tensor x;
  int64_t sample, pitch;  // distances of samples and of pixels
  explicit Pixels(const Tensor& t) : x(t) {
    const int64_t width = t.size(-1);
    if (!t.is_contiguous()) {
      int64_t first = 0, inner = 0;  // the pixels' pitch, and how many the dimensions so far have
      bool even = true;
      for (int64_t d = t.dim() - 2; d >= 1 && even; --d) {
        if (t.size(d) == 1) continue;
        if (!inner) first = t.stride(d), inner = 1;
        even = t.stride(d) == first * inner;
        inner *= t.size(d);
      }
      if (even && (t.stride(-1) == 1 || width == 1) && (!inner || first >= width)) {
        sample = t.stride(0);
        pitch = std::max(first, width);
        return;
      }
      x = t.contiguous();
    }
    sample = t.size(0) ? t.numel() / t.size(0) : 0;
    pitch = width;
  }
};

struct Sizes {
  uint64_t samples, pixels;
  uint32_t width, groups;
  int32_t dtype;
  Sizes(const Tensor& x, int64_t n_groups)
      : samples(x.size(0)), pixels(1), width(x.size(-1)), groups(n_groups), dtype(dtype_of(x)) {
    for (int64_t d = 1; d < x.dim() - 1; ++d) pixels *= x.size(d);
  }
  template <typename Q>
  uint64_t ask(Q* query) const { return query(samples, pixels, width, groups, dtype); }
};

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* target(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

Tensor bytes(uint64_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

tgs_stream_t stream_of(const Tensor& x) {
  return (tgs_stream_t)c10::hip::getCurrentHIPStream(x.device().index()).stream();
}

int32_t weight_dtype(const Sizes& sizes, const Tensor& weight, const Tensor& bias) {
  const Tensor& w = weight.defined() ? weight : bias;
  return w.defined() ? dtype_of(w) : sizes.dtype;
}

// Whether t is a leaf whose gradients are gathered on the default stream: by the node that an eager
// graph made there, as long as that graph lives.
bool gathered_by_default(const Tensor& t) {
  if (!t.defined() || !t.is_leaf() || !t.requires_grad()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  const auto stream = node ? node->stream() : std::nullopt;
  return stream && stream->id() == 0;  // (0: the default stream)
}

bool capturing(const Tensor& t) {
  const c10::DeviceGuard guard(t.device());
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

// {y, stats or none}
std::pair<Tensor, Tensor> forward(const Pixels& in, const Tensor& weight, const Tensor& bias,
                                  int64_t groups, double eps, int64_t act) {
  const c10::DeviceGuard guard(in.x.device());
  const Sizes s(in.x, groups);
  const Tensor y = at::empty(in.x.sizes(), in.x.options().memory_format(at::MemoryFormat::Contiguous));
  const Tensor stats = bytes(s.ask(abi.stats_size), y);
  const uint64_t need = s.ask(abi.fwd_workspace_size);
  const Tensor ws = bytes(need, y);
  check(abi.fwd(s.samples, s.pixels, s.width, s.groups, s.dtype, (int32_t)act, address(in.x),
                in.sample, in.pitch, address(weight), address(bias), weight_dtype(s, weight, bias),
                (float)eps, target(y), (float*)target(stats), target(ws), need, stream_of(y)),
        "tgs_group_norm_fwd");
  return {y, stats};
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  // (what is not there is no edge of the node: optional, where an undefined tensor would be one)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w,
                        const std::optional<Tensor>& b, int64_t groups, double eps, int64_t act) {
    const Pixels in(x);
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    auto [y, stats] = ::forward(in, weight, bias, groups, eps, act);
    ctx->save_for_backward({in.x, weight, bias, stats});
    const bool captured = capturing(x);
    ctx->saved_data["call"] = std::vector<int64_t>{
        in.sample, in.pitch, groups, act, captured && gathered_by_default(x),
        captured && gathered_by_default(weight), captured && gathered_by_default(bias)};
    ctx->saved_data["eps"] = eps;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    const auto call = ctx->saved_data["call"].toIntVector();
    const c10::DeviceGuard guard(x.device());
    const Sizes s(x, call[2]);
    size_t edge = 0;  // (of the tensors that there are)
    size_t k = 4;
    const auto made = [&](const Tensor& t) {
      const bool live = call[k++];
      if (!t.defined() || !ctx->needs_input_grad(edge++)) return Tensor();
      // the default stream cannot wait for a captured one, and torch ends the process over it
      TORCH_CHECK(!live, "an eager graph of the same tensor lives: release it (and what it computed) "
                         "before this backward is captured");
      return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
    };
    Tensor dx = made(x), dw = made(weight), db = made(bias);
    const Pixels dy(grads[0].defined() ? grads[0] : at::zeros(x.sizes(), x.options()));
    const uint64_t need = s.ask(abi.bwd_workspace_size);
    const Tensor ws = bytes(need, x);
    check(abi.bwd(s.samples, s.pixels, s.width, s.groups, s.dtype, (int32_t)call[3], address(x),
                  call[0], call[1], address(dy.x), dy.sample, dy.pitch, address(weight),
                  address(bias), weight_dtype(s, weight, bias),
                  (float)ctx->saved_data["eps"].toDouble(), (const float*)address(stats),
                  target(dx), target(dw), target(db), target(ws), need, stream_of(x)),
          "tgs_group_norm_bwd");
    variable_list out{dx, dw, db};
    if (at::GradMode::is_enabled()) {  // a graph of the backward is recorded: it ends here
      for (Tensor& t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
      out = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice: group_norm has no second derivative",
                (int64_t)out.size())->apply(std::move(out));
    }
    out.resize(6);  // (the sizes and the activation have no gradients)
    return out;
  }
};

// An argument's tensor, undefined for None.
Tensor tensor_of(PyObject* o) {
  if (o == Py_None) return {};
  TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor is needed");
  return THPVariable_Unpack(o);
}

// group_norm(x, weight, bias, groups, eps, act, recorded) -> y
PyObject* group_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(count == 7, "group_norm takes seven arguments");
  const Tensor x = tensor_of(args[0]), weight = tensor_of(args[1]), bias = tensor_of(args[2]);
  const int64_t groups = PyLong_AsLongLong(args[3]), act = PyLong_AsLongLong(args[5]);
  const double eps = PyFloat_AsDouble(args[4]);
  const int recorded = PyObject_IsTrue(args[6]);
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(abi.fwd, "group_norm is not bound");
  const auto given = [](const Tensor& t) {
    return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
  };
  return THPVariable_Wrap(
      recorded ? GroupNorm::apply(x, given(weight), given(bias), groups, eps, act)
               : forward(Pixels(x), weight, bias, groups, eps, act).first);
  END_HANDLE_TH_ERRORS
}

// pixels(x) -> (tensor as it is read, distance of samples, distance of pixels)
PyObject* pixels(PyObject*, PyObject* arg) {
  HANDLE_TH_ERRORS
  const Pixels p(tensor_of(arg));
  return Py_BuildValue("(NLL)", THPVariable_Wrap(p.x), (long long)p.sample, (long long)p.pitch);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the C ABI's entry points, in abi's order)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 6) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
    return nullptr;
  }
  void* at[6];
  for (int i = 0; i < 6; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  abi.last_error = (decltype(abi.last_error))at[0];
  abi.stats_size = (decltype(abi.stats_size))at[1];
  abi.fwd_workspace_size = (decltype(abi.fwd_workspace_size))at[2];
  abi.fwd = (decltype(abi.fwd))at[3];
  abi.bwd_workspace_size = (decltype(abi.bwd_workspace_size))at[4];
  abi.bwd = (decltype(abi.bwd))at[5];
  Py_RETURN_NONE;
}

// gathered_by_default(t) -> bool
PyObject* gathered(PyObject*, PyObject* arg) {
  HANDLE_TH_ERRORS
  return PyBool_FromLong(gathered_by_default(tensor_of(arg)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, "takes the entry points' addresses"},
    {"group_norm", (PyCFunction)(void (*)(void))group_norm, METH_FASTCALL,
     "group_norm(x, weight, bias, groups, eps, act, recorded) -> y"},
    {"pixels", pixels, METH_O, "(tensor as it is read, distance of samples, of pixels)"},
    {"gathered_by_default", gathered, METH_O,
     "whether a leaf's gradients are gathered on the default stream by a graph that lives"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_group_norm_node", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__group_norm_node(void) { return PyModule_Create(&module); }
