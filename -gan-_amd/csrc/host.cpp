// gan_amd._host: the host side of the normalisation and clipping operators as a native module.
//
// What a call of these costs on the host is what it costs in small problems: a Python autograd
// function runs its backward under the GIL on the engine's thread (measured: 160 us for a forward
// and backward whose kernels take 15), and a list of tensors read from Python takes 0.4 us a tensor.
// Here the autograd nodes are C++ and a list is read in one pass.  The kernels stay behind the C ABI
// of include/ganamd.h; gan_amd._lib hands its entry points over (init), so one library is loaded.
//
// No exception leaves a function that Python calls: refused arguments and failed launches become
// GanAmdError, torch's own errors (out of memory) what torch makes of them.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>

#include <cmath>
#include <cstring>
#include <limits>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/ganamd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

PyObject* g_error = nullptr;        // gan_amd._lib.GanAmdError
PyObject* g_flat_name = nullptr;    // "_gan_flat": set on a parameter that lives in a flat buffer

struct Abi {
  decltype(&ganamd_group_norm_workspace) norm_workspace;
  decltype(&ganamd_group_norm_fwd) norm_fwd;
  decltype(&ganamd_group_norm_bwd) norm_bwd;
  decltype(&ganamd_group_norm_bwd_bwd) norm_bwd_bwd;
  decltype(&ganamd_grad_norm_workspace) grad_workspace;
  decltype(&ganamd_grad_norm) grad_norm;
  decltype(&ganamd_grad_clip) grad_clip;
  decltype(&ganamd_adamw_clip_workspace) adamw_workspace;
  decltype(&ganamd_adamw_clip) adamw;
} abi = {};

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

int code(at::ScalarType t) {
  return t == at::kFloat ? GANAMD_F32 : t == at::kBFloat16 ? GANAMD_BF16 : t == at::kHalf ? GANAMD_F16 : -1;
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void done(int rc, const char* what) {
  if (rc != GANAMD_OK) throw Refused(std::string(what) + " failed with code " + std::to_string(rc));
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}

// ---------------------------------------------------------------------------- group norm
std::string pack(const ganamd_norm_desc& d) { return std::string(reinterpret_cast<const char*>(&d), sizeof d); }
ganamd_norm_desc unpack(AutogradContext* ctx) {
  ganamd_norm_desc d;
  std::memcpy(&d, ctx->saved_data["d"].toStringRef().data(), sizeof d);
  return d;
}

Tensor workspace(const ganamd_norm_desc& d, int op, const Tensor& x) {
  size_t n = 0;
  done(abi.norm_workspace(&d, op, &n), "group_norm_workspace");
  return scratch(n, x);
}
size_t bytes(const Tensor& t) { return t.defined() ? (size_t)t.numel() : 0; }

Tensor norm_forward(const ganamd_norm_desc& d, const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& slope,
                    Tensor& stats) {
  Tensor y = at::empty_like(x);
  stats = at::empty({d.B, d.G, 2}, x.options().dtype(at::kDouble).requires_grad(false));
  if (x.numel() == 0) return y;
  const c10::DeviceGuard guard(x.device());
  const Tensor ws = workspace(d, 0, x);
  done(abi.norm_fwd(&d, ptr(x), ptr(w), ptr(b), ptr(slope), ptr(y), stats.data_ptr<double>(), ptr(ws), bytes(ws),
                    stream_of(x)),
       "group_norm_fwd");
  return y;
}

// Whether p has hooks that autograd runs on its gradient: they see only gradients that the engine is handed.
bool hooked(const Tensor& p) {
  return !torch::autograd::impl::hooks(p).empty() || torch::autograd::impl::post_acc_grad_hooks(p) != nullptr;
}

// Where the gradients of w, b and slope go: new tensors; or, where every wanted one is of a
// parameter in a flat buffer and this is a first-order backward, the buffer's views themselves
// (added to; the engine then gets none).  The engine orders streams along the gradients that it is
// handed, so that takes the parameters' accumulators on the running node's own stream: what adds to
// them there, and who waits for that stream after the backward, is then in order.  (They are on another
// one where a parameter is used on two streams, or where an older graph of it still lives.)
struct Targets {
  Tensor g[3];
  bool flat = false;
};

Targets targets(const Tensor* par, const bool* want, int64_t flat) {
  Targets t;
  const auto self = torch::autograd::get_current_node();
  bool any = false, all = self && !at::GradMode::is_enabled();
  for (int i = 0; i < 3; ++i) {
    if (!want[i]) continue;
    any = true;
    if (!(flat >> i & 1) || par[i].scalar_type() != at::kFloat) {
      all = false;
      continue;
    }
    const Tensor& g = par[i].grad();
    all = all && g.defined() && g.is_contiguous() && g.scalar_type() == at::kFloat && g.numel() == par[i].numel();
    // a gradient that autograd.grad was asked for is returned, not added
    const auto node = torch::autograd::impl::try_get_grad_accumulator(par[i]);
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    all = all && node && node->stream() == self->stream() && !hooked(par[i]);
    if (node && info) {
      const auto it = info->find(node.get());
      if (it != info->end() && it->second.captures_) all = false;
    }
    // one parameter in two places: its two sums are added by different blocks, so not into one buffer
    for (int j = 0; j < i; ++j)
      if (want[j] && par[j].const_data_ptr() == par[i].const_data_ptr()) all = false;
  }
  t.flat = any && all;
  for (int i = 0; i < 3; ++i)
    if (want[i]) t.g[i] = t.flat ? par[i].grad() : at::empty_like(par[i]);
  return t;
}

void norm_backward(const ganamd_norm_desc& d, const Tensor& gy, const Tensor& x, const Tensor* par, const Tensor& stats,
                   const Tensor& gx, const Targets& t) {
  if (x.numel() == 0) {
    for (const Tensor& g : t.g)
      if (g.defined() && !t.flat) g.zero_();
    return;
  }
  const c10::DeviceGuard guard(x.device());
  const Tensor ws = workspace(d, 1, x);
  done(abi.norm_bwd(&d, ptr(gy), ptr(x), ptr(par[0]), ptr(par[1]), ptr(par[2]), stats.data_ptr<double>(), ptr(gx),
                    ptr(t.g[0]), ptr(t.g[1]), ptr(t.g[2]), t.flat, ptr(ws), bytes(ws), stream_of(x)),
       "group_norm_bwd");
}

// Which of the edges first, first + 1, .. the engine asks for: one each for the defined tensors.
void asked(AutogradContext* ctx, int first, const Tensor* par, bool* want) {
  int e = first;
  for (int i = 0; i < 3; ++i) want[i] = par[i].defined() && ctx->needs_input_grad(e++);
}

// Whether a gradient that `node` hands on along edge e goes to a node of the default stream from
// another one.  The engine makes that stream wait for this one, which no capture allows: while a graph
// is captured, its error comes where nothing catches it and ends the process.
bool leaves_for_default_stream(torch::autograd::Node& node, size_t e) {
  const auto& edges = node.next_edges();
  if (e >= edges.size() || !edges[e].is_valid()) return false;
  const auto from = node.stream(), to = edges[e].function->stream();
  return from && to && *from != *to && to->id() == 0;
}

// Refuses a backward under capture whose gradients would leave the capture: what an eager graph of the
// same leaves, still alive, makes of it.
void stay_in_capture(AutogradContext* ctx, const Tensor& like) {
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const size_t n = node->next_edges().size();
  bool leaves = false;
  for (size_t e = 0; e < n; ++e)
    if (ctx->needs_input_grad(e)) leaves = leaves || leaves_for_default_stream(*node, e);
  if (!leaves) return;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream_of(like), &status) != hipSuccess) throw Refused("hipStreamIsCapturing failed");
  if (status != hipStreamCaptureStatusNone)
    throw Refused("group_norm_act: a backward in a graph capture reaches what was recorded eagerly on the default "
                  "stream (delete the eager results that share its inputs before the capture)");
}

// (gx, gradients of the wanted parameters) as a function of (gy, x, w, b, slope): what a backward
// with create_graph makes, differentiable once more.
struct NormBackward : torch::autograd::Function<NormBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gy, const Tensor& x, const OptTensor& w,
                               const OptTensor& b, const OptTensor& slope, const Tensor& stats,
                               const ganamd_norm_desc& d, int64_t flat, int64_t wanted) {
    ctx->set_materialize_grads(false);
    const Tensor par[3] = {w.value_or(Tensor()), b.value_or(Tensor()), slope.value_or(Tensor())};
    ctx->save_for_backward({gy, x, par[0], par[1], par[2], stats});
    ctx->saved_data["d"] = pack(d);
    ctx->saved_data["flat"] = flat;
    ctx->saved_data["wanted"] = wanted;
    variable_list out{at::empty_like(x)};
    Targets t;
    for (int i = 0; i < 3; ++i)
      if (wanted >> i & 1) out.push_back(t.g[i] = at::empty_like(par[i]));
    norm_backward(d, gy, x, par, stats, out[0], t);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(9);
    const ganamd_norm_desc d = unpack(ctx);
    const auto s = ctx->get_saved_variables();
    const Tensor &gy = s[0], &x = s[1], &stats = s[5];
    const Tensor par[3] = {s[2], s[3], s[4]};
    const int64_t wanted = ctx->saved_data["wanted"].toInt(), flat = ctx->saved_data["flat"].toInt();
    Tensor gg[3], ggx = grads[0];
    bool any = ggx.defined();
    for (int i = 0, k = 1; i < 3; ++i)
      if (wanted >> i & 1) {
        gg[i] = grads[k++];
        any = any || gg[i].defined();
        if (gg[i].defined()) gg[i] = gg[i].detach().to(par[i].scalar_type()).contiguous();
      }
    if (!any) return none;
    const bool differentiable = at::GradMode::is_enabled();
    variable_list out(9);
    {
      const at::NoGradGuard plain;
      ggx = ggx.defined() ? ggx.to(x.scalar_type()).contiguous() : at::zeros_like(x);
      bool want[3];
      asked(ctx, 2, par, want);
      const Targets t = targets(par, want, differentiable ? 0 : flat);
      stay_in_capture(ctx, x);
      const Tensor g_gy = at::empty_like(x), g_x = at::empty_like(x);
      if (x.numel()) {
        const c10::DeviceGuard guard(x.device());
        const Tensor ws = workspace(d, 2, x);
        done(abi.norm_bwd_bwd(&d, ptr(ggx), ptr(gg[0]), ptr(gg[1]), ptr(gg[2]), ptr(gy), ptr(x), ptr(par[0]),
                              ptr(par[1]), ptr(par[2]), stats.data_ptr<double>(), ptr(g_gy), ptr(g_x), ptr(t.g[0]),
                              ptr(t.g[1]), ptr(t.g[2]), t.flat, ptr(ws), bytes(ws), stream_of(x)),
             "group_norm_bwd_bwd");
      } else {
        for (const Tensor& g : t.g)
          if (g.defined() && !t.flat) g.zero_();
      }
      out[0] = g_gy;
      out[1] = g_x;
      for (int i = 0; i < 3 && !t.flat; ++i) out[2 + i] = t.g[i];
    }
    if (!differentiable) return out;
    // asked for a third derivative: the results carry a node that says there is none
    variable_list some;
    for (Tensor& t : out)
      if (t.defined()) some.push_back(t.detach().requires_grad_(true));
    torch::autograd::DelayedError no("group_norm_act is twice differentiable, not three times", (int64_t)some.size());
    some = no.apply(std::move(some));
    size_t k = 0;
    for (Tensor& t : out)
      if (t.defined()) t = some[k++];
    return out;
  }
};

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b,
                        const OptTensor& slope, const ganamd_norm_desc& d, int64_t flat) {
    const Tensor par[3] = {w.value_or(Tensor()), b.value_or(Tensor()), slope.value_or(Tensor())};
    Tensor stats;
    const Tensor y = norm_forward(d, x, par[0], par[1], par[2], stats);
    ctx->save_for_backward({x, par[0], par[1], par[2], stats});
    ctx->saved_data["d"] = pack(d);
    ctx->saved_data["flat"] = flat;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const ganamd_norm_desc d = unpack(ctx);
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &stats = s[4];
    const Tensor par[3] = {s[1], s[2], s[3]};
    const int64_t flat = ctx->saved_data["flat"].toInt();
    const Tensor gy = grads[0].to(x.scalar_type()).contiguous();
    bool want[3];
    asked(ctx, 1, par, want);
    variable_list out(6);
    if (at::GradMode::is_enabled()) {
      stay_in_capture(ctx, x);
      const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
      const int64_t wanted = want[0] | want[1] << 1 | want[2] << 2;
      const variable_list g =
          NormBackward::apply(gy, x, opt(par[0]), opt(par[1]), opt(par[2]), stats, d, flat, wanted);
      out[0] = g[0];
      for (int i = 0, k = 1; i < 3; ++i)
        if (want[i]) out[1 + i] = g[k++];
      return out;
    }
    const Targets t = targets(par, want, flat);
    stay_in_capture(ctx, x);
    if (ctx->needs_input_grad(0)) out[0] = at::empty_like(x);
    norm_backward(d, gy, x, par, stats, out[0], t);
    for (int i = 0; i < 3 && !t.flat; ++i) out[1 + i] = t.g[i];
    return out;
  }
};

// ---------------------------------------------------------------------------- arguments

// No operator here pushes tangents forward.  A dual tensor does not require a gradient, so it would
// be taken as its primal and its tangent lost without a word.
void no_tangent(const Tensor& t, const char* what) {
  if (t._fw_grad(/*level=*/0).defined()) throw Refused(std::string(what) + ": a forward-mode tangent (not supported)");
}
const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Refused(std::string(what) + " is a tensor; got " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  no_tangent(t, what);
  return t;
}
Tensor maybe(PyObject* o, const char* what) { return o == Py_None ? Tensor() : tensor(o, what); }
double number(PyObject* o, const char* what) {
  const double v = PyFloat_Check(o) || PyLong_Check(o) ? PyFloat_AsDouble(o) : std::numeric_limits<double>::quiet_NaN();
  if ((v == -1.0 && PyErr_Occurred()) || (!PyFloat_Check(o) && !PyLong_Check(o))) {
    PyErr_Clear();
    throw Refused(std::string(what) + " is a number");
  }
  return v;
}
std::string text(PyObject* o) {
  const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
  if (!s) PyErr_Clear();
  return s ? s : "";
}

// Runs f, a body that returns a new reference; what it throws becomes a Python error.
template <class F>
PyObject* guarded(const char* who, F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(g_error, (std::string(who) + ": " + r.what()).c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

void arity(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw Refused("takes " + std::to_string(want) + " arguments");
}

// Whether t, the Python object o, is a parameter in an optimizer's flat buffer.
bool in_flat(PyObject* o, const Tensor& t) {
  PyObject* v = nullptr;
  if (!t.defined() || !t.requires_grad() || !t.is_leaf() || !t.is_contiguous()) return false;
  if (_PyObject_LookupAttr(o, g_flat_name, &v) < 0) {
    PyErr_Clear();
    return false;
  }
  if (!v) return false;
  const bool yes = v != Py_None;
  Py_DECREF(v);
  return yes;
}

// group_norm_act(x, groups, weight, bias, act, slope, eps, layout)
PyObject* group_norm_act(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("group_norm_act", [&]() -> PyObject* {
    arity(n, 8);
    Tensor x = tensor(a[0], "x"), w = maybe(a[2], "weight"), b = maybe(a[3], "bias"), slope;
    ganamd_norm_desc d = {};
    const std::string act = text(a[4]), layout = text(a[7]);
    d.act = act == "none" ? GANAMD_NORM_NONE : act == "silu" ? GANAMD_NORM_SILU : act == "leaky" ? GANAMD_NORM_LEAKY
          : act == "prelu" ? GANAMD_NORM_PRELU : -1;
    d.layout = layout == "nhwc" ? GANAMD_NORM_ROWS : layout == "cnhw" ? GANAMD_NORM_PLANES : -1;
    if (d.act < 0) throw Refused("act is none of 'none', 'silu', 'leaky', 'prelu'");
    if (d.layout < 0) throw Refused("layout is neither 'nhwc' nor 'cnhw'");
    if (d.act == GANAMD_NORM_PRELU) {
      slope = tensor(a[5], "act='prelu': slope");
    } else if (d.act == GANAMD_NORM_LEAKY) {
      d.slope = (float)number(a[5], "act='leaky': slope");
    } else if (a[5] != Py_None) {
      throw Refused("act '" + act + "' takes no slope");
    }
    d.eps = (float)number(a[6], "eps");
    if (!(d.eps > 0.f)) throw Refused("eps is more than 0");
    if (!PyLong_Check(a[1]) || PyBool_Check(a[1])) throw Refused("groups is a whole number");
    const long groups = PyLong_AsLong(a[1]);
    if (groups == -1 && PyErr_Occurred()) PyErr_Clear();
    if (!x.is_cuda()) throw Refused("x is on " + x.device().str());
    d.dtype = code(x.scalar_type());
    if (d.dtype < 0) throw Refused(std::string("x is ") + toString(x.scalar_type()) + ": float32, bfloat16 or float16");
    if (x.dim() < 2) throw Refused("x has a batch and a channel dimension at least");
    const int64_t B = d.layout == GANAMD_NORM_ROWS ? x.size(0) : x.size(1);
    const int64_t C = d.layout == GANAMD_NORM_ROWS ? x.size(-1) : x.size(0);
    if (groups < 1 || C < 1 || C % groups != 0)
      throw Refused(std::to_string(groups) + " groups do not divide " + std::to_string(C) + " channels");
    const int64_t L = x.numel() ? x.numel() / (B * C) : 1;
    if (B > INT32_MAX || C > (1 << 24) || L > (1 << 30)) throw Refused("x is too large");
    d.B = (int32_t)B;
    d.C = (int32_t)C;
    d.G = (int32_t)groups;
    d.L = L;
    d.param_dtype = GANAMD_F32;
    bool first = true;
    for (const Tensor* t : {&w, &b, &slope}) {
      if (!t->defined()) continue;
      const int c = code(t->scalar_type());
      if (t->numel() != C || t->device() != x.device())
        throw Refused("parameters are " + std::to_string(C) + " elements each, on x's device");
      if (c < 0 || (c != GANAMD_F32 && c != d.dtype) || (!first && c != d.param_dtype))
        throw Refused("parameters are all float32 or all of x's type");
      d.param_dtype = c;
      first = false;
    }
    const int64_t flat = (in_flat(a[2], w) ? 1 : 0) | (in_flat(a[3], b) ? 2 : 0) |
                         (d.act == GANAMD_NORM_PRELU && in_flat(a[5], slope) ? 4 : 0);
    // contiguous before the node: a copy made inside it would be saved without its history
    x = x.contiguous();
    for (Tensor* t : {&w, &b, &slope})
      if (t->defined()) *t = t->contiguous();
    bool grad = x.requires_grad();
    for (const Tensor* t : {&w, &b, &slope}) grad = grad || (t->defined() && t->requires_grad());
    grad = grad && at::GradMode::is_enabled();
    if (x.numel()) {                   // refuses what the kernels cannot take, before anything runs
      size_t need = 0;
      for (int op = 0; op < (grad ? 3 : 1); ++op)
        if (abi.norm_workspace(&d, op, &need) != GANAMD_OK) throw Refused("x is too large");
    }
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    if (grad) return THPVariable_Wrap(Norm::apply(x, opt(w), opt(b), opt(slope), d, flat));
    const at::NoGradGuard plain;
    Tensor stats;
    return THPVariable_Wrap(norm_forward(d, x, w, b, slope, stats));
  });
}

// ---------------------------------------------------------------------------- lists of gradients
// One tensor of the list `name`; throws what is wrong with it.
const Tensor& member(PyObject* o, const char* name, int& device) {
  const std::string what(name);
  if (!THPVariable_Check(o)) throw Refused(what + " are tensors; got " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  no_tangent(t, name);
  if (t.layout() != at::kStrided) throw Refused(what + " are dense tensors");
  if (!t.is_cuda()) throw Refused(what + " are on one GPU; got one on " + t.device().str());
  if (device < 0) device = t.get_device();
  if (t.get_device() != device) throw Refused(what + " are on one GPU; got several");
  if (code(t.scalar_type()) < 0)
    throw Refused(what + " are float32, bfloat16 or float16; got " + toString(t.scalar_type()));
  if (!t.is_non_overlapping_and_dense()) throw Refused(what + " are stored densely, each element once");
  return t;
}

// The table of the list `ts` and its outputs `outs` (a null pointer: none of their own).
std::vector<ganamd_tensor> table(PyObject* ts, PyObject* outs, bool writes, Tensor& like) {
  if (!PyList_Check(ts) || (outs && !PyList_Check(outs))) throw Refused("lists of tensors are wanted");
  const Py_ssize_t n = PyList_GET_SIZE(ts);
  if (outs && PyList_GET_SIZE(outs) != n)
    throw Refused(std::to_string(n) + " gradients, " + std::to_string(PyList_GET_SIZE(outs)) + " outputs");
  if (n > INT32_MAX) throw Refused("too many tensors");
  std::vector<ganamd_tensor> rows((size_t)n);
  int device = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const Tensor& t = member(PyList_GET_ITEM(ts, i), "gradients", device);
    const Tensor* o = &t;
    if (outs) {
      o = &member(PyList_GET_ITEM(outs, i), "outputs", device);
      if (o->numel() != t.numel()) throw Refused("an output has another number of elements than its gradient");
      if (!(t.is_contiguous() && o->is_contiguous()) && t.strides() != o->strides())
        throw Refused("a gradient that is not contiguous needs an output of its own strides");
      if (o->scalar_type() != t.scalar_type() && o->scalar_type() != at::kFloat)
        throw Refused("an output is of its gradient's type or float32");
    }
    if (writes && o->requires_grad()) throw Refused("writes into a tensor that requires a gradient (detach it)");
    ganamd_tensor& r = rows[(size_t)i];
    r.p = t.const_data_ptr();
    r.out = const_cast<void*>(o->const_data_ptr());
    r.n = t.numel();
    r.dtype = code(t.scalar_type());
    r.out_dtype = code(o->scalar_type());
    if (i == 0) like = t;
  }
  return rows;
}

// Counts a write into t: autograd notices it in a tensor it saved, the packed copies of a weight that they are stale.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// grad_norm(tensors, kind) of a list that is not empty
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("grad_norm", [&]() -> PyObject* {
    arity(n, 2);
    const at::NoGradGuard plain;
    Tensor like;
    const auto rows = table(a[0], nullptr, false, like);
    if (rows.empty()) throw Refused("no tensors");
    const c10::DeviceGuard guard(like.device());
    const Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
    const size_t need = abi.grad_workspace(rows.data(), (int)rows.size());
    const Tensor ws = scratch(need, like);
    done(abi.grad_norm(rows.data(), (int)rows.size(), (int)PyLong_AsLong(a[1]), norm.data_ptr<float>(), ptr(ws), need,
                       stream_of(like)),
         "grad_norm");
    return THPVariable_Wrap(norm);
  });
}

// clip(tensors, outs or None, max_norm, kind) of a list that is not empty
PyObject* clip(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("clip_grad_norm_", [&]() -> PyObject* {
    arity(n, 4);
    const at::NoGradGuard plain;
    Tensor like;
    const auto rows = table(a[0], a[1] == Py_None ? nullptr : a[1], true, like);
    if (rows.empty()) throw Refused("no tensors");
    const float most = (float)number(a[2], "max_norm");
    const c10::DeviceGuard guard(like.device());
    const Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
    const size_t need = abi.grad_workspace(rows.data(), (int)rows.size());
    const Tensor ws = scratch(need, like);
    const int rc = abi.grad_clip(rows.data(), (int)rows.size(), (int)PyLong_AsLong(a[3]), most, norm.data_ptr<float>(),
                                 ptr(ws), need, stream_of(like));
    if (rc == GANAMD_EINVAL) throw Refused("tensors that are written to share memory with others of the call");
    done(rc, "grad_clip");
    PyObject* outs = a[1] == Py_None ? a[0] : a[1];
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(outs); ++i) written(THPVariable_Unpack(PyList_GET_ITEM(outs, i)));
    return THPVariable_Wrap(norm);
  });
}

// clipped_adamw(param, grad, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps, weight_decay, max_norm, norm or None)
PyObject* clipped_adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("clipped_adamw_", [&]() -> PyObject* {
    arity(n, 12);
    const at::NoGradGuard plain;
    const char* names[4] = {"param", "grad", "exp_avg", "exp_avg_sq"};
    Tensor t[4];
    for (int i = 0; i < 4; ++i) t[i] = tensor(a[i], names[i]);
    for (int i = 0; i < 4; ++i) {
      if (!t[i].is_cuda() || t[i].scalar_type() != at::kFloat || !t[i].is_contiguous())
        throw Refused(std::string(names[i]) + " is a contiguous float32 tensor on the GPU");
      if (t[i].numel() != t[0].numel()) throw Refused(std::string(names[i]) + " has another number of elements than param");
    }
    const Tensor& step = tensor(a[4], "step");
    if (!step.is_cuda() || step.scalar_type() != at::kInt || step.numel() != 1)
      throw Refused("step is one int32 on the GPU");
    double k[5];
    const char* nums[5] = {"lr", "beta1", "beta2", "eps", "weight_decay"};
    for (int i = 0; i < 5; ++i) k[i] = number(a[5 + i], nums[i]);
    const float most = (float)number(a[10], "max_norm");
    if (!(most >= 0.f)) throw Refused("max_norm is 0 or more");
    const int64_t count = t[0].numel();
    for (int i = 0; i < 4; ++i) {
      if (t[i].device() != step.device()) throw Refused("the buffers and the counter are on one device");
      for (int j = 0; j < i && count; ++j) {
        const auto p = reinterpret_cast<uintptr_t>(t[i].data_ptr()), q = reinterpret_cast<uintptr_t>(t[j].data_ptr());
        if (p < q + 4 * count && q < p + 4 * count) throw Refused("four separate buffers are wanted");
      }
    }
    Tensor norm = maybe(a[11], "norm");
    if (norm.defined() && (norm.device() != step.device() || norm.scalar_type() != at::kFloat || norm.numel() != 1))
      throw Refused("norm is one float32 on the buffers' device");
    const void* small[2] = {step.const_data_ptr(), norm.defined() ? norm.const_data_ptr() : nullptr};
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 4 && count; ++j) {
        const auto p = reinterpret_cast<uintptr_t>(small[i]), q = reinterpret_cast<uintptr_t>(t[j].data_ptr());
        if (p < q + 4 * count && q < p + 4) throw Refused("step and norm lie outside the buffers");
      }
    if (small[0] == small[1]) throw Refused("step and norm are two tensors");
    const c10::DeviceGuard guard(step.device());
    if (!norm.defined()) norm = at::empty({}, step.options().dtype(at::kFloat));
    if (count) {
      const size_t need = abi.adamw_workspace();
      const Tensor ws = scratch(need, step);
      done(abi.adamw(t[0].data_ptr<float>(), t[1].data_ptr<float>(), t[2].data_ptr<float>(), t[3].data_ptr<float>(),
                     count, step.data_ptr<int32_t>(), k[0], k[1], k[2], k[3], k[4], most, norm.data_ptr<float>(),
                     ptr(ws), need, stream_of(step)),
           "adamw_clip");
    } else {
      norm.zero_();
      step.add_(1);
    }
    for (const Tensor& w : {t[0], t[2], t[3], step, norm}) written(w);
    return THPVariable_Wrap(norm);
  });
}

// Whether the node that made the tensor hands a gradient to the default stream from another one.
PyObject* crosses(PyObject*, PyObject* o) {
  return guarded("crosses", [&]() -> PyObject* {
    const auto node = tensor(o, "y").grad_fn();
    bool yes = false;
    for (size_t e = 0; node && e < node->next_edges().size(); ++e) yes = yes || leaves_for_default_stream(*node, e);
    return PyBool_FromLong(yes);
  });
}

// Whether stream s is recording into a graph.  (The default stream cannot, and may not be asked while another does.)
bool capturing(const c10::Stream& s) {
  if (s.id() == 0) return false;
  const auto type = c10::hip::getCurrentHIPStream(s.device_index()).unwrap().device_type();
  const auto h = c10::hip::HIPStream::unpack3(s.id(), s.device_index(), type);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(h.stream(), &status) != hipSuccess) throw Refused("hipStreamIsCapturing failed");
  return status != hipStreamCaptureStatusNone;
}

// apart(p): whether p's gradient has to be handed to the engine (gan_amd.ops.flat_grad): p has hooks, or the
// backward node that is running and the accumulator of p's gradient are on different streams that the engine
// could order.
// A node in a capture whose parameter's accumulator is outside it cannot be ordered with that at all: False.
PyObject* apart(PyObject*, PyObject* o) {
  return guarded("apart", [&]() -> PyObject* {
    const auto node = torch::autograd::get_current_node();
    const Tensor& p = tensor(o, "p");
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(p);
    if (!node || !acc) Py_RETURN_FALSE;
    if (hooked(p)) Py_RETURN_TRUE;
    const auto from = node->stream(), to = acc->stream();
    if (!from || !to || *from == *to || (capturing(*from) && !capturing(*to))) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
  });
}

// init(GanAmdError, {entry point: address})
PyObject* init(PyObject*, PyObject* args) {
  PyObject *error = nullptr, *where = nullptr;
  if (!PyArg_ParseTuple(args, "OO!", &error, &PyDict_Type, &where)) return nullptr;
  const struct {
    const char* name;
    void** to;
  } rows[] = {{"ganamd_group_norm_workspace", reinterpret_cast<void**>(&abi.norm_workspace)},
              {"ganamd_group_norm_fwd", reinterpret_cast<void**>(&abi.norm_fwd)},
              {"ganamd_group_norm_bwd", reinterpret_cast<void**>(&abi.norm_bwd)},
              {"ganamd_group_norm_bwd_bwd", reinterpret_cast<void**>(&abi.norm_bwd_bwd)},
              {"ganamd_grad_norm_workspace", reinterpret_cast<void**>(&abi.grad_workspace)},
              {"ganamd_grad_norm", reinterpret_cast<void**>(&abi.grad_norm)},
              {"ganamd_grad_clip", reinterpret_cast<void**>(&abi.grad_clip)},
              {"ganamd_adamw_clip_workspace", reinterpret_cast<void**>(&abi.adamw_workspace)},
              {"ganamd_adamw_clip", reinterpret_cast<void**>(&abi.adamw)}};
  for (const auto& r : rows) {
    PyObject* v = PyDict_GetItemString(where, r.name);
    *r.to = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!*r.to) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", r.name);
      return nullptr;
    }
  }
  Py_INCREF(error);
  g_error = error;
  if (!g_flat_name) g_flat_name = PyUnicode_InternFromString("_gan_flat");
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"group_norm_act", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(group_norm_act)), METH_FASTCALL, nullptr},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grad_norm)), METH_FASTCALL, nullptr},
    {"clip", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(clip)), METH_FASTCALL, nullptr},
    {"clipped_adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(clipped_adamw)), METH_FASTCALL, nullptr},
    {"crosses", crosses, METH_O, nullptr},
    {"apart", apart, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// SRC_HASH: hash of the sources this module was compiled with (set by __graft_entry__.build()); the loader
// compares it with libganamd.so's, whose structs this module fills in.
#ifndef GANAMD_SRC_HASH
#define GANAMD_SRC_HASH "unknown"
#endif
PyMODINIT_FUNC PyInit__host() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "SRC_HASH", GANAMD_SRC_HASH) < 0) Py_CLEAR(m);
  return m;
}
