// The Python module hdcmamba_b200._host: checks, allocation, launch and autograd nodes, in C++, of the operators whose
// kernels take less time than the same path would in Python (one token's decayed attention: a 2.6 us kernel; the
// addresses, types and sizes of some hundred gradients; the autograd engine's calls of a Python function, 50 us for
// an empty one).  It calls the library's C entry points on the current stream of the tensors' device, as
// hdcmamba_b200/ops.py does through ctypes, and raises what that raises: ValueError, TypeError, RuntimeError for CPU
// tensors, HdcError for a status of the library.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <memory>
#include <optional>
#include <vector>

#include "../../include/hdcmamba_b200.h"

// what this module was compiled against (hdcmamba_b200/build.py reads it from the file)
extern "C" __attribute__((used, visibility("default"))) const char hdc_host_tag[] = HDC_HOST_TAG;

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

PyObject* g_error = nullptr;  // _lib.HdcError

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void done(const char* name, int rc) {
  if (rc != 0) throw Failure(std::string(name) + " failed (" + std::to_string(rc) + "): " + hdc_error_string());
}

// ---------------------------------------------------------------- checks
int code_of(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return HDC_BF16;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "hdcmamba_b200: unsupported dtype ", t.scalar_type(),
                   " (float32 or bfloat16)");
  return HDC_F32;
}
void same_type(const Tensor& ref, const Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == ref.scalar_type(), "hdcmamba_b200: dtype mismatch (", t.scalar_type(), " vs ",
                   ref.scalar_type(), ")");
}
void on_device(const Tensor& ref, std::initializer_list<const Tensor*> rest) {
  TORCH_CHECK(ref.is_cuda(), "hdcmamba_b200 kernels run on CUDA tensors only (got a CPU tensor)");
  for (const Tensor* t : rest)
    if (t && t->defined()) {
      TORCH_CHECK(t->is_cuda(), "hdcmamba_b200 kernels run on CUDA tensors only (got a CPU tensor)");
      TORCH_CHECK_VALUE(t->device() == ref.device(), "tensors are on ", ref.device(), " and ", t->device());
    }
}
// An output lies apart from what the call reads, as far as the two tell (views with gaps: unless they begin alike).
void apart(const Tensor& out, std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs) {
    if (!t || !t->defined() || !out.is_alias_of(*t) || out.numel() == 0 || t->numel() == 0) continue;
    const auto s = at::get_overlap_status(out, *t);
    if (out.data_ptr() == t->data_ptr() || s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial)
      throw Failure(std::string("hdcmamba_b200: ") + what + " overlaps an input");
  }
}
const Tensor* at_of(const Maybe& t) { return t ? &*t : nullptr; }
template <typename T = void> T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T = void> T* ptr(const Maybe& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

// The tensors' device is current, and its stream at hand.
struct On {
  c10::cuda::CUDAGuard guard;
  hdc_stream_t stream;
  explicit On(const Tensor& t)
      : guard(t.device()),
        stream(reinterpret_cast<hdc_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream())) {}
};

// A tensor of the caller's that the call has written: autograd must not take what it saved of it before for what it was.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor make(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
  return at::empty(shape, like.options().dtype(type).requires_grad(false));
}
// Scratch memory of the current stream, given back at the end of the call (to kernels that come later there).
c10::DataPtr workspace(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// ---------------------------------------------------------------- linear attention with a decay for each head
void is_heads(const Tensor& t, const Tensor& q, const char* what) {
  TORCH_CHECK_VALUE(t.sizes() == q.sizes(), what, " must be ", q.sizes(), ", got ", t.sizes());
  TORCH_CHECK_VALUE(q.size(-1) <= 1 || t.stride(-1) == 1, what, " needs a unit stride within a head");
}
void is_state(const Maybe& s, const Tensor& q, const char* what) {
  if (!s) return;
  const int64_t B = q.size(0), H = q.size(-2), D = q.size(-1);
  TORCH_CHECK_VALUE(s->scalar_type() == at::kFloat && s->sizes() == at::IntArrayRef({B, H, D, D}) && s->is_contiguous(),
                    what, " must be a contiguous fp32 [", B, ", ", H, ", ", D, ", ", D, "] tensor");
}
struct Attn {
  Tensor q, k, v, g;
  int code;
  int64_t B, L, H, D;
  Attn(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, int64_t dims)
      : q(q_), k(k_), v(v_), code(code_of(q_)) {
    same_type(q, k);
    same_type(q, v);
    TORCH_CHECK_VALUE(q.dim() == dims, dims == 4 ? "q must be [B, L, H, D]" : "q must be [B, H, D]");
    B = q.size(0); L = dims == 4 ? q.size(1) : 1; H = q.size(-2); D = q.size(-1);
    TORCH_CHECK_VALUE(D >= 1 && D <= 128 && H >= 1, "heads of 1 to 128 elements are supported, got H=", H, ", D=", D);
    is_heads(q, q, "q");
    is_heads(k, q, "k");
    is_heads(v, q, "v");
    TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == H, "log_decay must be [", H, "], got ", log_decay.sizes());
    g = log_decay;
  }
  // after the device check
  void decays() {
    if (g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
    if (!g.is_contiguous()) g = g.contiguous();
  }
};
#define VIEW(t) ptr(t), (t).stride(0), (t).stride(1), (t).stride(2)

struct Out {
  Tensor o, state, states;
};
Out attn_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, double scale,
                 const Maybe& state, const Maybe& out, bool want_states) {
  Attn a(q, k, v, log_decay, 4);
  is_state(state, q, "state");
  if (out) {
    same_type(q, *out);
    is_heads(*out, q, "out");
    apart(*out, {&q, &k, &v, &log_decay, at_of(state)}, "out");
  }
  on_device(q, {&k, &v, &log_decay, at_of(state), at_of(out)});
  On on(q);
  a.decays();
  Out r;
  r.o = out ? *out : make({a.B, a.L, a.H, a.D}, q, q.scalar_type());
  r.state = make({a.B, a.H, a.D, a.D}, q, at::kFloat);
  const int64_t n = hdc_decay_attn_state_slots(a.code, a.B, a.L, a.H, a.D);
  if (want_states || n > 1) r.states = make({a.B, a.H, n, a.D, a.D}, q, at::kFloat);
  done("hdc_decay_attn_fwd",
       hdc_decay_attn_fwd(a.code, VIEW(q), VIEW(k), VIEW(v), ptr<float>(a.g), ptr<float>(state), (float)scale, VIEW(r.o),
                          ptr<float>(r.state), r.states.defined() ? ptr<float>(r.states) : nullptr, a.B, a.L, a.H, a.D,
                          on.stream));
  if (out) written(r.o);
  return r;
}

struct Grads {
  Tensor dq, dk, dv, dstate;
};
Grads attn_backward(Tensor dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                    const Tensor& states, double scale, const Maybe& dstate, bool need_dstate) {
  Attn a(q, k, v, log_decay, 4);
  same_type(q, dout);
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes(), "do must be ", q.sizes(), ", got ", dout.sizes());
  is_state(dstate, q, "dstate");
  const int64_t n = hdc_decay_attn_state_slots(a.code, a.B, a.L, a.H, a.D);
  TORCH_CHECK_VALUE(states.scalar_type() == at::kFloat && states.is_contiguous() &&
                        states.sizes() == at::IntArrayRef({a.B, a.H, n, a.D, a.D}),
                    "states must be a contiguous fp32 [", a.B, ", ", a.H, ", ", n, ", ", a.D, ", ", a.D, "] tensor");
  on_device(q, {&k, &v, &log_decay, &dout, &states, at_of(dstate)});
  On on(q);
  a.decays();
  if (a.D > 1 && dout.stride(3) != 1) dout = dout.contiguous();
  Grads r;
  for (Tensor* t : {&r.dq, &r.dk, &r.dv}) *t = make({a.B, a.L, a.H, a.D}, q, q.scalar_type());
  if (need_dstate) r.dstate = make({a.B, a.H, a.D, a.D}, q, at::kFloat);
  const size_t bytes = hdc_decay_attn_bwd_workspace_bytes(a.code, a.B, a.L, a.H, a.D);
  const auto ws = workspace(bytes);
  done("hdc_decay_attn_bwd",
       hdc_decay_attn_bwd(a.code, VIEW(q), VIEW(k), VIEW(v), VIEW(dout), ptr<float>(a.g), ptr<float>(states),
                          ptr<float>(dstate), (float)scale, VIEW(r.dq), VIEW(r.dk), VIEW(r.dv),
                          need_dstate ? ptr<float>(r.dstate) : nullptr, ws.get(), bytes, a.B, a.L, a.H, a.D, on.stream));
  return r;
}

void first_order_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "hdcmamba_b200: norm_conv1d, gated_scan, group_norm_act and decay_attention are differentiable once "
              "(create_graph=False)");
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// (q, k, v, log_decay, state, scale) -> (o, state after); gradients for q, k, v and state
struct DecayAttention : torch::autograd::Function<DecayAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& log_decay, const Maybe& state, double scale) {
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["state_type"] = state ? (int64_t)state->scalar_type() : (int64_t)-1;
    const Maybe s = state ? Maybe(state->to(at::kFloat).contiguous()) : std::nullopt;
    Out r = attn_forward(q, k, v, log_decay, scale, s, std::nullopt, true);
    ctx->save_for_backward({q, k, v, log_decay, r.states});
    return {r.o, r.state};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    first_order_only();
    const variable_list s = ctx->get_saved_variables();
    const Tensor dout = d[0].defined() ? d[0] : at::zeros(s[0].sizes(), s[0].options().requires_grad(false));
    const Maybe ds = d[1].defined() ? Maybe(d[1].contiguous()) : std::nullopt;
    const int64_t type = ctx->saved_data["state_type"].toInt();
    const bool need = type >= 0 && ctx->needs_input_grad(4);
    Grads r = attn_backward(dout, s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(), ds, need);
    if (need) r.dstate = r.dstate.to((at::ScalarType)type);
    return {r.dq, r.dk, r.dv, Variable(), need ? r.dstate : Variable(), Variable()};
  }
};

// ---------------------------------------------------------------- token embedding
int id_bytes(const Tensor& ids) {
  if (ids.scalar_type() == at::kLong) return 8;
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt, "hdcmamba_b200: ids must be int64 or int32, got ", ids.scalar_type());
  return 4;
}
void is_table(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) >= 1 && t.size(1) >= 1, what, " must be [rows, D], got ", t.sizes());
  TORCH_CHECK_VALUE(t.size(1) == 1 || t.stride(1) == 1, what, " needs a unit column stride");
}

// A tensor with memory of its own and no tangent: not a transform's or a subclass's stand-in for one.
bool ordinary(const Tensor& t) {
  return t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t._fw_grad(0).defined();
}
// whether `lookup` takes these: what nn.Embedding allows beyond is left to it
bool takes(const Tensor& ids, const Tensor& w) {
  return ordinary(ids) && ordinary(w) && (w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16) && w.is_cuda() &&
         w.dim() == 2 && w.stride(1) == 1 &&
         w.size(0) >= 1 && w.size(0) <= (int64_t(1) << 30) && w.size(1) >= 1 && w.size(1) <= 65536 &&
         (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt) && ids.device() == w.device() &&
         ids.numel() <= (int64_t(1) << 30);
}

Tensor lookup(const Tensor& ids, const Tensor& weight, double scale, const Maybe& out) {
  const int code = code_of(weight), bytes = id_bytes(ids);
  is_table(weight, "weight");
  const int64_t rows = weight.size(0), D = weight.size(1);
  at::DimVector shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(D);
  if (out) {
    same_type(weight, *out);
    TORCH_CHECK_VALUE(out->sizes() == at::IntArrayRef(shape) && out->is_contiguous(), "out must be a contiguous ",
                      at::IntArrayRef(shape), " tensor");
    apart(*out, {&ids, &weight}, "out");
  }
  on_device(weight, {&ids, at_of(out)});
  On on(weight);
  const Tensor i = ids.contiguous();
  Tensor y = out ? *out : make(shape, weight, weight.scalar_type());
  done("hdc_embedding_fwd", hdc_embedding_fwd(code, ptr(i), bytes, ptr(weight), weight.stride(0), ptr(y), D, (float)scale,
                                              i.numel(), rows, D, on.stream));
  if (out) written(y);
  return y;
}

Tensor lookup_backward(const Tensor& dy, const Tensor& ids, int64_t rows, double scale, int64_t skip, const Maybe& out) {
  const int code = code_of(dy), bytes = id_bytes(ids);
  TORCH_CHECK_VALUE(dy.dim() >= 1 && dy.sizes().slice(0, dy.dim() - 1) == ids.sizes() && dy.size(-1) >= 1, "dy ", dy.sizes(),
                    " must be ids' shape ", ids.sizes(), " and columns");
  const int64_t D = dy.size(-1);
  TORCH_CHECK_VALUE(rows >= 1, "rows must be positive, got ", rows);
  if (out) {
    same_type(dy, *out);
    TORCH_CHECK_VALUE(out->sizes() == at::IntArrayRef({rows, D}), "out must be [", rows, ", ", D, "]");
    is_table(*out, "out");
    apart(*out, {&dy, &ids}, "out");
  }
  on_device(dy, {&ids, at_of(out)});
  On on(dy);
  Tensor d = out ? *out : make({rows, D}, dy, dy.scalar_type());
  const Tensor i = ids.contiguous();
  Tensor g = dy.dim() == 2 ? dy : dy.reshape({-1, D});
  if (D > 1 && g.stride(1) != 1) g = g.contiguous();
  const size_t n = hdc_embedding_bwd_workspace_bytes(i.numel(), rows, D);
  const auto ws = workspace(n);
  done("hdc_embedding_bwd", hdc_embedding_bwd(code, ptr(i), bytes, ptr(g), g.stride(0), ptr(d), d.stride(0), (float)scale,
                                              skip, ws.get(), n, i.numel(), rows, D, on.stream));
  if (out) written(d);
  return d;
}

// The lookup is linear in its table and its gradient linear in dy, so that each is the other's derivative.
Variable embedding_grad(const Variable& dy, const Tensor& ids, int64_t rows, double scale, int64_t skip);

// (weight, ids, scale, padding id or -1) -> rows; gradient for weight
struct Embedding : torch::autograd::Function<Embedding> {
  static Variable forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t skip) {
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["skip"] = skip;
    ctx->save_for_backward({ids});
    return lookup(ids, weight, scale, std::nullopt);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    auto& s = ctx->saved_data;
    return {embedding_grad(d[0], ctx->get_saved_variables()[0], s["rows"].toInt(), s["scale"].toDouble(), s["skip"].toInt()),
            Variable(), Variable(), Variable()};
  }
};

// (dy, ids, rows, scale, padding id or -1) -> the table's gradient; gradient for dy: that of the padding's tokens is zero
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Variable forward(AutogradContext* ctx, const Tensor& dy, const Tensor& ids, int64_t rows, double scale, int64_t skip) {
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["skip"] = skip;
    ctx->save_for_backward({ids});
    return lookup_backward(dy, ids, rows, scale, skip, std::nullopt);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t skip = ctx->saved_data["skip"].toInt();
    Variable ddy;
    if (!d[0].has_storage()) {  // a transform's stand-in for several
      auto shape = ids.sizes().vec();
      shape.push_back(d[0].size(1));
      ddy = d[0].index_select(0, ids.reshape({-1})).reshape(shape);
      if (scale != 1.0) ddy = ddy * scale;
    } else {
      const Tensor table = d[0].size(1) == 1 || d[0].stride(1) == 1 ? d[0] : d[0].contiguous();
      ddy = at::GradMode::is_enabled() && table.requires_grad() ? Embedding::apply(table, ids, scale, skip)
                                                                : lookup(ids, table, scale, std::nullopt);
    }
    if (skip >= 0) ddy = ddy.masked_fill(ids.eq(skip).unsqueeze(-1), 0);
    return {ddy, Variable(), Variable(), Variable(), Variable()};
  }
};

Variable embedding_grad(const Variable& dy, const Tensor& ids, int64_t rows, double scale, int64_t skip) {
  if (!dy.has_storage()) {  // a transform's stand-in for several (is_grads_batched): operations that it can take apart
    const int64_t D = dy.size(-1);
    Tensor terms = dy.to(at::kFloat) * scale;
    if (skip >= 0) terms = terms.masked_fill(ids.eq(skip).unsqueeze(-1), 0);
    const Tensor zeros = at::zeros({rows, D}, ids.options().dtype(at::kFloat));
    return zeros.index_add(0, ids.reshape({-1}), terms.reshape({-1, D})).to(dy.scalar_type());
  }
  if (at::GradMode::is_enabled() && dy.requires_grad()) return EmbeddingGrad::apply(dy, ids, rows, scale, skip);
  return lookup_backward(dy, ids, rows, scale, skip, std::nullopt);
}

// ---------------------------------------------------------------- Python
const Tensor& tensor(PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), "hdcmamba_b200: a tensor is wanted, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
Maybe maybe(PyObject* o) { return o == Py_None ? std::nullopt : Maybe(tensor(o)); }
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... A> PyObject* tuple(const A&... a) {
  PyObject* t = PyTuple_New(sizeof...(A));
  if (!t) throw python_error();
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(t, i++, wrap(a)), ...);
  return t;
}

template <Py_ssize_t N, PyObject* (*F)(PyObject* const*)>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == N, "hdcmamba_b200._host: ", N, " arguments are wanted, got ", n);
  try {
    return F(a);
  } catch (const Failure& e) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_attn(PyObject* const* a) {
  const bool states = truth(a[7]);
  const Out r = attn_forward(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), number(a[4]), maybe(a[5]), maybe(a[6]), states);
  return states ? tuple(r.o, r.state, r.states) : tuple(r.o, r.state);
}
PyObject* py_attn_bwd(PyObject* const* a) {
  const Grads r = attn_backward(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5]),
                                number(a[6]), maybe(a[7]), truth(a[8]));
  return tuple(r.dq, r.dk, r.dv, r.dstate);
}
PyObject* py_attn_train(PyObject* const* a) {
  const variable_list r = DecayAttention::apply(tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), maybe(a[4]), number(a[5]));
  return tuple(r[0], r[1]);
}
PyObject* py_attn_step(PyObject* const* p) {
  const Tensor &q = tensor(p[0]), &k = tensor(p[1]), &v = tensor(p[2]), &g = tensor(p[3]), &state = tensor(p[4]);
  const double scale = number(p[5]);
  const Maybe out = maybe(p[6]), state_out = maybe(p[7]);
  Attn a(q, k, v, g, 3);
  is_state(state, q, "state");
  is_state(state_out, q, "state_out");
  if (out) {
    same_type(q, *out);
    is_heads(*out, q, "out");
    apart(*out, {&q, &k, &v, &g, &state, at_of(state_out)}, "out");
  }
  const Tensor& next = state_out ? *state_out : state;
  apart(next, {&q, &k, &v, &g}, "the new state");
  if (state_out && state_out->data_ptr() != state.data_ptr()) apart(next, {&state}, "state_out");
  on_device(q, {&k, &v, &g, &state, at_of(out), at_of(state_out)});
  On on(q);
  a.decays();
  const Tensor o = out ? *out : make({a.B, a.H, a.D}, q, q.scalar_type());
  done("hdc_decay_attn_step",
       hdc_decay_attn_step(a.code, ptr(q), q.stride(0), q.stride(1), ptr(k), k.stride(0), k.stride(1), ptr(v), v.stride(0),
                           v.stride(1), ptr<float>(a.g), ptr<float>(state), (float)scale, ptr(o), o.stride(0), o.stride(1),
                           ptr<float>(next), a.B, a.H, a.D, on.stream));
  if (out) written(o);
  written(next);
  return tuple(o, next);
}
PyObject* py_embedding(PyObject* const* a) { return wrap(lookup(tensor(a[0]), tensor(a[1]), number(a[2]), maybe(a[3]))); }
// (subclasses of Tensor, but for Parameter, may mean something else by a lookup)
PyObject* py_embedding_takes(PyObject* const* a) {
  return PyBool_FromLong(THPVariable_CheckExact(a[0]) && THPVariable_CheckExact(a[1]) && takes(tensor(a[0]), tensor(a[1])));
}
PyObject* py_embedding_bwd(PyObject* const* a) {
  return wrap(lookup_backward(tensor(a[0]), tensor(a[1]), whole(a[2]), number(a[3]), a[4] == Py_None ? -1 : whole(a[4]), maybe(a[5])));
}
PyObject* py_embedding_train(PyObject* const* a) {
  return wrap(Embedding::apply(tensor(a[1]), tensor(a[0]), number(a[2]), a[3] == Py_None ? (int64_t)-1 : whole(a[3])));
}

// a sequence's tensors: contiguous, of one device; their addresses, types and sizes.  It holds the tensors: a
// generator's would otherwise be gone before the kernels are launched, and their memory another tensor's.
struct List {
  std::vector<Tensor> tensors;
  std::vector<void*> at;
  std::vector<int> codes;
  std::vector<int64_t> sizes;
  Tensor first;
  explicit List(PyObject* sequence) {
    PyObject* s = PySequence_Fast(sequence, "hdcmamba_b200: a sequence of tensors is wanted");
    if (!s) throw python_error();
    const std::unique_ptr<PyObject, void (*)(PyObject*)> hold(s, [](PyObject* o) { Py_DECREF(o); });
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(s);
    tensors.reserve(n);
    at.reserve(n);
    codes.reserve(n);
    sizes.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const Tensor& t = tensor(PySequence_Fast_GET_ITEM(s, i));
      if (i == 0) first = t;
      TORCH_CHECK_VALUE(t.device() == first.device(), "tensors must be on one device (", first.device(), ", got ", t.device(), ")");
      TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.is_contiguous(), "clip_grads needs contiguous tensors");
      codes.push_back(code_of(t));
      tensors.push_back(t);
      at.push_back(t.data_ptr());
      sizes.push_back(t.numel());
    }
  }
};
PyObject* py_clip(PyObject* const* a) {
  const List grads(a[0]);
  const int64_t n = (int64_t)grads.at.size();
  TORCH_CHECK_VALUE(n > 0, "clip_grads needs at least one gradient");
  std::optional<List> out;
  if (a[2] != Py_None) {
    out.emplace(a[2]);
    TORCH_CHECK_VALUE(out->codes == grads.codes && out->sizes == grads.sizes, "outputs must have their gradients' number, sizes and types");
  }
  on_device(grads.first, {out ? &out->first : nullptr});
  On on(grads.first);
  const Tensor norm = make({}, grads.first, at::kFloat);
  const size_t bytes = hdc_clip_grads_workspace_bytes(n);
  const auto ws = workspace(bytes);
  const bool scale = a[1] != Py_None;
  void* const* to = out ? out->at.data() : grads.at.data();
  done("hdc_clip_grads", hdc_clip_grads(n, grads.codes.data(), const_cast<const void* const*>(grads.at.data()),
                                        scale ? to : nullptr, grads.sizes.data(), scale ? (float)number(a[1]) : 0.f,
                                        ptr<float>(norm), ws.get(), bytes, on.stream));
  if (scale)
    for (const Tensor& t : (out ? *out : grads).tensors) written(t);
  return wrap(norm);
}
PyObject* py_set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XDECREF(g_error);
  g_error = type;
  Py_RETURN_NONE;
}

template <Py_ssize_t N, PyObject* (*F)(PyObject* const*)> PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<N, F>)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {
    method<8, py_attn>("decay_attention"),
    method<9, py_attn_bwd>("decay_attention_bwd"),
    method<6, py_attn_train>("decay_attention_train"),
    method<8, py_attn_step>("decay_attention_step"),
    method<4, py_embedding>("embedding"),
    method<2, py_embedding_takes>("embedding_takes"),
    method<6, py_embedding_bwd>("embedding_bwd"),
    method<4, py_embedding_train>("embedding_train"),
    method<3, py_clip>("clip_grads"),
    {"set_error", py_set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&g_module); }
