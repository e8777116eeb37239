// The training operators' Python calls: arguments checked and packed, outputs allocated, the C entries
// of libtriposplat_b200 called on PyTorch's current stream.  train_ops.py documents them and is their only
// caller.  The same work in Python took 11 to 15 us per call, as long as the kernels of a small one;
// here 2 to 4.
//
// A refused argument is a ValueError, a status of the library a RuntimeError.  The library's functions come
// as addresses (bind), so that it is loaded in one place, from whatever file the environment names.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/triposplat_b200.h"

namespace {

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

struct Refusal : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <class... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refusal(s.str());
}

// ---- the library ----
struct Library {
  decltype(&triposplat_b200_set_stream) set_stream;
  decltype(&triposplat_b200_last_error) last_error;
  decltype(&triposplat_b200_axis_rope) axis_rope;
  decltype(&triposplat_b200_axis_rope_backward) axis_rope_backward;
  decltype(&triposplat_b200_norm_gate) norm_gate;
  decltype(&triposplat_b200_norm_gate_backward) norm_gate_backward;
  decltype(&triposplat_b200_attention_forward) attention_forward;
  decltype(&triposplat_b200_attention_backward) attention_backward;
  decltype(&triposplat_b200_clip_grad_norm) clip_grad_norm;
} lib;
constexpr int kFunctions = sizeof(Library) / sizeof(void*);

void use_stream(at::Device d) {
  if (!d.is_cuda()) refuse("expected CUDA tensors, got ", d);
  if (d.has_index() && d.index() != c10::cuda::current_device())
    refuse("expected tensors on the current CUDA device, got ", d);
  lib.set_stream(c10::cuda::getCurrentCUDAStream().stream());
}

void ok(int status, const char* name) {
  if (status == 0) return;
  std::ostringstream s;
  s << name << " returned status " << status << ": " << lib.last_error();
  throw std::runtime_error(s.str());
}

// ---- arguments ----
std::string text(IntArrayRef v) {
  std::ostringstream s;
  s << '(';
  for (size_t i = 0; i < v.size(); ++i) s << (i ? ", " : "") << v[i];
  s << (v.size() == 1 ? ",)" : ")");
  return s.str();
}

const char* text(ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    std::ostringstream s;
    s << name << " must be a tensor, got " << Py_TYPE(o)->tp_name;
    throw c10::TypeError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, s.str());
  }
  return THPVariable_Unpack(o);
}

// an undefined tensor for None
Tensor optional(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }

int dtype_code(ScalarType t) { return t == at::kFloat ? 0 : (t == at::kBFloat16 ? 1 : (t == at::kHalf ? 2 : -1)); }

// a tensor of this shape, type and device (no conversion)
const Tensor& check(const Tensor& t, const char* name, IntArrayRef shape, ScalarType dtype, at::Device device) {
  if (t.scalar_type() == dtype && t.sizes() == shape && t.device() == device) return t;
  if (t.device() != device) refuse(name, " must be on ", device, ", got ", t.device());
  if (t.scalar_type() != dtype) refuse(name, " must be ", text(dtype), ", got ", text(t.scalar_type()));
  refuse(name, " must have shape ", text(shape), ", got ", text(t.sizes()));
}

// a float32 parameter, contiguous; None stays undefined
Tensor param(PyObject* o, const char* name, IntArrayRef shape, at::Device device) {
  Tensor t = optional(o, name);
  return t.defined() ? check(t, name, shape, at::kFloat, device).contiguous() : t;
}

// a tensor with a contiguous last dimension (a copy only if it has none)
Tensor rows(const Tensor& t) { return t.stride(-1) != 1 && t.size(-1) != 1 ? t.contiguous() : t; }

// New tensors, past the dispatcher (half of an allocation's time).
Tensor fresh(IntArrayRef sizes, ScalarType dtype, at::Device device) {
  if (!device.is_cuda()) refuse("expected CUDA tensors, got ", device);
  return Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}
Tensor fresh(const Tensor& like) { return fresh(like.sizes(), like.scalar_type(), like.device()); }

// an output of x's shape and type: `o` if given (unit last stride), a new one otherwise
Tensor out_like(PyObject* o, const Tensor& x, const char* name) {
  if (o == Py_None) return fresh(x);
  const Tensor& t = check(tensor(o, name), name, x.sizes(), x.scalar_type(), x.device());
  if (t.stride(-1) != 1 && t.size(-1) != 1) refuse(name, " needs a contiguous last dimension");
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) refuse(name, " must not be expanded");
  return t;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

Tensor like_param(const Tensor& t) { return t.defined() ? fresh(t) : t; }

// the first `n` strides of each tensor, one after the other (zeros for one that is not there)
template <int N, size_t M>
std::array<int64_t, N * M> strides(const std::array<const Tensor*, M>& ts) {
  std::array<int64_t, N * M> s;
  for (size_t i = 0; i < M; ++i)
    for (int k = 0; k < N; ++k) s[i * N + k] = ts[i]->defined() ? ts[i]->stride(k) : 0;
  return s;
}

PyObject* wrap(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

PyObject* tuple(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New(ts.size());
  Py_ssize_t i = 0;
  if (r)
    for (const Tensor& t : ts) PyTuple_SET_ITEM(r, i++, wrap(t));
  return r;
}

// A sequence's items, held while they are used.
struct Items {
  PyObject* seq;
  explicit Items(PyObject* o, const char* what) : seq(PySequence_Fast(o, what)) {
    if (!seq) throw python_error();
  }
  ~Items() { Py_DECREF(seq); }
  Items(const Items&) = delete;
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq); }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
};

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

int integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v > 2147483647 || v < -2147483647 ? -1 : (int)v;
}

// ---- rotary positions ----
struct Rope {
  Tensor positions, inv_freq, gamma;
  int dtype, kind, B, H, D, axes, layout, pairs[4];
  int64_t apart, L;
};

Rope rope_args(const Tensor& x, PyObject* positions, PyObject* inv_freq, PyObject* axis_pairs, PyObject* gamma,
               PyObject* layout) {
  Rope r;
  r.dtype = x.dim() == 4 ? dtype_code(x.scalar_type()) : -1;
  if (r.dtype < 0) refuse("x must be [B, L, H, D] in float32, bfloat16 or float16");
  const int64_t B = x.size(0), H = x.size(2), D = x.size(3);
  r.L = x.size(1);
  if (D % 2 || D <= 0 || D > 256 || !B || !r.L || !H || B > 65535 || H > 2147483647)
    refuse("unsupported shape ", text(x.sizes()), ": no empty dimension, D even and up to 256");
  r.B = (int)B; r.H = (int)H; r.D = (int)D;
  r.layout = integer(layout);
  if (r.layout < 0) refuse("layout must be 'interleaved' or 'halves'");
  const Items pairs(axis_pairs, "axis_pairs must be a sequence");
  const Py_ssize_t axes = pairs.size();
  int64_t total = 0;
  bool good = axes >= 1 && axes <= 4;
  for (Py_ssize_t a = 0; good && a < axes; ++a) {
    r.pairs[a] = integer(pairs[a]);
    good = r.pairs[a] >= 0;
    total += r.pairs[a];
  }
  if (!good || total > D / 2) refuse("axis_pairs must be 1 to 4 counts of at most ", D / 2, " pairs in all");
  r.axes = (int)axes;
  const Tensor& p = tensor(positions, "positions");
  r.kind = p.scalar_type() == at::kInt ? 0 : (p.scalar_type() == at::kLong ? 1 : (p.scalar_type() == at::kFloat ? 2 : -1));
  if (r.kind < 0) refuse("positions must be int32, int64 or float32, got ", text(p.scalar_type()));
  if (p.sizes() == IntArrayRef({r.L, (int64_t)axes})) r.apart = 0;
  else if (p.sizes() == IntArrayRef({B, r.L, (int64_t)axes})) r.apart = r.L * axes;
  else refuse("positions must be [L, axes] or [B, L, axes], got ", text(p.sizes()));
  if (p.device() != x.device()) refuse("positions must be on ", x.device());
  r.positions = p.contiguous();
  r.inv_freq = check(tensor(inv_freq, "inv_freq"), "inv_freq", {total}, at::kFloat, x.device()).contiguous();
  r.gamma = param(gamma, "gamma", {H, D}, x.device());
  return r;
}

PyObject* axis_rope(PyObject* const* a) {  // x, positions, inv_freq, axis_pairs, gamma, layout, out
  const Tensor& given = tensor(a[0], "x");
  const Rope r = rope_args(given, a[1], a[2], a[3], a[4], a[5]);
  const Tensor x = rows(given), y = out_like(a[6], x, "out");
  const auto s = strides<3, 2>({&x, &y});
  use_stream(x.device());
  ok(lib.axis_rope(ptr(x), ptr(r.positions), fptr(r.inv_freq), fptr(r.gamma), ptr(y), s.data(), r.dtype, r.kind, r.apart,
                   r.B, r.L, r.H, r.D, r.pairs, r.axes, r.layout), "axis_rope");
  return wrap(y);
}

PyObject* axis_rope_backward(PyObject* const* a) {  // dy, x, positions, inv_freq, axis_pairs, gamma, layout, out
  const Tensor& given = tensor(a[0], "dy");
  const Rope r = rope_args(given, a[2], a[3], a[4], a[5], a[6]);
  const Tensor dy = rows(given), dx = out_like(a[7], dy, "out");
  Tensor x, dgamma;
  if (r.gamma.defined()) {
    x = rows(check(tensor(a[1], "x"), "x", dy.sizes(), dy.scalar_type(), dy.device()));
    dgamma = like_param(r.gamma);
  }
  const auto s = strides<3, 3>({&dy, &x, &dx});
  use_stream(dy.device());
  ok(lib.axis_rope_backward(ptr(dy), ptr(x), ptr(r.positions), fptr(r.inv_freq), fptr(r.gamma), ptr(dx), fptr(dgamma),
                            s.data(), r.dtype, r.kind, r.apart, r.B, r.L, r.H, r.D, r.pairs, r.axes, r.layout),
     "axis_rope_backward");
  return tuple({dx, dgamma});
}

// ---- norms with gate and residual ----
struct Norm {
  Tensor x, y, gate, scale, shift, wpre, wpost;
  int dtype, pre, post, B, C;
  int64_t L;
  float rho;
};

// a: x, y, then gate, scale, shift, pre, pre_weight, post, post_weight, residual_scale
Norm norm_args(PyObject* px, PyObject* py, PyObject* const* a) {
  Norm n;
  const Tensor& x = tensor(px, "x");
  n.dtype = x.dim() == 3 ? dtype_code(x.scalar_type()) : -1;
  if (n.dtype < 0) refuse("x must be [B, L, C] in float32, bfloat16 or float16");
  const int64_t B = x.size(0), C = x.size(2);
  n.L = x.size(1);
  if (!B || !n.L || !C || C > 8192 || B > 65535)
    refuse("unsupported shape ", text(x.sizes()), ": no empty dimension, C up to 8192");
  n.B = (int)B; n.C = (int)C;
  n.pre = integer(a[3]);
  n.post = integer(a[5]);
  if (n.pre < 0 || n.post < 0) refuse("pre and post must be 'layer', 'rms' or None");
  if ((a[1] == Py_None) != (a[2] == Py_None)) refuse("scale and shift come together");
  if (n.pre == 0 && (a[1] != Py_None || a[4] != Py_None)) refuse("scale, shift and pre_weight need a pre norm");
  if (n.post == 0 && a[6] != Py_None) refuse("post_weight needs a post norm");
  const at::Device d = x.device();
  n.y = rows(check(tensor(py, "y"), "y", x.sizes(), x.scalar_type(), d));
  n.gate = param(a[0], "gate", {B, C}, d);
  n.scale = param(a[1], "scale", {B, C}, d);
  n.shift = param(a[2], "shift", {B, C}, d);
  n.wpre = param(a[4], "pre_weight", {C}, d);
  n.wpost = param(a[6], "post_weight", {C}, d);
  n.rho = (float)number(a[7]);
  n.x = rows(x);
  return n;
}

PyObject* norm_gate(PyObject* const* a) {  // x, y, the eight of norm_args, eps
  const Norm n = norm_args(a[0], a[1], a + 2);
  const float eps = (float)number(a[10]);
  const Tensor z = fresh(n.x), h = n.pre ? fresh(n.x) : Tensor(), stats = fresh({n.B, n.L, 4}, at::kFloat, n.x.device());
  const auto s = strides<2, 2>({&n.x, &n.y});
  use_stream(n.x.device());
  ok(lib.norm_gate(ptr(n.x), ptr(n.y), s.data(), fptr(n.gate), fptr(n.scale), fptr(n.shift), fptr(n.wpre), fptr(n.wpost),
                   ptr(z), ptr(h), fptr(stats), n.dtype, n.B, n.L, n.C, n.pre, n.post, n.rho, eps), "norm_gate");
  return tuple({z, h, stats});
}

PyObject* norm_gate_backward(PyObject* const* a) {  // dz, dh, x, y, stats, the eight of norm_args
  const Norm n = norm_args(a[2], a[3], a + 5);
  if (a[0] == Py_None && a[1] == Py_None) refuse("at least one of dz and dh is needed");
  if (a[1] != Py_None && n.pre == 0) refuse("dh needs a pre norm");
  auto grad = [&](PyObject* o, const char* name) {
    return o == Py_None ? Tensor() : rows(check(tensor(o, name), name, n.x.sizes(), n.x.scalar_type(), n.x.device()));
  };
  const Tensor dz = grad(a[0], "dz"), dh = grad(a[1], "dh");
  const Tensor stats = check(tensor(a[4], "stats"), "stats", {n.B, n.L, 4}, at::kFloat, n.x.device()).contiguous();
  const Tensor dx = fresh(n.x), dy = fresh(n.x);
  const Tensor dgate = like_param(n.gate), dscale = like_param(n.scale), dshift = like_param(n.shift),
               dwpre = like_param(n.wpre), dwpost = like_param(n.wpost);
  const auto s = strides<2, 4>({&n.x, &n.y, &dz, &dh});
  use_stream(n.x.device());
  ok(lib.norm_gate_backward(ptr(dz), ptr(dh), ptr(n.x), ptr(n.y), s.data(), fptr(stats), fptr(n.gate), fptr(n.scale),
                            fptr(n.wpre), fptr(n.wpost), ptr(dx), ptr(dy), fptr(dgate), fptr(dscale), fptr(dshift),
                            fptr(dwpre), fptr(dwpost), n.dtype, n.B, n.L, n.C, n.pre, n.post, n.rho),
     "norm_gate_backward");
  return tuple({dx, dy, dgate, dscale, dshift, dwpre, dwpost});
}

// ---- attention ----
struct Attention {
  Tensor q, k, v, bias;
  int B, H, Lq, Lk, bias_b = 1, bias_h = 1;
  at::Device device = at::kCPU;
};

Attention attention_args(PyObject* pq, PyObject* pk, PyObject* pv, PyObject* pbias) {
  Attention t;
  const Tensor &q = tensor(pq, "q"), &k = tensor(pk, "k"), &v = tensor(pv, "v");
  if (q.dim() != 4 || k.dim() != 4) refuse("q, k, v must be [B, H, L, 64]");
  const int64_t B = q.size(0), H = q.size(1), Lq = q.size(2), Lk = k.size(2);
  if (q.size(3) != 64 || !B || !H || !Lq || !Lk || std::max(std::max(B, H), std::max(Lq, Lk)) > 2147483647)
    refuse("unsupported shapes ", text(q.sizes()), ", ", text(k.sizes()), ": head_dim 64, no empty dimension");
  t.device = q.device();
  t.q = rows(check(q, "q", q.sizes(), at::kFloat, t.device));
  t.k = rows(check(k, "k", {B, H, Lk, 64}, at::kFloat, t.device));
  t.v = rows(check(v, "v", {B, H, Lk, 64}, at::kFloat, t.device));
  t.B = (int)B; t.H = (int)H; t.Lq = (int)Lq; t.Lk = (int)Lk;
  if (pbias != Py_None) {
    const Tensor& b = tensor(pbias, "key_bias");
    const IntArrayRef s = b.sizes();
    if (s == IntArrayRef({B, H, Lk})) { t.bias_b = t.B; t.bias_h = t.H; }
    else if (s == IntArrayRef({B, Lk})) t.bias_b = t.B;
    else if (s != IntArrayRef({Lk})) refuse("key_bias must be [Lk], [B, Lk] or [B, H, Lk], got ", text(s));
    t.bias = check(b, "key_bias", s, at::kFloat, t.device).contiguous();
  }
  return t;
}

// a new [B, H, L, 64] in token-major storage [B, L, H, 64]
Tensor token_major(const Attention& t, int64_t L) {
  if (!t.device.is_cuda()) refuse("expected CUDA tensors, got ", t.device);
  return Tensor(at::detail::empty_strided_cuda({t.B, t.H, L, 64}, {L * t.H * 64, 64, (int64_t)t.H * 64, 1}, at::kFloat, t.device));
}

PyObject* attention_forward(PyObject* const* a) {  // q, k, v, key_bias
  const Attention t = attention_args(a[0], a[1], a[2], a[3]);
  const Tensor out = token_major(t, t.Lq), stats = fresh({t.B, t.H, t.Lq + 1, 2}, at::kFloat, t.device);
  const auto s = strides<3, 3>({&t.q, &t.k, &t.v});
  use_stream(t.device);
  ok(lib.attention_forward(fptr(t.q), fptr(t.k), fptr(t.v), s.data(), fptr(t.bias), t.bias_b, t.bias_h, fptr(out),
                           fptr(stats), t.B, t.H, t.Lq, t.Lk), "attention_forward");
  return tuple({out, stats});
}

PyObject* attention_backward(PyObject* const* a) {  // dout, q, k, v, out, stats, key_bias, grads, bias_grad
  const Attention t = attention_args(a[1], a[2], a[3], a[6]);
  const Tensor dout = rows(check(tensor(a[0], "dout"), "dout", t.q.sizes(), at::kFloat, t.device));
  const Tensor out = rows(check(tensor(a[4], "out"), "out", t.q.sizes(), at::kFloat, t.device));
  const Tensor stats =
      check(tensor(a[5], "stats"), "stats", {t.B, t.H, (int64_t)t.Lq + 1, 2}, at::kFloat, t.device).contiguous();
  Tensor dq, dk, dv, dbias;
  if (a[7] == Py_None) {
    dq = token_major(t, t.Lq);
    dk = token_major(t, t.Lk);
    dv = token_major(t, t.Lk);
  } else {
    const Items grads(a[7], "grads must be a sequence");
    if (grads.size() != 3) refuse("grads must be three tensors, got ", grads.size());
    for (int i = 0; i < 3; ++i)
      if (grads[i] == Py_None) refuse("grads must be three tensors");
    dq = out_like(grads[0], t.q, "grads");
    dk = out_like(grads[1], t.k, "grads");
    dv = out_like(grads[2], t.v, "grads");
  }
  const int want = PyObject_IsTrue(a[8]);
  if (want < 0) throw python_error();
  if (want) dbias = like_param(t.bias);
  const auto s = strides<3, 8>({&dout, &t.q, &t.k, &t.v, &out, &dq, &dk, &dv});
  use_stream(t.device);
  ok(lib.attention_backward(fptr(dout), fptr(t.q), fptr(t.k), fptr(t.v), fptr(out), fptr(stats), s.data(), fptr(t.bias),
                            t.bias_b, t.bias_h, fptr(dq), fptr(dk), fptr(dv), fptr(dbias), t.B, t.H, t.Lq, t.Lk),
     "attention_backward");
  return tuple({dq, dk, dv, dbias});
}

// ---- gradient norm, clipping ----
PyObject* clip_grad_norm(PyObject* const* a) {  // grads, max_norm, out
  const Items grads(a[0], "grads must be a sequence");
  const Items outs(a[2] == Py_None ? grads.seq : a[2], "out must be a sequence");
  const Py_ssize_t n = grads.size();
  if (outs.size() != n) refuse(n, " gradients and ", outs.size(), " outputs");
  if (n == 0) refuse("no gradients");
  if (n > 2147483647) refuse("too many gradients");
  const float max_norm = (float)number(a[1]);
  if (!(max_norm >= 0.0f)) refuse("max_norm must be zero or more, got ", max_norm);
  std::vector<const void*> in(n);
  std::vector<void*> to(n);
  std::vector<int64_t> sizes(n);
  std::vector<int> types(n);
  const at::Device device = tensor(grads[0], "grads").device();
  for (Py_ssize_t i = 0; i < n; ++i) {
    const Tensor &g = tensor(grads[i], "grads"), &o = tensor(outs[i], "out");
    types[i] = dtype_code(g.scalar_type());
    if (g.device() != device || o.device() != device || types[i] < 0 || o.scalar_type() != g.scalar_type())
      refuse("gradients and outputs must be float32, bfloat16 or float16 tensors of one device, an output of its "
             "gradient's type");
    if (!g.is_contiguous() || !o.is_contiguous() || o.sizes() != g.sizes())
      refuse("gradients and outputs must be contiguous, an output of its gradient's shape");
    in[i] = g.data_ptr();
    to[i] = o.data_ptr();
    sizes[i] = g.numel();
  }
  use_stream(device);
  const Tensor norm = fresh({}, at::kFloat, device);
  ok(lib.clip_grad_norm(in.data(), a[2] == Py_None ? nullptr : to.data(), sizes.data(), types.data(), (int)n, max_norm,
                        fptr(norm)), "clip_grad_norm");
  return wrap(norm);
}

// ---- the module ----
// One function of N positional arguments.  Below autograd: what is allocated or copied here has no history.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N || !lib.set_stream) {
    PyErr_SetString(PyExc_TypeError, n != N ? "wrong number of arguments" : "bind() has not been called");
    return nullptr;
  }
  try {
    const at::AutoDispatchBelowADInplaceOrView below;
    return F(args);
  } catch (const Refusal& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* addresses) {
  HANDLE_TH_ERRORS
  const Items a(addresses, "bind() takes a sequence of addresses");
  if (a.size() != kFunctions) {
    PyErr_Format(PyExc_ValueError, "bind() takes %d addresses", kFunctions);
    return nullptr;
  }
  void* f[kFunctions];
  for (int i = 0; i < kFunctions; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind(): an address is null");
      return nullptr;
    }
  }
  static_assert(sizeof(f) == sizeof(lib), "one address per function");
  memcpy(static_cast<void*>(&lib), f, sizeof(f));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_O, nullptr},
                         ENTRY(axis_rope, 7),
                         ENTRY(axis_rope_backward, 8),
                         ENTRY(norm_gate, 11),
                         ENTRY(norm_gate_backward, 13),
                         ENTRY(attention_forward, 4),
                         ENTRY(attention_backward, 9),
                         ENTRY(clip_grad_norm, 3),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "train_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_train_calls() { return PyModule_Create(&module); }
