// torch front-end of cross attention and of the query / key norm with rotation:
// argument checks, allocation and autograd nodes in C++.  A call of one token
// takes the host a few microseconds here; the same steps in Python took 18 us
// forward, and a backward, whose Python would run on autograd's own thread,
// 150 us more than the kernels of a small step.
//
// Holds no kernels: bind() takes the addresses of the C entries (tgfr.h) from
// the library that the process has loaded.
#include <limits>

#include <ATen/Functions.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <sstream>

#include "tgfr.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

decltype(&tgfr_cross_attention_ws) c_attn_ws;
decltype(&tgfr_cross_attention_fwd) c_attn_fwd;
decltype(&tgfr_cross_attention_bwd) c_attn_bwd;
decltype(&tgfr_qk_norm_rope_ws) c_norm_ws;
decltype(&tgfr_qk_norm_rope_fwd) c_norm_fwd;
decltype(&tgfr_qk_norm_rope_bwd) c_norm_bwd;

void bind(const std::map<std::string, uintptr_t>& at) {
  c_attn_ws = (decltype(c_attn_ws))at.at("tgfr_cross_attention_ws");
  c_attn_fwd = (decltype(c_attn_fwd))at.at("tgfr_cross_attention_fwd");
  c_attn_bwd = (decltype(c_attn_bwd))at.at("tgfr_cross_attention_bwd");
  c_norm_ws = (decltype(c_norm_ws))at.at("tgfr_qk_norm_rope_ws");
  c_norm_fwd = (decltype(c_norm_fwd))at.at("tgfr_qk_norm_rope_fwd");
  c_norm_bwd = (decltype(c_norm_bwd))at.at("tgfr_qk_norm_rope_bwd");
}

template <class... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
template <class... A>
[[noreturn]] void bad_value(const A&... a) {
  throw py::value_error(text(a...));
}
template <class... A>
[[noreturn]] void bad_type(const A&... a) {
  throw py::type_error(text(a...));
}
void done(const char* name, int rc) {
  if (rc != 0) throw std::runtime_error(text(name, " failed with code ", rc));
}

// the tensor behind a Python argument; None: an undefined one
Tensor given(py::handle h, const char* name) {
  if (h.is_none()) return Tensor();
  if (!THPVariable_Check(h.ptr())) bad_type(name, " must be a tensor");
  return THPVariable_Unpack(h.ptr());
}
py::object wrapped(const Tensor& t) {
  if (!t.defined()) return py::none();
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(t));
}

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : t == at::kHalf ? 2 : -1;
}
void head_tensor(const char* name, const Tensor& x) {
  if (x.dim() != 4)
    bad_value(name, " must be [batch, tokens, heads, head_dim], got ", x.sizes());
  if (type_code(x.scalar_type()) < 0)
    bad_type(name, " must be float32, bfloat16 or float16, got ", x.scalar_type());
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// last axis dense (a copy only where it is not)
Tensor dense(const Tensor& t) {
  return !t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}
// (that of an axis of one means nothing and may be anything)
int64_t stride(const Tensor& t, int axis) { return t.size(axis) == 1 ? 0 : t.stride(axis); }
// the kernels reach the rows of a tile by 32-bit offsets: tensors whose tokens
// (or shared heads) lie further apart are copied
Tensor near(const Tensor& t, int64_t heads) {
  const Tensor d = dense(t);
  const int64_t size = (int64_t)d.element_size();
  return (160 * stride(d, 1) + heads * stride(d, 2) + 256) * size < (1LL << 31) ? d
                                                                              : d.contiguous();
}
Tensor floats(int64_t n, const Tensor& like) {
  return at::empty({n}, like.options().dtype(at::kFloat).requires_grad(false));
}
Tensor shaped(const Tensor& t, at::ScalarType type) {
  return at::empty(t.sizes(), t.options().dtype(type).requires_grad(false));
}
void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
// the refusal that comes last, so that every other one needs no GPU
void on_device(const Tensor& x, std::initializer_list<std::pair<const char*, Tensor>> others) {
  for (const auto& o : others)
    if (o.second.defined() && o.second.device() != x.device())
      throw std::runtime_error(
          text(o.first, " is on ", o.second.device(), ", the others on ", x.device()));
  if (!x.is_cuda())
    throw std::runtime_error("tgfr kernels take device tensors only (no CPU path)");
}
void no_second_derivative(const char* name) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(text("the backward of ", name, " is not differentiable"));
}

// A node is made by requires_grad alone: a tangent would be lost in silence.
void no_tangent(const char* name, std::initializer_list<Tensor> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : inputs)
    if (t.defined() && t._fw_grad(0).defined())
      throw std::runtime_error(text(name, " has no forward-mode derivative"));
}

// A trace would record the output's allocation and not the kernel.
void no_trace(const char* name) {
  if (torch::jit::tracer::isTracing())
    throw std::runtime_error(text(name, " cannot be traced"));
}

// --------------------------------------------------------- cross attention ---
struct Attn {
  Tensor q, k, v, q_lens, kv_lens, mask;
  float scale;
  int64_t b, tq, tk, h, hk, d;
  int type;
  bool empty() const { return !q.numel() || !k.numel(); }
  void sizes() {
    b = q.size(0), tq = q.size(1), h = q.size(2), d = q.size(3);
    tk = k.size(1), hk = k.size(2);
    type = type_code(q.scalar_type());
  }
  int64_t mask_sb() const { return mask.defined() ? mask.stride(0) : 0; }
};
int64_t* strides(int64_t* s, const Tensor& t) {
  for (int i = 0; i < 3; ++i) *s++ = stride(t, i);
  return s;
}

Tensor attn_forward(const Attn& a, Tensor* lse) {
  const c10::DeviceGuard guard(a.q.device());
  Tensor o = shaped(a.q, a.q.scalar_type());
  if (lse) *lse = at::empty({a.b, a.hk, a.tq * (a.h / a.hk)}, o.options().dtype(at::kFloat));
  if (a.empty()) return o.zero_();
  long long n = 0, s[12];
  done("tgfr_cross_attention_ws",
       c_attn_ws(a.b, a.tq, a.tk, a.h, a.hk, a.d, a.type, 0, &n));
  const Tensor ws = n ? floats(n, a.q) : Tensor();
  strides((int64_t*)s, a.q);
  strides((int64_t*)s + 3, a.k);
  strides((int64_t*)s + 6, a.v);
  strides((int64_t*)s + 9, o);
  done("tgfr_cross_attention_fwd",
       c_attn_fwd(ptr(a.q), ptr(a.k), ptr(a.v), ptr(o), s, (const int*)ptr(a.q_lens),
                  (const int*)ptr(a.kv_lens), (const uint8_t*)ptr(a.mask), a.mask_sb(), a.b, a.tq,
                  a.tk, a.h, a.hk, a.d, a.scale, a.type, lse ? (float*)ptr(*lse) : nullptr,
                  (float*)ptr(ws), stream_of(a.q)));
  return o;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Attn* a) {
    Tensor lse;
    Tensor o = attn_forward(*a, &lse);
    ctx->save_for_backward({a->q, a->k, a->v, o, lse, a->q_lens, a->kv_lens, a->mask});
    ctx->saved_data["scale"] = (double)a->scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("cross_attention");
    const variable_list s = ctx->get_saved_variables();
    Attn a;
    a.q = s[0], a.k = s[1], a.v = s[2], a.q_lens = s[5], a.kv_lens = s[6], a.mask = s[7];
    a.sizes();
    a.scale = (float)ctx->saved_data["scale"].toDouble();
    const Tensor &o = s[3], &lse = s[4];
    const c10::DeviceGuard guard(a.q.device());
    const bool want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dq = shaped(a.q, a.q.scalar_type()), dk, dv;
    if (want_kv) {
      dk = shaped(a.k, a.k.scalar_type());
      dv = shaped(a.k, a.k.scalar_type());
    }
    if (a.empty()) {
      dq.zero_();
      if (want_kv) dk.zero_(), dv.zero_();
      return {dq, dk, dv, Tensor()};
    }
    const Tensor g = near(grads[0], a.h / a.hk);
    long long n = 0, st[24] = {};
    done("tgfr_cross_attention_ws",
         c_attn_ws(a.b, a.tq, a.tk, a.h, a.hk, a.d, a.type, 1, &n));
    const Tensor ws = floats(n, a.q);
    int64_t* at = (int64_t*)st;
    for (const Tensor& t : variable_list{a.q, a.k, a.v, o, g, dq}) at = strides(at, t);
    if (want_kv) strides(strides(at, dk), dv);
    done("tgfr_cross_attention_bwd",
         c_attn_bwd(ptr(a.q), ptr(a.k), ptr(a.v), ptr(o), ptr(g), ptr(dq), ptr(dk), ptr(dv), st,
                    (const int*)ptr(a.q_lens), (const int*)ptr(a.kv_lens),
                    (const uint8_t*)ptr(a.mask), a.mask_sb(), a.b, a.tq, a.tk, a.h, a.hk, a.d,
                    a.scale, a.type, (const float*)ptr(lse), (float*)ptr(ws), stream_of(a.q)));
    return {dq, dk, dv, Tensor()};
  }
};

Tensor lens_given(py::handle h, const char* name, int64_t n) {
  if (h.is_none()) return Tensor();
  const bool is = THPVariable_Check(h.ptr());
  const Tensor t = is ? THPVariable_Unpack(h.ptr()) : Tensor();
  if (!is || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.dim() != 1 ||
      t.size(0) != n)
    bad_value(name, " must be an int32 or int64 tensor of ", n, " lengths");
  return t;
}

py::object cross_attention(py::handle hq, py::handle hk, py::handle hv, py::handle hscale,
                           py::handle hql, py::handle hkl, py::handle hmask) {
  no_trace("cross_attention");
  Attn a;
  a.q = given(hq, "q"), a.k = given(hk, "k"), a.v = given(hv, "v");
  for (const auto& x : {std::make_pair("q", &a.q), std::make_pair("k", &a.k),
                        std::make_pair("v", &a.v)}) {
    if (!x.second->defined()) bad_type(x.first, " must be a tensor");
    head_tensor(x.first, *x.second);
  }
  if (a.k.sizes() != a.v.sizes()) bad_value("k and v differ: ", a.k.sizes(), ", ", a.v.sizes());
  if (a.k.scalar_type() != a.q.scalar_type() || a.v.scalar_type() != a.q.scalar_type())
    bad_type("q, k and v need one type, got ", a.q.scalar_type(), ", ", a.k.scalar_type(), ", ",
             a.v.scalar_type());
  a.sizes();
  if (a.k.size(0) != a.b || a.k.size(3) != a.d)
    bad_value("q ", a.q.sizes(), " and k ", a.k.sizes(), " need one batch and head size");
  if (a.d < 1 || a.d > 256) bad_value("head size must be 1 to 256, got ", a.d);
  if (a.hk < 1 || a.h < 1 || a.h % a.hk)
    bad_value(a.h, " query heads are no multiple of ", a.hk, " key heads");
  constexpr int64_t most = 1LL << 30;
  if (a.tq > most || a.tk > most || a.b > most || a.h > most ||
      (double)a.b * a.h * std::max(a.tq, a.tk) > (double)most)
    bad_value("at most 2^30 rows of queries or keys");
  if (a.b * a.hk >= 1LL << 24) bad_value("at most 2^24 - 1 key heads of all samples");
  const double scale = hscale.is_none() ? 1.0 / std::sqrt((double)a.d) : hscale.cast<double>();
  if (!((float)scale > 0.f) || std::isinf((float)scale))
    bad_value("scale must be positive and finite, got ", scale);
  a.scale = (float)scale;
  a.q_lens = lens_given(hql, "q_lens", a.b);
  a.kv_lens = lens_given(hkl, "kv_lens", a.b);
  a.mask = given(hmask, "mask");
  if (a.mask.defined() && (a.mask.scalar_type() != at::kBool || a.mask.dim() != 2 ||
                           a.mask.size(0) != a.b || a.mask.size(1) != a.tk))
    bad_value("mask must be a bool tensor [", a.b, ", ", a.tk, "]");
  no_tangent("cross_attention", {a.q, a.k, a.v});
  on_device(a.q, {{"k", a.k}, {"v", a.v}, {"q_lens", a.q_lens}, {"kv_lens", a.kv_lens},
                  {"mask", a.mask}});
  for (at::Tensor* lens : {&a.q_lens, &a.kv_lens})
    if (lens->defined()) {
      if (lens->scalar_type() == at::kLong)             // (must not wrap)
        *lens = lens->clamp(-1, std::numeric_limits<int>::max()).to(at::kInt);
      *lens = lens->contiguous();
    }
  if (a.mask.defined()) a.mask = dense(a.mask);
  const bool grad = at::GradMode::is_enabled() &&
                    (a.q.requires_grad() || a.k.requires_grad() || a.v.requires_grad());
  a.q = near(a.q, a.h / a.hk), a.k = near(a.k, 1), a.v = near(a.v, 1);
  return wrapped(grad ? CrossAttention::apply(a.q, a.k, a.v, (const Attn*)&a)
                      : attn_forward(a, nullptr));
}

// ------------------------------------------------- norm of heads + rotation ---
struct Norm {
  Tensor x[2], w[2], pos[2], turn;
  int64_t ps[2][3] = {};       // strides of the positions
  double eps;
  int64_t rot, axes, d;
  bool interleaved;
  at::ScalarType out;
  const Tensor& any() const { return x[0].defined() ? x[0] : x[1]; }
};

void norm_call(const Norm& a, const Tensor* g, const Tensor* y, const Tensor* ws,
               const Tensor* dw) {
  const Tensor& x = a.any();
  const c10::DeviceGuard guard(x.device());
  long long s[30] = {};
  for (int i = 0; i < 2; ++i) {
    if (!a.x[i].defined()) continue;
    int64_t* t = (int64_t*)s + 15 * i;
    for (int j = 0; j < 3; ++j) t[j] = a.x[i].size(j);
    strides(t + 3, a.x[i]);
    if (g) strides(t + 6, g[i]);
    strides(t + 9, y[i]);
    for (int j = 0; j < 3; ++j) t[12 + j] = a.ps[i][j];
  }
  const Tensor& pos = a.pos[0].defined() ? a.pos[0] : a.pos[1];
  const int p32 = pos.defined() && pos.scalar_type() == at::kInt;
  const auto* turn = (const unsigned long long*)ptr(a.turn);
  const int ti = type_code(x.scalar_type()), to = type_code(a.out);
  if (g)
    done("tgfr_qk_norm_rope_bwd",
         c_norm_bwd(ptr(a.x[0]), ptr(a.x[1]), ptr(g[0]), ptr(g[1]), ptr(y[0]), ptr(y[1]), s,
                    (const float*)ptr(a.w[0]), (const float*)ptr(a.w[1]), ptr(a.pos[0]),
                    ptr(a.pos[1]), p32, turn, a.rot, a.axes, a.interleaved, a.d, a.eps, ti, to,
                    (float*)ptr(*ws), (float*)ptr(dw[0]), (float*)ptr(dw[1]), stream_of(x)));
  else
    done("tgfr_qk_norm_rope_fwd",
         c_norm_fwd(ptr(a.x[0]), ptr(a.x[1]), ptr(y[0]), ptr(y[1]), s, (const float*)ptr(a.w[0]),
                    (const float*)ptr(a.w[1]), ptr(a.pos[0]), ptr(a.pos[1]), p32, turn, a.rot,
                    a.axes, a.interleaved, a.d, a.eps, ti, to, stream_of(x)));
}

void norm_forward(const Norm& a, Tensor* y) {
  const c10::DeviceGuard guard(a.any().device());
  for (int i = 0; i < 2; ++i)
    if (a.x[i].defined()) y[i] = shaped(a.x[i], a.out);
  norm_call(a, nullptr, y, nullptr, nullptr);
}

variable_list norm_node(AutogradContext* ctx, const Norm& a) {
  Tensor y[2];
  norm_forward(a, y);
  ctx->save_for_backward({a.x[0], a.x[1], a.w[0], a.w[1], a.pos[0], a.pos[1], a.turn});
  std::vector<int64_t> n;
  for (const auto& p : a.ps) n.insert(n.end(), p, p + 3);
  n.insert(n.end(), {a.rot, a.axes, a.interleaved, (int64_t)a.out});
  ctx->saved_data["n"] = n;
  ctx->saved_data["eps"] = a.eps;
  variable_list out;
  for (const Tensor& t : y)
    if (t.defined()) out.push_back(t);
  return out;
}
// gradients of the parts that are there, then of their weights
variable_list norm_node_backward(AutogradContext* ctx, const variable_list& grads) {
  no_second_derivative("qk_norm_rope");
  const variable_list s = ctx->get_saved_variables();
  const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
  Norm a;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = s[i], a.w[i] = s[2 + i], a.pos[i] = s[4 + i];
    for (int j = 0; j < 3; ++j) a.ps[i][j] = n[3 * i + j];
  }
  a.turn = s[6];
  a.eps = ctx->saved_data["eps"].toDouble();
  a.rot = n[6], a.axes = n[7], a.interleaved = n[8], a.out = (at::ScalarType)n[9];
  a.d = a.any().size(3);
  const c10::DeviceGuard guard(a.any().device());
  const int parts = (int)grads.size();
  Tensor g[2], dx[2], dw[2], ws;
  int part = 0;
  for (int i = 0; i < 2; ++i)
    if (a.x[i].defined()) {
      g[i] = dense(grads[part]);
      dx[i] = shaped(a.x[i], a.x[i].scalar_type());
      if (ctx->needs_input_grad(parts + part)) dw[i] = floats(a.d, a.any());
      ++part;
    }
  if (dw[0].defined() || dw[1].defined()) {
    long long f = 0;
    done("tgfr_qk_norm_rope_ws", c_norm_ws(a.d, &f));
    ws = floats(f, a.any());
  }
  norm_call(a, g, dx, &ws, dw);
  variable_list out;
  for (const auto& both : {dx, dw})
    for (int i = 0; i < 2; ++i)
      if (a.x[i].defined()) out.push_back(both[i]);
  out.emplace_back();
  return out;
}
struct NormBoth : torch::autograd::Function<NormBoth> {
  static variable_list forward(AutogradContext* ctx, const Tensor&, const Tensor&, const Tensor&,
                               const Tensor&, const Norm* a) {
    return norm_node(ctx, *a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return norm_node_backward(ctx, g);
  }
};
struct NormOne : torch::autograd::Function<NormOne> {
  static variable_list forward(AutogradContext* ctx, const Tensor&, const Tensor&,
                               const Norm* a) {
    return norm_node(ctx, *a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return norm_node_backward(ctx, g);
  }
};

void positions(const char* name, Norm& a, int i, bool rope) {
  const Tensor &p = a.pos[i], &x = a.x[i];
  if (!p.defined()) {
    if (a.axes > 1) bad_value(a.axes, " position axes need ", name);
    return;
  }
  if (!rope) bad_value(name, " without a rope");
  if (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)
    bad_type(name, " must be int32 or int64, got ", p.scalar_type());
  const int64_t tail = a.axes > 1 ? 2 : 1, lead = p.dim() - tail;
  bool ok = (lead == 0 || (lead == 1 && p.size(0) == x.size(0))) && p.size(lead) == x.size(1) &&
            (a.axes == 1 || p.size(lead + 1) == a.axes);
  if (!ok)
    bad_value(name, " must be [", x.size(1), a.axes > 1 ? ", axes]" : "]",
              " or the same for each sample, got ", p.sizes());
  a.ps[i][0] = lead ? p.stride(0) : 0;
  a.ps[i][1] = p.stride(lead);
  a.ps[i][2] = a.axes > 1 ? p.stride(lead + 1) : 0;
}

py::object qk_norm_rope(py::handle hq, py::handle hk, py::handle hwq, py::handle hwk, double eps,
                        py::handle hturn, int64_t rot, int64_t axes, bool interleaved,
                        py::handle hqp, py::handle hkp, py::handle hout) {
  no_trace("qk_norm_rope");
  Norm a;
  a.x[0] = given(hq, "q"), a.x[1] = given(hk, "k");
  a.turn = given(hturn, "rope");
  a.eps = eps, a.rot = rot, a.axes = axes, a.interleaved = interleaved;
  if (!a.x[0].defined() && !a.x[1].defined()) bad_value("neither q nor k");
  const Tensor& x = a.any();
  const char *names[2] = {"q", "k"}, *wn[2] = {"q_weight", "k_weight"}, *pn[2] = {"q_pos", "k_pos"};
  for (int i = 0; i < 2; ++i) {
    if (!a.x[i].defined()) continue;
    head_tensor(names[i], a.x[i]);
    if (a.x[i].scalar_type() != x.scalar_type() || a.x[i].size(3) != x.size(3))
      bad_value("q and k need one type and head size");
    a.w[i] = given(i ? hwk : hwq, wn[i]);
    if (!a.w[i].defined() || a.w[i].scalar_type() != at::kFloat || a.w[i].dim() != 1 ||
        a.w[i].size(0) != x.size(3))
      bad_value(wn[i], " must be float32 [", x.size(3), "]");
  }
  a.d = x.size(3);
  if (a.d % 2 || a.d < 2 || a.d > 256) bad_value("head size must be even and 2 to 256, got ", a.d);
  if (rot > a.d) bad_value("the rotation covers ", rot, " of ", a.d, " elements");
  if (!(eps >= 0.0)) bad_value("eps must not be negative, got ", eps);
  a.out = x.scalar_type();
  if (!hout.is_none()) {
    if (!THPDtype_Check(hout.ptr())) bad_type("out_dtype must be a torch.dtype");
    a.out = ((THPDtype*)hout.ptr())->scalar_type;
  }
  if (a.out != x.scalar_type() && (x.scalar_type() != at::kFloat || type_code(a.out) < 0))
    bad_type(x.scalar_type(), " cannot be written as ", a.out);
  for (int i = 0; i < 2; ++i)
    if (a.x[i].defined()) {
      a.pos[i] = given(i ? hkp : hqp, pn[i]);
      positions(pn[i], a, i, a.turn.defined());
    }
  if (a.pos[0].defined() && a.pos[1].defined() &&
      a.pos[0].scalar_type() != a.pos[1].scalar_type())
    bad_type("q_pos and k_pos need one type");
  constexpr int64_t most = 1LL << 30;
  for (const Tensor& t : a.x)
    if (t.defined() && (t.size(0) > most || t.size(1) > most || t.size(2) > most ||
                        t.size(0) * t.size(1) > most))
      bad_value("at most 2^30 tokens, and heads of one");
  if (a.turn.defined() &&
      (a.turn.scalar_type() != at::kLong || a.turn.dim() != 1 || !a.turn.is_contiguous() ||
       rot < 2 || axes < 1 || rot % (2 * axes) || a.turn.size(0) != rot / 2))
    bad_value("rope does not hold ", rot, " / 2 steps over ", axes, " axes");
  no_tangent("qk_norm_rope", {a.x[0], a.x[1], a.w[0], a.w[1]});
  on_device(x, {{"k", a.x[1]}, {"q_weight", a.w[0]}, {"k_weight", a.w[1]}, {"q_pos", a.pos[0]},
                {"k_pos", a.pos[1]}, {"rope", a.turn}});
  bool grad = false;
  for (int i = 0; i < 2; ++i)
    if (a.x[i].defined()) {
      grad = grad || a.x[i].requires_grad() || a.w[i].requires_grad();
      a.x[i] = dense(a.x[i]);
      a.w[i] = a.w[i].contiguous();
    }
  Tensor y[2];
  if (grad && at::GradMode::is_enabled()) {
    const int one = a.x[0].defined() ? 0 : 1;
    const variable_list o =
        a.x[0].defined() && a.x[1].defined()
            ? NormBoth::apply(a.x[0], a.x[1], a.w[0], a.w[1], (const Norm*)&a)
            : NormOne::apply(a.x[one], a.w[one], (const Norm*)&a);
    int at = 0;
    for (int i = 0; i < 2; ++i)
      if (a.x[i].defined()) y[i] = o[at++];
  } else {
    norm_forward(a, y);
  }
  return py::make_tuple(wrapped(y[0]), wrapped(y[1]));
}

}  // namespace

PYBIND11_MODULE(tgfr_front, m) {
  m.def("bind", &bind);
  m.def("cross_attention", &cross_attention);
  m.def("qk_norm_rope", &qk_norm_rope);
}
