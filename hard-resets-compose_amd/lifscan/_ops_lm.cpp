// The language-model operators (lifscan/hip_linattn.py, hip_lm.py, hip_gated.py) over the lifscan C ABI: argument
// checks, workspaces and autograd functions in C++, one Python -> C++ crossing a call.  (From Python the
// checks and the engine's calls back into the interpreter cost some 60 us a forward and backward, several
// times the kernels of small steps.)
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <map>
#include <string>
#include <tuple>

#include "lifscan_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = c10::optional<Tensor>;

struct Entry {
#define LSH_ENTRIES(X)            \
  X(lsh_status_string)            \
  X(lsh_linattn_workspace)        \
  X(lsh_linattn_fwd)              \
  X(lsh_linattn_bwd_workspace)    \
  X(lsh_linattn_bwd)              \
  X(lsh_linattn_step)             \
  X(lsh_block_norm_fwd)           \
  X(lsh_block_norm_bwd_workspace) \
  X(lsh_block_norm_bwd)           \
  X(lsh_embed_fwd)                \
  X(lsh_embed_bwd_workspace)      \
  X(lsh_embed_bwd)                \
  X(lsh_distill_workspace)        \
  X(lsh_distill_fwd)              \
  X(lsh_distill_bwd)              \
  X(lsh_gated_workspace)          \
  X(lsh_gated_saved)              \
  X(lsh_gated_fwd)                \
  X(lsh_gated_bwd)                \
  X(lsh_gated_step)               \
  X(lsh_rotate_fwd)               \
  X(lsh_rotate_bwd_workspace)     \
  X(lsh_rotate_bwd)               \
  X(lsh_score_workspace)          \
  X(lsh_score_fwd)                \
  X(lsh_score_bwd)
#define LSH_MEMBER(name) decltype(&::name) name = nullptr;
  LSH_ENTRIES(LSH_MEMBER)
#undef LSH_MEMBER
} g;
bool g_set = false;

void set_entry_points(const std::map<std::string, int64_t>& addresses) {
#define LSH_SET(name) g.name = reinterpret_cast<decltype(&::name)>(addresses.at(#name));
  LSH_ENTRIES(LSH_SET)
#undef LSH_SET
  g_set = true;
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  const std::string msg = std::string(what) + ": " + g.lsh_status_string(rc) + " (status " + std::to_string(rc) + ")";
  if (rc == -1 || rc == -2 || rc == -3) TORCH_CHECK_VALUE(false, msg);
  TORCH_CHECK(false, msg);
}

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}
Tensor workspace(size_t bytes, const Tensor& like) {
  if (bytes == 0) return Tensor();
  return torch::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(torch::kUInt8));
}
void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fp(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// LSH_F32, LSH_BF16, LSH_F16, or -1
int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return LSH_F32;
    case torch::kBFloat16: return LSH_BF16;
    case torch::kFloat16: return LSH_F16;
    default: return -1;
  }
}
void check_float(const Tensor& t, const char* name) {
  TORCH_CHECK(g_set, "lifscan ops: entry points not set");
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU (HIP) tensor");
  TORCH_CHECK_VALUE(code_of(t) >= 0, name, " must be float32, bfloat16 or float16");
}
bool grad_wanted(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// What looks at the calls from outside sees none of the kernels: a trace would record outputs that nothing fills,
// a forward-mode tangent would be lost, and the values behind a lazily negated view have the other sign.
template <class Tensors>
void check_plain(const char* what, const Tensors& ts) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be recorded by a trace (torch.jit.trace)");
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(!t._fw_grad(0).defined(), what, " has no forward-mode derivatives");
    TORCH_CHECK_VALUE(!t.is_neg(), what, ": an argument is a lazily negated view (pass its resolve_neg())");
  }
}
void check_plain(const char* what, std::initializer_list<Tensor> ts) {
  check_plain<std::initializer_list<Tensor>>(what, ts);
}
Tensor of(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
// autograd functions take no undefined tensors
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// The kernels' gradients have no graph of their own.  What arrives may be a lazily negated view.
variable_list first_order(variable_list grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "the language-model operators have no second derivatives (create_graph)");
  for (Tensor& t : grads)
    if (t.defined() && t.is_neg()) t = t.resolve_neg();
  check_plain("a language-model operator's gradient", grads);
  return grads;
}
// A saved tensor as the kernels read it: a saved-tensor hook may hand back another one than it was given.
Tensor unpacked(const Tensor& t, torch::IntArrayRef sizes, torch::ScalarType type, const Tensor& like) {
  TORCH_CHECK_VALUE(t.defined() && t.device() == like.device() && t.scalar_type() == type && t.sizes() == sizes,
                    "a saved tensor was unpacked to something else than the ", type, " ", sizes, " tensor on ",
                    like.device(), " that was saved");
  return t;
}

// Operands of a step, which updates the state in place: what shares memory with the state would be read by some
// workgroups while others write it, so it is copied first, as it was before the call.  By the ranges of their addresses:
// a state is contiguous, so what lies between a view's elements counts as the view's.
bool meets(const Tensor& t, const Tensor& state) {
  if (t.numel() == 0 || state.numel() == 0) return false;
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t last = 0;
  for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
  const uintptr_t a = (uintptr_t)t.data_ptr(), b = (uintptr_t)state.data_ptr();
  return a < b + state.nbytes() && b < a + (last + 1) * t.element_size();
}
Tensor apart(const Tensor& t, const Tensor& state) {
  return meets(t, state) ? t.clone(at::MemoryFormat::Contiguous) : t;
}

// ------------------------------------------------------------------------------- linear attention
// An operand whose last axis is contiguous.
Tensor rows_of(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

void check_operand(const Tensor& t, const char* name, int64_t dims, const Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == dims, name, " must be a ", dims, "-D [", dims == 4 ? "T, " : "", "B, heads, D] tensor");
  if (!like.defined()) {
    check_float(t, name);
    return;
  }
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == like.scalar_type(), name, " must be ",
                    like.scalar_type(), " on ", like.device());
  TORCH_CHECK_VALUE(t.size(0) == like.size(0) && (dims == 3 || t.size(1) == like.size(1)), name,
                    " must have the rows and batches of q");
}

struct Attn {
  Tensor q, k, v, beta;
  lsh_linattn a = {};
  std::vector<int64_t> state() const { return {a.B, a.H, a.Dk, a.Dv}; }
  void check_state(const Tensor& s, const char* name) const {
    TORCH_CHECK_VALUE(s.scalar_type() == torch::kFloat32 && s.device() == q.device() && s.sizes() == state(), name,
                      " must be float32 ", state(), " on ", q.device());
  }
};

Attn attn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& beta, double scale, int64_t dims) {
  check_operand(q, "q", dims, Tensor());
  check_operand(k, "k", dims, q);
  check_operand(v, "v", dims, q);
  const int64_t Dk = q.size(-1), Dv = v.size(-1);
  TORCH_CHECK_VALUE(k.size(-1) == Dk, "q and k must have the same width, got ", Dk, " and ", k.size(-1));
  TORCH_CHECK_VALUE(Dk >= 1 && Dv >= 1 && Dk <= LSH_LINATTN_MAX_D && Dv <= LSH_LINATTN_MAX_D, "widths ", Dk, " and ",
                    Dv, ": 1 to ", LSH_LINATTN_MAX_D, " are supported");
  TORCH_CHECK_VALUE(beta.dim() == 1 && beta.device() == q.device() && beta.is_floating_point(),
                    "beta must be a number or a [heads] tensor on ", q.device());
  const int64_t H = beta.size(0);
  TORCH_CHECK_VALUE(H >= 1, "beta has no decays");
  for (const Tensor& t : {q, k, v})
    TORCH_CHECK_VALUE(t.size(-2) >= 1 && H % t.size(-2) == 0, H, " decays: the heads of q, k and v (", q.size(-2), ", ",
                      k.size(-2), ", ", v.size(-2), ") must divide them");
  Attn r;
  r.q = rows_of(q), r.k = rows_of(k), r.v = rows_of(v);
  r.beta = beta.detach().to(torch::kFloat32).contiguous();
  lsh_linattn& a = r.a;
  a.dtype = code_of(q), a.Dk = (int)Dk, a.Dv = (int)Dv;
  a.q_heads = (int)q.size(-2), a.k_heads = (int)k.size(-2), a.v_heads = (int)v.size(-2);
  a.T = dims == 4 ? q.size(0) : 1, a.B = q.size(-3), a.H = H;
  a.q = r.q.data_ptr(), a.k = r.k.data_ptr(), a.v = r.v.data_ptr(), a.beta = fp(r.beta);
  a.q_sb = r.q.stride(-3), a.q_sh = r.q.stride(-2);
  a.k_sb = r.k.stride(-3), a.k_sh = r.k.stride(-2);
  a.v_sb = r.v.stride(-3), a.v_sh = r.v.stride(-2);
  if (dims == 4) a.q_st = r.q.stride(0), a.k_st = r.k.stride(0), a.v_st = r.v.stride(0);
  a.scale = (float)scale;
  return r;
}

struct AttnOut {
  Tensor o, s_end, ws;
};
AttnOut attn_forward(Attn& r, const Tensor& s0) {
  const c10::DeviceGuard guard(r.q.device());
  AttnOut out;
  out.o = torch::empty({r.a.T, r.a.B, r.a.H, r.a.Dv}, r.q.options());
  out.s_end = torch::empty(r.state(), r.beta.options());
  r.a.s0 = fp(s0), r.a.o = out.o.data_ptr(), r.a.s_end = fp(out.s_end);
  const size_t nb = g.lsh_linattn_workspace(&r.a);
  out.ws = workspace(nb, r.q);
  check(g.lsh_linattn_fwd(&r.a, raw(out.ws), nb, stream_of(r.q)), "lsh_linattn_fwd");
  return out;
}

struct LinAttn : public torch::autograd::Function<LinAttn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& beta, const Maybe& s0_in, double scale) {
    const Tensor s0 = of(s0_in);
    Attn r = attn(q, k, v, beta, scale, 4);
    const AttnOut out = attn_forward(r, s0);
    // ws: the states before the row segments
    ctx->save_for_backward({r.q, r.k, r.v, r.beta, s0, out.ws});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["s0"] = s0.defined();
    ctx->saved_data["ws"] = out.ws.defined() ? out.ws.numel() : (int64_t)0;
    ctx->saved_data["sizes"] = std::vector<int64_t>{r.a.T, r.a.B, r.a.H, r.a.Dk, r.a.Dv, r.a.q_heads, r.a.k_heads, r.a.v_heads};
    ctx->saved_data["ds0"] = s0.defined() && s0.requires_grad();
    ctx->set_materialize_grads(false);
    return {out.o, out.s_end};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    variable_list none(6);
    const Tensor &d_o = grads[0], &d_s = grads[1];
    if (!d_o.defined() && !d_s.defined()) return none;
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["sizes"].toIntVector();
    const Tensor& like = d_o.defined() ? d_o : d_s;
    const auto type = saved[0].scalar_type();
    TORCH_CHECK_VALUE(!d_o.defined() || type == d_o.scalar_type(), "a saved tensor was unpacked to another type");
    const Tensor q = unpacked(saved[0], {n[0], n[1], n[5], n[3]}, type, like),
                 k = unpacked(saved[1], {n[0], n[1], n[6], n[3]}, type, like),
                 v = unpacked(saved[2], {n[0], n[1], n[7], n[4]}, type, like),
                 beta = unpacked(saved[3], {n[2]}, torch::kFloat32, like);
    Attn r = attn(q, k, v, beta, ctx->saved_data["scale"].toDouble(), 4);
    const c10::DeviceGuard guard(r.q.device());
    Tensor s0, starts;
    if (ctx->saved_data["s0"].toBool()) {
      s0 = unpacked(saved[4], r.state(), torch::kFloat32, like).contiguous();
      r.a.s0 = fp(s0);
    }
    if (const int64_t bytes = ctx->saved_data["ws"].toInt())
      starts = unpacked(saved[5], {bytes}, torch::kUInt8, like).contiguous();
    Tensor go = d_o.defined() ? rows_of(d_o)
                              : torch::zeros({}, r.q.options()).expand({r.a.T, r.a.B, r.a.H, r.a.Dv}).contiguous();
    Tensor gs;
    if (d_s.defined()) {
      r.check_state(d_s, "the final state's gradient");
      gs = d_s.contiguous();
    }
    const Tensor dq = torch::empty(r.q.sizes(), r.q.options()), dk = torch::empty(r.k.sizes(), r.q.options()),
                 dv = torch::empty(r.v.sizes(), r.q.options());
    Tensor ds0;
    if (ctx->saved_data["ds0"].toBool()) ds0 = torch::empty(r.state(), r.beta.options());
    const size_t nb = g.lsh_linattn_bwd_workspace(&r.a);
    const Tensor ws = workspace(nb, r.q);
    check(g.lsh_linattn_bwd(&r.a, raw(starts), raw(go), go.stride(0), go.stride(1), go.stride(2), fp(gs), raw(dq),
                            raw(dk), raw(dv), fp(ds0), raw(ws), nb, stream_of(r.q)),
          "lsh_linattn_bwd");
    return {dq, dk, dv, Tensor(), ds0, Tensor()};
  }
};

std::tuple<Tensor, Tensor> lin_attn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& beta,
                                    const Maybe& s0_in, double scale) {
  Tensor s0 = of(s0_in);
  check_plain("lin_attn", {q, k, v, beta, s0});
  if (grad_wanted({q, k, v, beta, s0})) {
    TORCH_CHECK_VALUE(!beta.requires_grad(), "beta is a constant of lin_attn: it gets no gradient (pass beta.detach())");
    const Attn r = attn(q, k, v, beta, scale, 4);
    if (s0.defined()) {
      r.check_state(s0, "s0");
      s0 = s0.contiguous();
    }
    // what was laid out anew, with its gradient: once a call
    const auto out = LinAttn::apply(r.q, r.k, r.v, r.beta, maybe(s0), scale);
    return {out[0], out[1]};
  }
  Attn r = attn(q.detach(), k.detach(), v.detach(), beta, scale, 4);
  if (s0.defined()) {
    r.check_state(s0, "s0");
    s0 = s0.detach().contiguous();
  }
  const AttnOut out = attn_forward(r, s0);
  return {out.o, out.s_end};
}

Tensor lin_attn_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& beta, const Tensor& state,
                     double scale) {
  check_plain("lin_attn_step", {q, k, v, beta, state});
  TORCH_CHECK_VALUE(!grad_wanted({q, k, v, beta, state}),
                    "lin_attn_step has no gradients (q, k, v, beta or the state asks for one): call it under "
                    "torch.no_grad, or lin_attn");
  Attn r = attn(q, k, v, beta, scale, 3);
  r.check_state(state, "state");
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is updated in place");
  if (meets(r.q, state) || meets(r.k, state) || meets(r.v, state) || meets(r.beta, state))
    r = attn(apart(r.q, state), apart(r.k, state), apart(r.v, state), apart(r.beta, state), scale, 3);
  const c10::DeviceGuard guard(r.q.device());
  const Tensor o = torch::empty({r.a.B, r.a.H, r.a.Dv}, r.q.options());
  r.a.o = o.data_ptr();
  check(g.lsh_linattn_step(&r.a, fp(state), stream_of(r.q)), "lsh_linattn_step");
  // a graph that has saved the state from before is told, as by torch's own in-place operations
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return o;
}

// ------------------------------------------------------------------------------- norms of a block
Tensor channel(const Tensor& w, int64_t D, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(w.device() == like.device() && w.dim() == 1 && w.size(0) == D && code_of(w) >= 0, name,
                    " must be a float [", D, "] tensor on ", like.device());
  return w.to(torch::kFloat32).contiguous();  // differentiable
}

lsh_block_norm norm_args(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& w_post,
                         const Tensor& w_pre, const Tensor& scale, double scale1, double eps, int64_t act) {
  lsh_block_norm a = {};
  a.x_dtype = code_of(x), a.dtype = code_of(y), a.act = (int)act, a.D = (int)x.size(-1);
  a.rows = x.numel() / a.D;
  a.x = raw(x), a.y = raw(y), a.gate = raw(gate);
  a.w_post = fp(w_post), a.w_pre = fp(w_pre), a.scale = fp(scale);
  a.scale1 = (float)scale1, a.eps = (float)eps;
  return a;
}
variable_list norm_forward(const lsh_block_norm& a, const Tensor& x, const Tensor& y) {
  const c10::DeviceGuard guard(x.device());
  const Tensor x_new = torch::empty_like(x), z = torch::empty_like(y);
  check(g.lsh_block_norm_fwd(&a, raw(x_new), raw(z), stream_of(x)), "lsh_block_norm_fwd");
  return {x_new, z};
}

struct BlockNorm : public torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Maybe& gate_in,
                               const Tensor& w_post, const Tensor& w_pre, const Maybe& scale_in, double scale1,
                               double eps, int64_t act) {
    const Tensor gate = of(gate_in), scale = of(scale_in);
    // x_new is computed again in the backward: nothing is kept but the operands
    ctx->save_for_backward({x, y, gate, w_post, w_pre, scale});
    ctx->saved_data["c"] = std::vector<double>{scale1, eps};
    auto wants = [](const Tensor& t) -> int64_t { return t.defined() && t.requires_grad(); };
    ctx->saved_data["n"] = std::vector<int64_t>{wants(x), wants(y), wants(gate), wants(w_post), wants(w_pre),
                                                wants(scale), act, gate.defined(), scale.defined()};
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return norm_forward(norm_args(x, y, gate, w_post, w_pre, scale, scale1, eps, act), x, y);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(9);
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const auto c = ctx->saved_data["c"].toDoubleVector();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const Tensor& like = grads[0].defined() ? grads[0] : grads[1];
    const auto tx = grads[0].defined() ? grads[0].scalar_type() : saved[0].scalar_type();
    const auto ty = grads[1].defined() ? grads[1].scalar_type() : saved[1].scalar_type();
    TORCH_CHECK_VALUE(code_of(saved[0]) >= 0 && code_of(saved[1]) >= 0 &&
                          (tx == torch::kFloat32 || tx == ty), "a saved tensor was unpacked to another type");
    const int64_t D = sizes.back();
    const Tensor x = unpacked(saved[0], sizes, tx, like).contiguous(), y = unpacked(saved[1], sizes, ty, like).contiguous();
    const Tensor gate = n[7] ? unpacked(saved[2], sizes, ty, like).contiguous() : Tensor();
    const Tensor w_post = unpacked(saved[3], {D}, torch::kFloat32, like).contiguous(),
                 w_pre = unpacked(saved[4], {D}, torch::kFloat32, like).contiguous();
    const Tensor scale = n[8] ? unpacked(saved[5], {D}, torch::kFloat32, like).contiguous() : Tensor();
    const c10::DeviceGuard guard(x.device());
    const lsh_block_norm a = norm_args(x, y, gate, w_post, w_pre, scale, c[0], c[1], n[6]);
    const Tensor gx = grads[0].defined() ? grads[0].contiguous() : Tensor(),
                 gz = grads[1].defined() ? grads[1].contiguous() : Tensor();
    const Tensor dx = torch::empty_like(x), dy = torch::empty_like(y);
    const Tensor dgate = n[2] ? torch::empty_like(gate) : Tensor();
    const Tensor dpost = n[3] ? torch::empty_like(w_post) : Tensor(), dpre = n[4] ? torch::empty_like(w_pre) : Tensor();
    const Tensor dscale = n[5] ? torch::empty_like(scale) : Tensor();
    const size_t nb = g.lsh_block_norm_bwd_workspace(&a);
    const Tensor ws = workspace(nb, x);
    check(g.lsh_block_norm_bwd(&a, raw(gx), raw(gz), raw(dx), raw(dy), raw(dgate), fp(dpost), fp(dpre), fp(dscale),
                               raw(ws), nb, stream_of(x)),
          "lsh_block_norm_bwd");
    return {n[0] ? dx : Tensor(), n[1] ? dy : Tensor(), dgate, dpost, dpre, dscale, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> block_norm(const Tensor& x_in, const Tensor& y_in, const Tensor& w_post_in,
                                      const Tensor& w_pre_in, const Maybe& gate_in, const Maybe& scale_in,
                                      double scale1, double eps, int64_t act) {
  check_plain("block_norm", {x_in, y_in, w_post_in, w_pre_in, of(gate_in), of(scale_in)});
  check_float(x_in, "x");
  check_float(y_in, "y");
  TORCH_CHECK_VALUE(x_in.dim() >= 1 && x_in.sizes() == y_in.sizes() && x_in.device() == y_in.device(),
                    "x and y must have one shape and device, got ", x_in.sizes(), " and ", y_in.sizes());
  TORCH_CHECK_VALUE(x_in.scalar_type() == torch::kFloat32 || x_in.scalar_type() == y_in.scalar_type(),
                    "x must be float32 or ", y_in.scalar_type());
  const int64_t D = x_in.size(-1);
  TORCH_CHECK_VALUE(D >= 1 && D <= LSH_BLOCK_NORM_MAX_D, D, " channels: 1 to ", LSH_BLOCK_NORM_MAX_D, " are supported");
  Tensor gate = of(gate_in), scale = of(scale_in);
  if (gate.defined()) {
    TORCH_CHECK_VALUE(gate.sizes() == y_in.sizes() && gate.scalar_type() == y_in.scalar_type() &&
                          gate.device() == y_in.device(), "gate must be ", y_in.scalar_type(), " ", y_in.sizes(), " on ",
                      y_in.device());
    gate = gate.contiguous();
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps=", eps, " must not be negative");
  const Tensor w_post = channel(w_post_in, D, x_in, "w_post"), w_pre = channel(w_pre_in, D, x_in, "w_pre");
  if (scale.defined()) scale = channel(scale, D, x_in, "res_scale");
  const Tensor x = x_in.contiguous(), y = y_in.contiguous();
  if (!gate.defined()) act = LSH_GATE_NONE;
  const auto out = grad_wanted({x, y, gate, w_post, w_pre, scale})
                       ? BlockNorm::apply(x, y, maybe(gate), w_post, w_pre, maybe(scale), scale1, eps, act)
                       : norm_forward(norm_args(x, y, gate, w_post, w_pre, scale, scale1, eps, act), x, y);
  return {out[0], out[1]};
}

// ------------------------------------------------------------------------------- embedding
Tensor embed_forward(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  const c10::DeviceGuard guard(weight.device());
  auto sizes = tokens.sizes().vec();
  sizes.push_back(weight.size(1));
  const Tensor out = torch::empty(sizes, weight.options());
  check(g.lsh_embed_fwd(code_of(weight), tokens.data_ptr<int64_t>(), raw(weight), raw(out), tokens.numel(),
                        weight.size(0), weight.size(1), padding, (float)scale, stream_of(weight)),
        "lsh_embed_fwd");
  return out;
}

struct Embed : public torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& weight, double scale,
                        int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["n"] = std::vector<int64_t>{weight.size(0), weight.size(1), padding};
    ctx->saved_data["sizes"] = tokens.sizes().vec();
    return embed_forward(tokens, weight, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    const auto n = ctx->saved_data["n"].toIntVector();
    const Tensor dout = grads[0].contiguous();
    const Tensor tokens = unpacked(ctx->get_saved_variables()[0], ctx->saved_data["sizes"].toIntVector(),
                                   torch::kInt64, dout).contiguous();
    const c10::DeviceGuard guard(dout.device());
    const Tensor dw = torch::empty({n[0], n[1]}, dout.options());
    const size_t nb = g.lsh_embed_bwd_workspace(tokens.numel(), n[0]);
    const Tensor ws = workspace(nb, dout);
    check(g.lsh_embed_bwd(code_of(dout), tokens.data_ptr<int64_t>(), raw(dout), raw(dw), tokens.numel(), n[0], n[1],
                          n[2], (float)ctx->saved_data["scale"].toDouble(), raw(ws), nb, stream_of(dout)),
          "lsh_embed_bwd");
    return {Tensor(), dw, Tensor(), Tensor()};
  }
};

Tensor embed(const Tensor& tokens_in, const Tensor& weight_in, double scale, c10::optional<int64_t> padding_idx) {
  check_plain("embed", {weight_in});
  check_float(weight_in, "weight");
  TORCH_CHECK_VALUE(weight_in.dim() == 2 && weight_in.size(1) >= 1, "weight must be a [V, D] tensor");
  TORCH_CHECK_VALUE(tokens_in.device() == weight_in.device(), "tokens must be on ", weight_in.device());
  TORCH_CHECK_VALUE(tokens_in.scalar_type() == torch::kInt64 || tokens_in.scalar_type() == torch::kInt32,
                    "tokens must be int64 or int32");
  int64_t padding = -1;
  if (padding_idx.has_value()) {
    padding = *padding_idx;
    TORCH_CHECK_VALUE(padding >= 0 && padding < weight_in.size(0), "padding_idx=", padding,
                      " must be in the table of ", weight_in.size(0), " rows");
  }
  const Tensor tokens = tokens_in.to(torch::kInt64).contiguous(), weight = weight_in.contiguous();
  return grad_wanted({weight}) ? Embed::apply(tokens, weight, scale, padding)
                               : embed_forward(tokens, weight, scale, padding);
}

// ------------------------------------------------------------------------------- distillation
std::tuple<Tensor, Tensor> distill_forward(const Tensor& z, const Tensor& values, const Tensor& index, double tau) {
  const c10::DeviceGuard guard(z.device());
  const int64_t rows = z.size(0), V = z.size(1);
  const auto f32 = z.options().dtype(torch::kFloat32);
  const Tensor loss = torch::empty({rows}, f32), stats = torch::empty({4, rows}, f32);
  const size_t nb = g.lsh_distill_workspace(rows, V);
  const Tensor ws = workspace(nb, z);
  check(g.lsh_distill_fwd(code_of(z), raw(z), z.stride(0), code_of(values), raw(values), index.data_ptr<int64_t>(),
                          fp(loss), fp(stats), rows, V, (int)values.size(1), (float)tau, raw(ws), nb, stream_of(z)),
        "lsh_distill_fwd");
  return {loss, stats};
}

struct Distill : public torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& values, const Tensor& index, double tau) {
    const auto [loss, stats] = distill_forward(z, values, index, tau);
    ctx->save_for_backward({z, values, index, stats});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["n"] = std::vector<int64_t>{z.size(0), z.size(1), values.size(1), (int64_t)z.scalar_type(),
                                                (int64_t)values.scalar_type()};
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Tensor& gr = grads[0];
    Tensor z = unpacked(saved[0], {n[0], n[1]}, (torch::ScalarType)n[3], gr);
    if (z.stride(1) != 1 && n[1] > 1) z = z.contiguous();
    const Tensor values = unpacked(saved[1], {n[0], n[2]}, (torch::ScalarType)n[4], gr).contiguous(),
                 index = unpacked(saved[2], {n[0], n[2]}, torch::kInt64, gr).contiguous(),
                 stats = unpacked(saved[3], {4, n[0]}, torch::kFloat32, gr).contiguous();
    const c10::DeviceGuard guard(z.device());
    const Tensor dz = torch::empty({n[0], n[1]}, z.options());
    check(g.lsh_distill_bwd(code_of(z), raw(z), z.stride(0), code_of(values), raw(values), index.data_ptr<int64_t>(),
                            fp(stats), fp(gr), gr.stride(0), raw(dz), n[0], n[1], (int)n[2],
                            (float)ctx->saved_data["tau"].toDouble(), stream_of(z)),
          "lsh_distill_bwd");
    return {dz, Tensor(), Tensor(), Tensor()};
  }
};

Tensor distill_topk(const Tensor& logits, const Tensor& values_in, const Tensor& index_in, double tau) {
  check_plain("distill_topk", {logits, values_in});
  check_float(logits, "logits");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [*rows, V]");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(values_in.sizes() == index_in.sizes() && values_in.dim() == logits.dim() &&
                        values_in.sizes().slice(0, values_in.dim() - 1) == lead,
                    "top_values and top_index must be [*rows, K] with the rows of logits ", lead);
  TORCH_CHECK_VALUE(values_in.device() == logits.device() && index_in.device() == logits.device(),
                    "top_values and top_index must be on ", logits.device());
  const int64_t K = values_in.size(-1), V = logits.size(-1);
  TORCH_CHECK_VALUE(K <= LSH_DISTILL_MAX_K, K, " teacher logits a row: up to ", LSH_DISTILL_MAX_K, " are supported");
  TORCH_CHECK_VALUE(index_in.scalar_type() == torch::kInt64, "top_index must be int64");
  TORCH_CHECK_VALUE(values_in.is_floating_point(), "top_values must be of a float type");
  TORCH_CHECK_VALUE(tau > 0 && tau < std::numeric_limits<double>::infinity(), "temperature=", tau,
                    " must be positive and finite");
  const int64_t rows = logits.numel() / V;
  Tensor z = logits.dim() == 2 ? logits : logits.reshape({rows, V});  // a view costs the engine a node
  if (z.stride(1) != 1 && V > 1) z = z.contiguous();
  Tensor values = values_in.detach();
  if (values.scalar_type() != logits.scalar_type()) values = values.to(torch::kFloat32);
  values = values.reshape({rows, K}).contiguous();
  const Tensor index = index_in.reshape({rows, K}).contiguous();
  const Tensor loss = grad_wanted({z}) ? Distill::apply(z, values, index, tau)
                                       : std::get<0>(distill_forward(z, values, index, tau));
  return logits.dim() == 2 ? loss : loss.reshape(lead);
}

// ------------------------------------------------------------------------------- log probabilities of tokens
struct Scores {
  Tensor logp, entropy, stats, top_logp, top_index;
  variable_list outputs() const {
    if (!top_logp.defined()) return {logp, entropy};
    return {logp, entropy, top_logp, top_index};
  }
};
Scores score_forward(const Tensor& z, const Tensor& tokens, double tau, int64_t K, bool train) {
  const c10::DeviceGuard guard(z.device());
  const int64_t rows = z.size(0), V = z.size(1);
  const auto f32 = z.options().dtype(torch::kFloat32);
  Scores r;
  r.logp = torch::empty({rows}, f32), r.entropy = torch::empty({rows}, f32);
  if (train) r.stats = torch::empty({3, rows}, f32);
  if (K > 0) r.top_logp = torch::empty({rows, K}, f32), r.top_index = torch::empty({rows, K}, tokens.options());
  const size_t nb = g.lsh_score_workspace(rows, V, (int)K);
  const Tensor ws = workspace(nb, z);
  check(g.lsh_score_fwd(code_of(z), raw(z), z.stride(0), tokens.data_ptr<int64_t>(), fp(r.logp), fp(r.entropy),
                        fp(r.stats), fp(r.top_logp), K > 0 ? r.top_index.data_ptr<int64_t>() : nullptr, rows, V, (int)K,
                        (float)tau, raw(ws), nb, stream_of(z)),
        "lsh_score_fwd");
  return r;
}

struct Score : public torch::autograd::Function<Score> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& tokens, double tau, int64_t K) {
    const Scores r = score_forward(z, tokens, tau, K, true);
    ctx->save_for_backward({z, tokens, r.stats});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["n"] = std::vector<int64_t>{z.size(0), z.size(1), (int64_t)z.scalar_type()};
    if (K > 0) ctx->mark_non_differentiable({r.top_logp, r.top_index});
    ctx->set_materialize_grads(false);
    return r.outputs();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    const Tensor &gl = grads[0], &ge = grads[1];
    if (!gl.defined() && !ge.defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Tensor& like = gl.defined() ? gl : ge;
    Tensor z = unpacked(saved[0], {n[0], n[1]}, (torch::ScalarType)n[2], like);
    if (z.stride(1) != 1 && n[1] > 1) z = z.contiguous();
    const Tensor tokens = unpacked(saved[1], {n[0]}, torch::kInt64, like).contiguous(),
                 stats = unpacked(saved[2], {3, n[0]}, torch::kFloat32, like).contiguous();
    const c10::DeviceGuard guard(z.device());
    const Tensor dz = torch::empty({n[0], n[1]}, z.options());
    check(g.lsh_score_bwd(code_of(z), raw(z), z.stride(0), tokens.data_ptr<int64_t>(), fp(stats), fp(gl),
                          gl.defined() ? gl.stride(0) : 0, fp(ge), ge.defined() ? ge.stride(0) : 0, raw(dz), n[0], n[1],
                          (float)ctx->saved_data["tau"].toDouble(), stream_of(z)),
          "lsh_score_bwd");
    return {dz, Tensor(), Tensor(), Tensor()};
  }
};

variable_list token_logprobs(const Tensor& logits, const Tensor& tokens_in, double tau, int64_t K) {
  check_plain("token_logprobs", {logits});
  check_float(logits, "logits");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [*rows, V]");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(tokens_in.device() == logits.device() && tokens_in.sizes() == lead, "tokens must be ", lead, " on ",
                    logits.device(), ", one for each row of logits");
  TORCH_CHECK_VALUE(tokens_in.scalar_type() == torch::kInt64 || tokens_in.scalar_type() == torch::kInt32,
                    "tokens must be int64 or int32");
  TORCH_CHECK_VALUE(tau > 0 && tau < std::numeric_limits<double>::infinity(), "temperature=", tau,
                    " must be positive and finite");
  TORCH_CHECK_VALUE(K >= 0 && K <= LSH_SCORE_MAX_TOP && K <= V, "top=", K, ": 0 to ",
                    std::min<int64_t>(LSH_SCORE_MAX_TOP, V), " alternatives of ", V, " are supported");
  const int64_t rows = logits.numel() / V;
  Tensor z = logits.dim() == 2 ? logits : logits.reshape({rows, V});
  if (z.stride(1) != 1 && V > 1) z = z.contiguous();
  const Tensor tokens = tokens_in.to(torch::kInt64).reshape({rows}).contiguous();
  variable_list out =
      grad_wanted({z}) ? Score::apply(z, tokens, tau, K) : score_forward(z, tokens, tau, K, false).outputs();
  if (logits.dim() == 2) return out;
  auto wide = lead.vec();
  wide.push_back(K);
  for (size_t i = 0; i < out.size(); ++i) out[i] = out[i].reshape(i < 2 ? lead : torch::IntArrayRef(wide));
  return out;
}

// ------------------------------------------------------------------------------- gated linear recurrence
// A stride, 0 where it leads nowhere: the kernels ask that strides are whole pieces.
int64_t step_of(const Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

struct Gates {
  Tensor x, gate, starts;
  lsh_gated a = {};
  std::vector<int64_t> state() const { return {a.B, a.D}; }
  void check_state(const Tensor& s, const char* name) const {
    TORCH_CHECK_VALUE(s.scalar_type() == torch::kFloat32 && s.device() == x.device() && s.sizes() == state(), name,
                      " must be float32 ", state(), " on ", x.device());
  }
};
Gates gates(const Tensor& x, const Tensor& gate, const Tensor& starts, int64_t decay, bool mix, int64_t dims) {
  check_float(x, "x");
  TORCH_CHECK_VALUE(x.dim() == dims && x.size(-1) >= 1, "x must be a ", dims, "-D [", dims == 3 ? "T, " : "", "B, D] tensor");
  TORCH_CHECK_VALUE(gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type() && gate.device() == x.device(),
                    "gate must be ", x.scalar_type(), " ", x.sizes(), " on ", x.device());
  Gates r;
  r.x = rows_of(x), r.gate = rows_of(gate);
  lsh_gated& a = r.a;
  a.dtype = code_of(x), a.decay = (int)decay, a.mix = mix;
  a.T = dims == 3 ? x.size(0) : 1, a.B = x.size(-2), a.D = x.size(-1);
  a.x = raw(r.x), a.gate = raw(r.gate);
  a.x_sb = step_of(r.x, -2), a.g_sb = step_of(r.gate, -2);
  if (dims == 3) a.x_st = step_of(r.x, 0), a.g_st = step_of(r.gate, 0);
  if (starts.defined()) {
    TORCH_CHECK_VALUE((starts.scalar_type() == torch::kBool || starts.scalar_type() == torch::kUInt8) &&
                          starts.device() == x.device() && starts.dim() == 2 && starts.size(0) == a.T &&
                          starts.size(1) == a.B, "starts must be bool [", a.T, ", ", a.B, "] on ", x.device());
    r.starts = starts.contiguous();
    a.starts = static_cast<const uint8_t*>(r.starts.data_ptr());
  }
  return r;
}
struct GatedOut {
  Tensor h, h_end, saved;
};
GatedOut gated_forward(Gates& r, const Tensor& h0, bool train) {
  const c10::DeviceGuard guard(r.x.device());
  const auto f32 = r.x.options().dtype(torch::kFloat32);
  GatedOut out;
  out.h = torch::empty({r.a.T, r.a.B, r.a.D}, r.x.options());
  out.h_end = torch::empty(r.state(), f32);
  r.a.h0 = fp(h0);
  if (train) out.saved = torch::empty({g.lsh_gated_saved(&r.a)}, f32);
  const size_t nb = g.lsh_gated_workspace(&r.a);
  const Tensor ws = workspace(nb, r.x);
  check(g.lsh_gated_fwd(&r.a, raw(out.h), fp(out.h_end), fp(out.saved), raw(ws), nb, stream_of(r.x)), "lsh_gated_fwd");
  return out;
}

struct Gated : public torch::autograd::Function<Gated> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& h0_in,
                               const Maybe& starts_in, int64_t decay, bool mix) {
    const Tensor h0 = of(h0_in);
    Gates r = gates(x, gate, of(starts_in), decay, mix, 3);
    const GatedOut out = gated_forward(r, h0, true);
    ctx->save_for_backward({r.x, r.gate, r.starts, out.saved});
    ctx->saved_data["n"] = std::vector<int64_t>{r.a.T, r.a.B, r.a.D, decay, mix, r.starts.defined(),
                                                h0.defined() && h0.requires_grad(), out.saved.numel(),
                                                r.starts.defined() ? (int64_t)r.starts.scalar_type() : 0};
    ctx->set_materialize_grads(false);
    return {out.h, out.h_end};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    const Tensor& d_end = grads[1];
    if (!grads[0].defined() && !d_end.defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Tensor& like = grads[0].defined() ? grads[0] : d_end;
    const auto type = saved[0].scalar_type();
    TORCH_CHECK_VALUE(!grads[0].defined() || type == grads[0].scalar_type(), "a saved tensor was unpacked to another type");
    const Tensor x = unpacked(saved[0], {n[0], n[1], n[2]}, type, like),
                 gate = unpacked(saved[1], {n[0], n[1], n[2]}, type, like);
    const Tensor starts = n[5] ? unpacked(saved[2], {n[0], n[1]}, (torch::ScalarType)n[8], like) : Tensor();
    const Tensor states = unpacked(saved[3], {n[7]}, torch::kFloat32, like).contiguous();
    const Gates r = gates(x, gate, starts, n[3], n[4], 3);
    const c10::DeviceGuard guard(r.x.device());
    Tensor dh, gs, dh0;
    if (grads[0].defined()) dh = rows_of(grads[0]);
    if (d_end.defined()) {
      r.check_state(d_end, "the final state's gradient");
      gs = d_end.contiguous();
    }
    const Tensor dx = torch::empty(r.x.sizes(), r.x.options()), dgate = torch::empty(r.x.sizes(), r.x.options());
    if (n[6]) dh0 = torch::empty(r.state(), states.options());
    const size_t nb = g.lsh_gated_workspace(&r.a);
    const Tensor ws = workspace(nb, r.x);
    check(g.lsh_gated_bwd(&r.a, fp(states), raw(dh), dh.defined() ? step_of(dh, 0) : 0, dh.defined() ? step_of(dh, 1) : 0,
                          fp(gs), raw(dx), raw(dgate), fp(dh0), raw(ws), nb, stream_of(r.x)),
          "lsh_gated_bwd");
    return {dx, dgate, dh0, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gate, const Maybe& h0_in, const Maybe& starts_in,
                                      int64_t decay, bool mix) {
  Tensor h0 = of(h0_in);
  check_plain("gated_scan", {x, gate, h0});
  const bool train = grad_wanted({x, gate, h0});
  Gates r = train ? gates(x, gate, of(starts_in), decay, mix, 3)
                  : gates(x.detach(), gate.detach(), of(starts_in), decay, mix, 3);
  if (h0.defined()) {
    r.check_state(h0, "h0");
    h0 = train ? h0.contiguous() : h0.detach().contiguous();
  }
  if (train) {
    // what was laid out anew, with its gradient: once a call
    const auto out = Gated::apply(r.x, r.gate, maybe(h0), maybe(r.starts), decay, mix);
    return {out[0], out[1]};
  }
  const GatedOut out = gated_forward(r, h0, false);
  return {out.h, out.h_end};
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state, int64_t decay, bool mix) {
  check_plain("gated_scan_step", {x, gate, state});
  TORCH_CHECK_VALUE(!grad_wanted({x, gate, state}),
                    "gated_scan_step has no gradients (x, gate or the state asks for one): call it under torch.no_grad, "
                    "or gated_scan");
  Gates r = gates(x, gate, Tensor(), decay, mix, 2);
  r.check_state(state, "state");
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is updated in place");
  if (meets(r.x, state) || meets(r.gate, state))
    r = gates(apart(r.x, state), apart(r.gate, state), Tensor(), decay, mix, 2);
  const c10::DeviceGuard guard(r.x.device());
  const Tensor h = torch::empty({r.a.B, r.a.D}, r.x.options());
  check(g.lsh_gated_step(&r.a, fp(state), raw(h), stream_of(r.x)), "lsh_gated_step");
  // a graph that has saved the state from before is told, as by torch's own in-place operations
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return h;
}

// ------------------------------------------------------------------------------- norms and rotation of heads
struct Heads {
  Tensor q, k, positions, freq, wq, wk;
  lsh_rotate a = {};
};
// The sizes and what does not depend on q's and k's values.  lead: [T, B], or [B].
void heads_of(Heads& r, torch::IntArrayRef lead, int64_t H, int64_t HK, int64_t D, double eps, bool neighbours) {
  lsh_rotate& a = r.a;
  const bool one = lead.size() == 1;
  a.T = one ? 1 : lead[0], a.B = lead[one ? 0 : 1], a.H = H, a.HK = HK, a.D = (int)D;
  a.neighbours = neighbours, a.eps = (float)eps;
  if (r.freq.defined()) {
    a.rot = 2 * (int)r.freq.size(0), a.inv_freq = r.freq.data_ptr<double>();
    a.positions = r.positions.data_ptr<int64_t>();
    if (one)
      a.p_sb = r.positions.stride(0);
    else
      a.p_st = r.positions.stride(0), a.p_sb = r.positions.dim() == 2 ? r.positions.stride(1) : 0;
  }
  a.q_weight = fp(r.wq), a.k_weight = fp(r.wk);
}
void heads_data(Heads& r, const Tensor& q, const Tensor& k) {
  lsh_rotate& a = r.a;
  r.q = rows_of(q), r.k = rows_of(k);
  a.dtype = code_of(q), a.q = raw(r.q), a.k = raw(r.k);
  a.q_sb = step_of(r.q, -3), a.q_sh = step_of(r.q, -2), a.k_sb = step_of(r.k, -3), a.k_sh = step_of(r.k, -2);
  if (q.dim() == 4) a.q_st = step_of(r.q, 0), a.k_st = step_of(r.k, 0);
}
variable_list rotate_forward(const Heads& r) {
  const c10::DeviceGuard guard(r.q.device());
  const Tensor qo = torch::empty(r.q.sizes(), r.q.options()), ko = torch::empty(r.k.sizes(), r.k.options());
  check(g.lsh_rotate_fwd(&r.a, raw(qo), raw(ko), stream_of(r.q)), "lsh_rotate_fwd");
  return {qo, ko};
}

struct NormRotate : public torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Maybe& positions,
                               const Maybe& freq, const Maybe& wq, const Maybe& wk, double eps, bool neighbours) {
    Heads r;
    r.positions = of(positions), r.freq = of(freq), r.wq = of(wq), r.wk = of(wk);
    heads_data(r, q, k);
    heads_of(r, q.sizes().slice(0, q.dim() - 2), q.size(-2), k.size(-2), q.size(-1), eps, neighbours);
    const bool norm = r.wq.defined();
    // a rotation alone needs no operand to go back
    ctx->save_for_backward({norm ? r.q : Tensor(), norm ? r.k : Tensor(), r.positions, r.freq, r.wq, r.wk});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["q"] = q.sizes().vec();
    ctx->saved_data["k"] = k.sizes().vec();
    ctx->saved_data["p"] = r.positions.defined() ? r.positions.sizes().vec() : std::vector<int64_t>{};
    ctx->saved_data["n"] = std::vector<int64_t>{neighbours, norm, r.freq.defined(), r.freq.defined() ? r.freq.size(0) : 0,
                                                (int64_t)q.scalar_type(), norm && r.wq.requires_grad(),
                                                norm && r.wk.requires_grad()};
    ctx->set_materialize_grads(false);
    return rotate_forward(r);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads_in) {
    const variable_list grads = first_order(std::move(grads_in));
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(8);
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const auto qs = ctx->saved_data["q"].toIntVector(), ks = ctx->saved_data["k"].toIntVector();
    const Tensor& like = grads[0].defined() ? grads[0] : grads[1];
    const auto type = (torch::ScalarType)n[4];
    const int64_t D = qs.back();
    const auto lead = torch::IntArrayRef(qs).slice(0, qs.size() - 2);
    Heads r;
    if (n[2]) {
      r.positions = unpacked(saved[2], ctx->saved_data["p"].toIntVector(), torch::kInt64, like);
      r.freq = unpacked(saved[3], {n[3]}, torch::kFloat64, like).contiguous();
    }
    const c10::DeviceGuard guard(like.device());
    if (n[1]) {
      r.wq = unpacked(saved[4], {D}, torch::kFloat32, like).contiguous();
      r.wk = unpacked(saved[5], {D}, torch::kFloat32, like).contiguous();
      heads_data(r, unpacked(saved[0], qs, type, like), unpacked(saved[1], ks, type, like));
    }
    // heads whose outputs were not used leave no gradient
    heads_of(r, lead, grads[0].defined() ? qs[qs.size() - 2] : 0, grads[1].defined() ? ks[ks.size() - 2] : 0, D,
             ctx->saved_data["eps"].toDouble(), n[0]);
    r.a.dtype = code_of(like);
    Tensor gq, gk, dq, dk;
    int64_t st[6] = {};
    auto strides = [&](const Tensor& t, int64_t* to) {
      to[0] = t.dim() == 4 ? step_of(t, 0) : 0, to[1] = step_of(t, -3), to[2] = step_of(t, -2);
    };
    if (grads[0].defined()) {
      gq = rows_of(grads[0]), dq = torch::empty(qs, gq.options());
      strides(gq, st);
    }
    if (grads[1].defined()) {
      gk = rows_of(grads[1]), dk = torch::empty(ks, gk.options());
      strides(gk, st + 3);
    }
    Tensor dwq, dwk;
    if (n[5]) dwq = torch::empty({D}, r.wq.options());
    if (n[6]) dwk = torch::empty({D}, r.wk.options());
    const size_t nb = g.lsh_rotate_bwd_workspace(&r.a);
    const Tensor ws = workspace(nb, like);
    check(g.lsh_rotate_bwd(&r.a, raw(gq), st[0], st[1], st[2], raw(gk), st[3], st[4], st[5], raw(dq), raw(dk), fp(dwq),
                           fp(dwk), raw(ws), nb, stream_of(like)),
          "lsh_rotate_bwd");
    return {dq, dk, Tensor(), Tensor(), dwq, dwk, Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> norm_rotate(const Tensor& q, const Tensor& k, const Maybe& positions_in, const Maybe& freq_in,
                                       const Maybe& wq_in, const Maybe& wk_in, double eps, bool neighbours) {
  check_plain("norm_rotate", {q, k, of(freq_in), of(wq_in), of(wk_in)});
  check_float(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 4 || q.dim() == 3, "q must be a [T, B, heads, D] tensor, or [B, heads, D]");
  const auto lead = q.sizes().slice(0, q.dim() - 2);
  const int64_t D = q.size(-1);
  TORCH_CHECK_VALUE(k.dim() == q.dim() && k.sizes().slice(0, k.dim() - 2) == lead && k.size(-1) == D &&
                        k.scalar_type() == q.scalar_type() && k.device() == q.device(),
                    "k must be ", q.scalar_type(), " with the rows, batches and width of q on ", q.device(), ", got ",
                    k.sizes(), " for ", q.sizes());
  TORCH_CHECK_VALUE(D >= 2 && D % 2 == 0 && D <= LSH_ROTATE_MAX_D, "heads of ", D, ": even widths from 2 to ",
                    LSH_ROTATE_MAX_D, " are supported");
  TORCH_CHECK_VALUE(wq_in.has_value() == wk_in.has_value(), "q_weight and k_weight come together");
  TORCH_CHECK_VALUE(eps >= 0, "eps=", eps, " must not be negative");
  Heads r;
  TORCH_CHECK_VALUE(freq_in.has_value() == positions_in.has_value(), "positions and inv_freq come together: a rotation "
                    "needs both, and heads that are only normed neither");
  if (freq_in.has_value()) {
    const Tensor &f = *freq_in, &p = *positions_in;
    TORCH_CHECK_VALUE(f.dim() == 1 && f.device() == q.device() && f.is_floating_point() && f.size(0) <= D / 2,
                      "inv_freq must be a float tensor of up to ", D / 2, " frequencies on ", q.device());
    TORCH_CHECK_VALUE(!grad_wanted({f}), "inv_freq is a constant of norm_rotate: it gets no gradient (pass inv_freq.detach())");
    TORCH_CHECK_VALUE((p.scalar_type() == torch::kInt64 || p.scalar_type() == torch::kInt32) && p.device() == q.device(),
                      "positions must be int64 or int32 on ", q.device());
    TORCH_CHECK_VALUE(p.sizes() == lead || (lead.size() == 2 && p.dim() == 1 && p.size(0) == lead[0]),
                      "positions must be ", lead, lead.size() == 2 ? ", or one for each row" : "", ", got ", p.sizes());
    r.freq = f.detach().to(torch::kFloat64).contiguous();
    r.positions = p.to(torch::kInt64);
  }
  if (wq_in.has_value()) r.wq = channel(*wq_in, D, q, "q_weight"), r.wk = channel(*wk_in, D, q, "k_weight");
  if (grad_wanted({q, k, r.wq, r.wk})) {
    const auto out = NormRotate::apply(q, k, maybe(r.positions), maybe(r.freq), maybe(r.wq), maybe(r.wk), eps, neighbours);
    return {out[0], out[1]};
  }
  heads_data(r, q.detach(), k.detach());
  heads_of(r, lead, q.size(-2), k.size(-2), D, eps, neighbours);
  const auto out = rotate_forward(r);
  return {out[0], out[1]};
}

}  // namespace

void register_lm_ops(pybind11::module_& m) {
  m.def("set_lm_entry_points", &set_entry_points, "addresses of the C-ABI entry points, by name");
  m.def("lin_attn", &lin_attn, "linear attention over a sequence: o, state after the last row");
  m.def("lin_attn_step", &lin_attn_step, "linear attention of one token, the state updated in place: o");
  m.def("block_norm", &block_norm, "norm after a block, gate, residual scale, norm before the next: x_new, z");
  m.def("embed", &embed, "embedding lookup with scaling");
  m.def("distill_topk", &distill_topk, "loss against a teacher's top logits, by row");
  m.def("token_logprobs", &token_logprobs, "log probabilities of given tokens, entropy, top alternatives, by row");
  m.def("gated_scan", &gated_scan, "gated linear recurrence over a sequence: h, state after the last row");
  m.def("gated_scan_step", &gated_scan_step, "gated linear recurrence of one token, the state updated in place: h");
  m.def("norm_rotate", &norm_rotate, "norms of queries and keys for each head and their rotation by position: q, k");
}
