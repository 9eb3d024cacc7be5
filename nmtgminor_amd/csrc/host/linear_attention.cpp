// Linear attention with a decay for each head as an autograd node, its recurrent step, and the norms of queries and keys with their
// rotation as an autograd node.
#include "host.h"
#include <limits>

namespace nmtg_host {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

// [len, batch, heads, head_dim] with a contiguous head_dim, 16-byte aligned, strides the kernels take (linear attention's positions are
// less than 2^24 elements apart); anything else is copied
Tensor view_of(const Tensor& x, int64_t below = 1 << 24) {
  const bool ok = x.stride(3) == 1 && (x.size(0) == 1 || x.stride(0) < below) && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && x.stride(2) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}
Tensor norm_view(const Tensor& x) { return view_of(x, std::numeric_limits<int64_t>::max()); }
template <size_t N>
void put_strides(int64_t (&to)[N], std::initializer_list<const Tensor*> tensors) {
  size_t i = 0;
  for (const Tensor* t : tensors)
    for (int j = 0; j < 3; ++j) to[i++] = t->stride(j);
}
// integers as the kernels take them; what 32 bits do not hold goes to their ends
Tensor narrow32(const Tensor& t) {
  const auto limits = std::numeric_limits<int32_t>();
  return contiguous(t.scalar_type() == at::kLong ? t.clamp(limits.min(), limits.max()).to(at::kInt) : t);
}
bool integers(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
// 16-byte aligned and contiguous
Tensor dense(const Tensor& t) {
  const Tensor c = contiguous(t);
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
// an operand that may be left out, as a node takes it
optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(dense(t)) : std::nullopt; }
const int32_t* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

void check_half(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "expected a tensor in device memory (HIP); this op has no CPU path");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, ": fp16 or bf16 tensors required");
}
void no_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  if (!forward_mode()) return;
  for (const Tensor* t : tensors) TORCH_CHECK(!has_tangent(*t), what, ": jvp is not implemented");
}
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ----------------------------------------------------------------------------------------------- norms with rotation
struct NormArgs {
  Tensor cos, sin, positions;       // tables [rows, head_dim], positions undefined, [batch] or [len, batch]
  int64_t start = 0;
  double eps = 0;
};
int mode_of(const NormArgs& a) { return a.positions.defined() ? static_cast<int>(a.positions.dim()) : 0; }

std::pair<Tensor, Tensor> norm_fwd(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const NormArgs& a) {
  Launch on(q);
  Tensor qo = empty_like_sized(q, q.sizes()), ko = empty_like_sized(k, k.sizes());
  int64_t strides[12];
  put_strides(strides, {&q, &k, &qo, &ko});
  check(api.qk_norm_rotary_fwd(ptr(q), ptr(k), ptr(qo), ptr(ko), ptr(wq), ptr(wk), ptr(a.cos), ptr(a.sin), ints(a.positions), strides, a.start, a.cos.size(0),
                               q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), static_cast<float>(a.eps), mode_of(a), dtype_code(q),
                               wq.defined() ? dtype_code(wq) : dtype_code(q), dtype_code(a.cos), on.stream), "nmtg_qk_norm_rotary_fwd");
  return {qo, ko};
}

struct NormNode : Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const optional<Tensor>& q_weight, const optional<Tensor>& k_weight,
                               const NormArgs* a) {
    const Tensor wq = q_weight.value_or(Tensor()), wk = k_weight.value_or(Tensor());
    ctx->saved_data["start"] = a->start;
    ctx->saved_data["eps"] = a->eps;
    ctx->save_for_backward({q, k, wq, wk, a->cos, a->sin, a->positions});
    auto out = norm_fwd(q, k, wq, wk, *a);
    return {out.first, out.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3];
    NormArgs a{s[4], s[5], s[6], ctx->saved_data["start"].toInt(), ctx->saved_data["eps"].toDouble()};
    Launch on(q);
    const Tensor gq = norm_view(g[0]), gk = norm_view(g[1]);
    Tensor dq = empty_like_sized(q, q.sizes()), dk = empty_like_sized(k, k.sizes()), dwq, dwk;
    if (wq.defined()) {
      dwq = empty_like_sized(wq, wq.sizes());
      dwk = empty_like_sized(wk, wk.sizes());
    }
    int64_t strides[18];
    put_strides(strides, {&gq, &gk, &q, &k, &dq, &dk});
    const Scratch ws(q, std::max<int64_t>(api.qk_norm_rotary_bwd_workspace_bytes(q.size(0), q.size(1), q.size(2), k.size(2), q.size(3)), 16));
    check(api.qk_norm_rotary_bwd(ptr(gq), ptr(gk), ptr(q), ptr(k), ptr(dq), ptr(dk), ptr(wq), ptr(wk), ptr(dwq), ptr(dwk), ptr(a.cos), ptr(a.sin),
                                 ints(a.positions), strides, a.start, a.cos.size(0), q.size(0), q.size(1), q.size(2), k.size(2), q.size(3),
                                 static_cast<float>(a.eps), mode_of(a), dtype_code(q), wq.defined() ? dtype_code(wq) : dtype_code(q), dtype_code(a.cos),
                                 ws.get(), ws.bytes, on.stream), "nmtg_qk_norm_rotary_bwd");
    return {dq, dk, dwq, dwk, Tensor()};
  }
};

// [rows, head_dim] from the reference's [rows, 1, head_dim] or that itself
Tensor table_of(const Tensor& t, const Tensor& q) {
  check_device(t, q);
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), "qk_norm_rotary: the tables of positions have no gradient");
  no_tangents("qk_norm_rotary", {&t});
  TORCH_CHECK(t.dim() >= 2 && t.numel() == t.size(0) * q.size(3) && t.size(-1) == q.size(3), "qk_norm_rotary: tables must be [positions, head_dim] or [positions, 1, head_dim], got ",
              t.sizes());
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == q.scalar_type(), "qk_norm_rotary: tables must be fp32 or of the rows' type");
  return dense(t.view({t.size(0), q.size(3)}));
}

// ---------------------------------------------------------------------------------------------------- linear attention
struct LinearArgs {
  Tensor log_decay, lengths;
  double scale = 1;
};
struct LinearOut { Tensor out, state, segments; };      // segments: the states in front of them, for the backward

LinearOut linear_fwd_core(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& state, bool want_state, const Tensor& to, bool keep, const LinearArgs& a) {
  const int64_t t = q.size(0), b = q.size(1), h = q.size(2), d = q.size(3);
  Launch on(q);
  LinearOut r{empty_like_sized(q, q.sizes()), to.defined() ? to : want_state ? empty_as(q, {b, h, d, d}, at::kFloat) : Tensor(), Tensor()};
  int64_t strides[12];
  put_strides(strides, {&q, &k, &v, &r.out});
  const int64_t need = api.linear_attn_fwd_workspace_bytes(t, b, h, d);
  if (keep && need > 0) r.segments = empty_as(q, {need / 4}, at::kFloat);
  const Scratch ws = !keep && need > 0 ? Scratch(q, need) : Scratch();
  check(api.linear_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(r.out), floats(a.log_decay), ints(a.lengths), floats(state), floats(r.state), strides, t, b, h, d,
                            static_cast<float>(a.scale), dtype_code(q), r.segments.defined() ? ptr(r.segments) : ws.get(), need, on.stream), "nmtg_linear_attn_fwd");
  return r;
}

struct LinearNode : Function<LinearNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& given, bool want_state,
                               const LinearArgs* a) {
    const Tensor state = given.value_or(Tensor());
    LinearOut r = linear_fwd_core(q, k, v, state, want_state, Tensor(), true, *a);
    ctx->saved_data["scale"] = a->scale;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, state, a->log_decay, a->lengths, r.segments});
    return want_state ? variable_list{r.out, r.state} : variable_list{r.out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &state = s[3], &log_decay = s[4], &lengths = s[5];
    const int64_t t = q.size(0), b = q.size(1), h = q.size(2), d = q.size(3);
    Launch on(q);
    const Tensor dout = g[0].defined() ? view_of(g[0]) : at::zeros(q.sizes(), q.options().requires_grad(false));
    const Tensor dlast = g.size() > 1 && g[1].defined() ? dense(g[1]) : Tensor();
    Tensor dq = empty_like_sized(q, q.sizes()), dk = empty_like_sized(q, q.sizes()), dv = empty_like_sized(q, q.sizes());
    Tensor dfirst = state.defined() && ctx->needs_input_grad(3) ? empty_like_sized(state, state.sizes()) : Tensor();
    int64_t strides[21];
    put_strides(strides, {&dout, &q, &k, &v, &dq, &dk, &dv});
    const int64_t need = api.linear_attn_bwd_workspace_bytes(t, b, h, d);
    const Scratch ws = need > 0 ? Scratch(q, need) : Scratch();
    check(api.linear_attn_bwd(ptr(dout), ptr(q), ptr(k), ptr(v), ptr(dq), ptr(dk), ptr(dv), floats(log_decay), ints(lengths), floats(state), floats(s[6]), floats(dlast),
                              floats(dfirst), strides, t, b, h, d, static_cast<float>(ctx->saved_data["scale"].toDouble()), dtype_code(q), ws.get(), need, on.stream),
          "nmtg_linear_attn_bwd");
    return {dq, dk, dv, dfirst, Tensor(), Tensor()};
  }
};

void check_rows(const char* what, const Tensor& q, const Tensor& k, const Tensor& v) {
  for (const Tensor* t : {&q, &k, &v}) {
    check_half(*t, what);
    check_device(*t, q);
    TORCH_CHECK(t->dim() == 4 && t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type(), what, ": q, k and v must be [T, B, H, D] of one dtype");
  }
}
LinearArgs linear_args(const char* what, const Tensor& q, const Tensor& log_decay, optional<double> scale, const optional<Tensor>& lengths) {
  check_device(log_decay, q);
  TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == q.size(2) && log_decay.scalar_type() == at::kFloat, what, ": log_decay must be fp32 [heads]");
  TORCH_CHECK(!(at::GradMode::is_enabled() && log_decay.requires_grad()), what, ": the decays have no gradient");
  no_tangents(what, {&log_decay});
  LinearArgs a{contiguous(log_decay), Tensor(), scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3)))};
  if (lengths.has_value() && lengths->defined()) {
    check_device(*lengths, q);
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == q.size(1) && integers(*lengths), what, ": lengths must be integers [batch]");
    a.lengths = narrow32(*lengths);
  }
  return a;
}
void check_state(const char* what, const Tensor& s, const Tensor& q) {
  check_device(s, q);
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 4 && s.size(0) == q.size(1) && s.size(1) == q.size(2) && s.size(2) == q.size(3) && s.size(3) == q.size(3), what,
              ": a state must be fp32 [", q.size(1), ", ", q.size(2), ", ", q.size(3), ", ", q.size(3), "]");
}
// one that is written where it is
void check_state_in_place(const char* what, const Tensor& s, const Tensor& q) {
  check_state(what, s, q);
  TORCH_CHECK(s.is_contiguous() && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0, what, ": states must be contiguous and 16-byte aligned");
}
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void define_linear_attention(pybind11::module_& m) {
  m.def("qk_norm_rotary", [](const Tensor& q, const Tensor& k, const optional<Tensor>& q_weight, const optional<Tensor>& k_weight, const Tensor& cos, const Tensor& sin,
                             const optional<Tensor>& positions, int64_t start, double eps) {
    const char* what = "qk_norm_rotary";
    for (const Tensor* t : {&q, &k}) {
      check_half(*t, what);
      check_device(*t, q);
      TORCH_CHECK(t->dim() == 4 && t->scalar_type() == q.scalar_type(), what, ": q [T, B, H, D] and k [T, B, H_kv, D] of one dtype");
    }
    TORCH_CHECK(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3), what, ": k must have q's positions, batch and head dimension");
    const Tensor wq = q_weight.value_or(Tensor()), wk = k_weight.value_or(Tensor());
    TORCH_CHECK(wq.defined() == wk.defined(), what, ": weights for both queries and keys, or for neither");
    if (wq.defined()) {
      for (const Tensor* w : {&wq, &wk}) {
        check_device(*w, q);
        TORCH_CHECK(w->dim() == 1 && w->size(0) == q.size(3) && w->scalar_type() == wq.scalar_type() && (w->scalar_type() == at::kFloat || w->scalar_type() == q.scalar_type()),
                    what, ": weights must be [head_dim], fp32 or of the rows' type, both alike");
      }
    }
    NormArgs a{table_of(cos, q), table_of(sin, q), Tensor(), start, eps};
    TORCH_CHECK(a.cos.size(0) == a.sin.size(0) && a.cos.scalar_type() == a.sin.scalar_type(), what, ": the tables must be alike");
    if (positions.has_value() && positions->defined()) {
      const Tensor& p = *positions;
      check_device(p, q);
      TORCH_CHECK(integers(p) && ((p.dim() == 1 && p.size(0) == q.size(1)) || (p.dim() == 2 && p.size(0) == q.size(0) && p.size(1) == q.size(1))), what,
                  ": positions must be integers [B] (of every sequence's first row) or [T, B]");
      TORCH_CHECK(a.cos.size(0) > 0, what, ": the tables are empty");
      a.positions = narrow32(p);
    }
    if (!wants_grad({&q, &k, &wq, &wk})) {
      no_tangents(what, {&q, &k, &wq, &wk});
      auto out = norm_fwd(norm_view(q), norm_view(k), wq.defined() ? dense(wq) : wq, wk.defined() ? dense(wk) : wk, a);
      return std::make_tuple(out.first, out.second);
    }
    const variable_list out = NormNode::apply(norm_view(q), norm_view(k), some(wq), some(wk), &a);
    return std::make_tuple(out[0], out[1]);
  });
  m.def("linear_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, optional<double> scale, const optional<Tensor>& lengths,
                               const optional<Tensor>& state, bool return_state, const optional<Tensor>& state_out) {
    const char* what = "linear attention";
    check_rows(what, q, k, v);
    const LinearArgs a = linear_args(what, q, log_decay, scale, lengths);
    const Tensor s = state.value_or(Tensor());
    if (s.defined()) check_state(what, s, q);
    const Tensor to = state_out.value_or(Tensor());
    if (to.defined()) {
      check_state_in_place(what, to, q);
      TORCH_CHECK(!wants_grad({&q, &k, &v, &s, &to}), what, " with state_out has no gradient: call it under torch.no_grad() or on detached tensors");
      no_tangents(what, {&to});
    }
    if (!wants_grad({&q, &k, &v, &s})) {
      no_tangents(what, {&q, &k, &v, &s});
      LinearOut r = linear_fwd_core(view_of(q), view_of(k), view_of(v), s.defined() ? dense(s) : s, return_state, to, false, a);
      if (to.defined()) written(to);
      return std::make_tuple(r.out, optional<Tensor>(return_state ? optional<Tensor>(r.state) : std::nullopt));
    }
    const variable_list r = LinearNode::apply(view_of(q), view_of(k), view_of(v), some(s), return_state, &a);
    return std::make_tuple(r[0], optional<Tensor>(return_state ? optional<Tensor>(r[1]) : std::nullopt));
  });
  m.def("linear_attention_step", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const optional<Tensor>& state_out,
                                    optional<double> scale, const optional<Tensor>& lengths) {
    const char* what = "linear_attn_step";
    check_rows(what, q, k, v);
    const LinearArgs a = linear_args(what, q, log_decay, scale, lengths);
    const Tensor& to = state_out.has_value() && state_out->defined() ? *state_out : state;
    for (const Tensor* s : {&state, &to}) check_state_in_place(what, *s, q);
    TORCH_CHECK(!wants_grad({&q, &k, &v, &state, &to}), what, " has no gradient: call it under torch.no_grad() or on detached tensors");
    no_tangents(what, {&q, &k, &v, &state, &to});
    Launch on(q);
    const Tensor qq = view_of(q), kk = view_of(k), vv = view_of(v);
    Tensor out = empty_like_sized(q, q.sizes());
    int64_t strides[12];
    put_strides(strides, {&qq, &kk, &vv, &out});
    check(api.linear_attn_step(ptr(qq), ptr(kk), ptr(vv), ptr(out), floats(a.log_decay), ints(a.lengths), floats(state), floats(to), strides, q.size(0), q.size(1),
                               q.size(2), q.size(3), static_cast<float>(a.scale), dtype_code(q), on.stream), "nmtg_linear_attn_step");
    written(to);
    return out;
  });
}

}  // namespace nmtg_host
