// The operators of long-context decoders: attention with a sliding window and sinks as an autograd node, on three tensors or on the
// heads of one projection, and the rows of the quantised key / value cache written, read back and attended to.
#include "host.h"
#include <limits>

namespace nmtg_host {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

struct Window {
  int64_t window, sinks;
  double scale;
  Tensor lengths;
  bool gradient = false;          // whether the backward will be run
};

// [len, batch, heads, head_dim] with a contiguous head_dim, 16-byte aligned, strides the kernels take (of a single position's there is
// none); anything else is copied
Tensor view_of(const Tensor& x) {
  const bool ok = x.stride(3) == 1 && (x.size(0) == 1 || x.stride(0) < (1 << 24)) && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && x.stride(2) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}
void put_strides(int64_t* to, const Tensor& x) {
  for (int i = 0; i < 3; ++i) to[i] = x.stride(i);
}
// positions as the kernels take them; what 32 bits do not hold stays outside of every sequence and cache
Tensor narrow32(const Tensor& t) {
  const auto limits = std::numeric_limits<int32_t>();
  return contiguous(t.scalar_type() == at::kLong ? t.clamp(limits.min(), limits.max()).to(at::kInt) : t);
}
const int32_t* lengths_of(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

struct Forward { Tensor out, rest, lse; };
Forward window_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Window& w) {
  const int64_t t = q.size(0), b = q.size(1), h = q.size(2), d = q.size(3);
  Launch on(q);
  Forward r{empty_like_sized(q, {t, b, h, d}), w.gradient ? empty_as(q, {b, h, (t + 31) / 32 * 32, d}, at::kByte) : Tensor(), empty_as(q, {b, h, t}, at::kFloat)};
  int64_t strides[12];
  const Tensor* tensors[4] = {&q, &k, &v, &r.out};
  for (int i = 0; i < 4; ++i) put_strides(strides + 3 * i, *tensors[i]);
  check(api.window_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(r.out), w.gradient ? r.rest.data_ptr<uint8_t>() : nullptr, r.lse.data_ptr<float>(), lengths_of(w.lengths), strides, t, b, h, k.size(2), d,
                            w.window, w.sinks, static_cast<float>(w.scale), dtype_code(q), on.stream), "nmtg_window_attn_fwd");
  return r;
}
void window_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Forward& f, const Tensor& dq, const Tensor& dk,
                const Tensor& dv, const Window& w) {
  const int64_t t = q.size(0), b = q.size(1), h = q.size(2), d = q.size(3), hk = k.size(2);
  if (q.numel() == 0) return;
  Launch on(q);
  int64_t strides[24];
  const Tensor* tensors[8] = {&dout, &q, &k, &v, &f.out, &dq, &dk, &dv};
  for (int i = 0; i < 8; ++i) put_strides(strides + 3 * i, *tensors[i]);
  const Scratch ws(q, std::max<int64_t>(api.window_attn_bwd_workspace_bytes(t, b, h, hk, d, w.window, w.sinks), 16));
  check(api.window_attn_bwd(ptr(dout), ptr(q), ptr(k), ptr(v), ptr(f.out), f.rest.data_ptr<uint8_t>(), f.lse.data_ptr<float>(), ptr(dq), ptr(dk), ptr(dv),
                            lengths_of(w.lengths), strides, t, b, h, hk, d, w.window, w.sinks, static_cast<float>(w.scale), dtype_code(q), ws.get(),
                            ws.bytes, on.stream), "nmtg_window_attn_bwd");
}

void keep(AutogradContext* ctx, const Window& w) {
  ctx->saved_data["w"] = w.window;
  ctx->saved_data["n"] = w.sinks;
  ctx->saved_data["s"] = w.scale;
}
Window kept(AutogradContext* ctx, const Tensor& lengths) {
  return {ctx->saved_data["w"].toInt(), ctx->saved_data["n"].toInt(), ctx->saved_data["s"].toDouble(), lengths, true};
}

struct WindowNode : Function<WindowNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Window* w) {
    Forward r = window_fwd(q, k, v, *w);
    keep(ctx, *w);
    ctx->save_for_backward({q, k, v, r.out, r.rest, r.lse, w->lengths});
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2];
    Tensor dq = empty_like_sized(q, q.sizes()), dk = empty_like_sized(k, k.sizes()), dv = empty_like_sized(v, v.sizes());
    window_bwd(view_of(g[0]), q, k, v, {s[3], s[4], s[5]}, dq, dk, dv, kept(ctx, s[6]));
    return {dq, dk, dv, Tensor()};
  }
};

// lin [len, batch, (heads + 2 kv_heads) * head_dim]: queries, keys, values; their gradients go into one tensor of its shape
struct Slots { Tensor q, k, v; };
Slots slots_of(const Tensor& lin, int64_t heads, int64_t kv_heads) {
  const int64_t d = lin.size(2) / (heads + 2 * kv_heads);
  auto part = [&](int64_t from, int64_t n) {
    return lin.as_strided({lin.size(0), lin.size(1), n, d}, {lin.stride(0), lin.stride(1), d, 1}, lin.storage_offset() + from * d);
  };
  return {part(0, heads), part(heads, kv_heads), part(heads + kv_heads, kv_heads)};
}
struct WindowProjectionNode : Function<WindowProjectionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& lin, int64_t heads, int64_t kv_heads, const Window* w) {
    Slots s = slots_of(lin, heads, kv_heads);
    Forward r = window_fwd(s.q, s.k, s.v, *w);
    keep(ctx, *w);
    ctx->saved_data["h"] = heads;
    ctx->saved_data["k"] = kv_heads;
    ctx->save_for_backward({lin, r.out, r.rest, r.lse, w->lengths});
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const int64_t heads = ctx->saved_data["h"].toInt(), kv_heads = ctx->saved_data["k"].toInt();
    Tensor dlin = empty_like_sized(s[0], s[0].sizes());
    const Slots x = slots_of(s[0], heads, kv_heads), d = slots_of(dlin, heads, kv_heads);
    window_bwd(view_of(g[0]), x.q, x.k, x.v, {s[1], s[2], s[3]}, d.q, d.k, d.v, kept(ctx, s[4]));
    return {dlin, Tensor(), Tensor(), Tensor()};
  }
};

Window window_args(const Tensor& q, int64_t batch, int64_t head_dim, int64_t window, int64_t sinks, optional<double> scale, const optional<Tensor>& lengths) {
  TORCH_CHECK(window >= 1, "window attention: a window of ", window, " positions (at least 1)");
  TORCH_CHECK(sinks >= 0, "window attention: ", sinks, " sinks");
  Window w{window, sinks, scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(head_dim)), Tensor(), false};
  if (lengths.has_value() && lengths->defined()) {
    check_device(*lengths, q);
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == batch, "window attention: lengths must be [batch]");
    TORCH_CHECK(lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong, "window attention: lengths must be integers");
    w.lengths = narrow32(*lengths);
  }
  return w;
}
void check_half(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "expected a tensor in device memory (HIP); this op has no CPU path");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, ": fp16 or bf16 tensors required");
}

// ------------------------------------------------------------------------------------------------------ quantised cache
struct Cache {
  int64_t batch, kv_heads, capacity, dim;
  int bits;
  uint8_t *kc, *ks, *vc, *vs;
};
Cache cache_of(const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs) {
  for (const Tensor* t : {&kc, &ks, &vc, &vs}) {
    TORCH_CHECK(t->is_cuda(), "expected a tensor in device memory (HIP); this op has no CPU path");
    check_device(*t, kc);
    TORCH_CHECK(t->scalar_type() == at::kByte && t->dim() == 4 && t->is_contiguous(), "kv cache: codes and scales must be contiguous uint8 [batch, kv_heads, capacity, bytes]");
  }
  TORCH_CHECK(vc.sizes() == kc.sizes() && vs.sizes() == ks.sizes() && ks.sizes().slice(0, 3) == kc.sizes().slice(0, 3),
              "kv cache: codes and scales of keys and values must share batch, heads and capacity");
  const int64_t dim = 32 * ks.size(3);
  TORCH_CHECK(dim > 0 && (kc.size(3) == dim / 2 || kc.size(3) == dim), "kv cache: ", kc.size(3), " code bytes and ", ks.size(3),
              " scales per row are neither 4 nor 8 bits per element");
  return {kc.size(0), kc.size(1), kc.size(2), dim, kc.size(3) == dim ? 8 : 4, kc.data_ptr<uint8_t>(), ks.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(),
          vs.data_ptr<uint8_t>()};
}
Tensor int32_of(const Tensor& t, const Tensor& operand, int64_t batch, const char* what) {
  check_device(t, operand);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == batch && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong), "kv cache: ", what,
              " must be integers [batch]");
  return narrow32(t);
}
void no_gradient(const Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, " has no gradient: call it under torch.no_grad() or on detached tensors");
  TORCH_CHECK(!(forward_mode() && has_tangent(t)), what, ": jvp is not implemented");
}

}  // namespace

void define_long_context(pybind11::module_& m) {
  m.def("window_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, optional<double> scale,
                               const optional<Tensor>& lengths) {
    for (const Tensor* t : {&q, &k, &v}) {
      check_half(*t, "window attention");
      check_device(*t, q);
      TORCH_CHECK(t->dim() == 4 && t->scalar_type() == q.scalar_type(), "window attention: q [T, B, H, D], k and v [T, B, H_kv, D] of one dtype");
    }
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3),
                "window attention: k and v must have q's positions, batch and head dimension");
    TORCH_CHECK(k.size(2) > 0 && q.size(2) % k.size(2) == 0, "window attention: ", q.size(2), " query heads do not share ", k.size(2),
                " key / value heads evenly");
    Window w = window_args(q, q.size(1), q.size(3), window, sinks, scale, lengths);
    if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      TORCH_CHECK(!forward_mode() || !(has_tangent(q) || has_tangent(k) || has_tangent(v)), "window attention: jvp is not implemented");
      return window_fwd(view_of(q), view_of(k), view_of(v), w).out;
    }
    w.gradient = true;
    return WindowNode::apply(view_of(q), view_of(k), view_of(v), &w);
  });
  m.def("window_attention_projection", [](const Tensor& lin, int64_t heads, int64_t kv_heads, int64_t window, int64_t sinks, optional<double> scale,
                                          const optional<Tensor>& lengths) {
    check_half(lin, "window attention");
    TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && lin.dim() == 3 && lin.size(2) % (8 * (heads + 2 * kv_heads)) == 0,
                "window attention: a projection [T, B, (H + 2 H_kv) D] whose heads share key / value heads evenly");
    Window w = window_args(lin, lin.size(1), lin.size(2) / (heads + 2 * kv_heads), window, sinks, scale, lengths);
    w.gradient = at::GradMode::is_enabled() && lin.requires_grad();
    return WindowProjectionNode::apply(contiguous(lin), heads, kv_heads, &w);
  });
  m.def("kv_cache_write", [](const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& k, const Tensor& v, const optional<Tensor>& starts,
                             int64_t start) {
    const Cache c = cache_of(kc, ks, vc, vs);
    for (const Tensor* t : {&k, &v}) {
      check_half(*t, "kv cache");
      check_device(*t, kc);
      no_gradient(*t, "kv_cache_write");
      TORCH_CHECK(t->dim() == 4 && t->sizes() == k.sizes() && t->scalar_type() == k.scalar_type() && t->size(1) == c.batch && t->size(2) == c.kv_heads &&
                  t->size(3) == c.dim, "kv cache: k and v must be [count, ", c.batch, ", ", c.kv_heads, ", ", c.dim, "] of one dtype");
    }
    Launch on(kc);
    const Tensor kk = view_of(k), vv = view_of(v), at = starts.has_value() ? int32_of(*starts, kc, c.batch, "start") : Tensor();
    check(api.kv_cache_write(ptr(kk), kk.stride(0), kk.stride(1), kk.stride(2), ptr(vv), vv.stride(0), vv.stride(1), vv.stride(2), c.kc, c.ks, c.vc,
                             c.vs, lengths_of(at), start, k.size(0), c.batch, c.kv_heads, c.dim, c.capacity, c.bits, dtype_code(k), on.stream),
          "nmtg_kv_cache_write");
  });
  m.def("kv_cache_read", [](const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const optional<Tensor>& starts, int64_t start, int64_t count,
                            py::object dtype) {
    const Cache c = cache_of(kc, ks, vc, vs);
    const at::ScalarType type = torch::python::detail::py_object_to_dtype(dtype);
    TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, "kv cache: fp16 or bf16 tensors required");
    TORCH_CHECK(count >= 0, "kv cache: ", count, " rows");
    Launch on(kc);
    const Tensor at = starts.has_value() ? int32_of(*starts, kc, c.batch, "start") : Tensor();
    Tensor k = empty_as(kc, {count, c.batch, c.kv_heads, c.dim}, type), v = empty_as(kc, {count, c.batch, c.kv_heads, c.dim}, type);
    check(api.kv_cache_read(c.kc, c.ks, c.vc, c.vs, ptr(k), ptr(v), lengths_of(at), start, count, c.batch, c.kv_heads, c.dim, c.capacity, c.bits,
                            dtype_code(k), on.stream), "nmtg_kv_cache_read");
    return std::make_tuple(k, v);
  });
  m.def("kv_cache_attend", [](const Tensor& q, const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& lengths, int64_t longest,
                              int64_t window, int64_t sinks, optional<double> scale) {
    const Cache c = cache_of(kc, ks, vc, vs);
    check_half(q, "kv cache");
    check_device(q, kc);
    no_gradient(q, "kv_cache_attend");
    TORCH_CHECK(q.dim() == 4 && q.size(1) == c.batch && q.size(3) == c.dim && c.kv_heads > 0 && q.size(2) % c.kv_heads == 0 && q.size(2) > 0,
                "kv cache: queries must be [tq, ", c.batch, ", heads, ", c.dim, "] with heads that share ", c.kv_heads, " key / value heads evenly");
    Launch on(q);
    const Tensor x = view_of(q), n = int32_of(lengths, kc, c.batch, "lengths");
    const int64_t tq = q.size(0), h = q.size(2);
    Tensor out = empty_like_sized(q, {tq, c.batch, h, c.dim});
    const int64_t need = api.kv_cache_attn_workspace_bytes(tq, c.batch, h, c.kv_heads, c.dim, longest, window, sinks);
    const Scratch ws = need > 0 ? Scratch(q, need) : Scratch();
    check(api.kv_cache_attn(ptr(x), x.stride(0), x.stride(1), x.stride(2), c.kc, c.ks, c.vc, c.vs, lengths_of(n), ptr(out), out.stride(0),
                            out.stride(1), out.stride(2), tq, c.batch, h, c.kv_heads, c.dim, c.capacity, longest, window, sinks,
                            static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(c.dim))), c.bits, dtype_code(q), ws.get(),
                            need, on.stream), "nmtg_kv_cache_attn");
    return out;
  });
}

}  // namespace nmtg_host
