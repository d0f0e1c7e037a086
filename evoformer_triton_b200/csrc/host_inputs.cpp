// The autograd boundary of the operators before the attention (layer norm, relative position bias, pair-bias
// projection), in native code for the same reason as the attention's: small calls are bound by the host.
// A call reads sizes and strides, allocates its results and goes to the C ABI (evoattn.h); one that needs
// no gradient leaves out the autograd node.
#include "host_common.h"

#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <ATen/cuda/CUDAContext.h>

namespace evohost {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] void type_error(const std::string& text) { raise(PyExc_TypeError, text.c_str()); }
[[noreturn]] void value_error(const std::string& text) { raise(PyExc_ValueError, text.c_str()); }
[[noreturn]] void runtime_error(const std::string& text) { raise(PyExc_RuntimeError, text.c_str()); }

void check_main(const Tensor& t, const char* op, const char* name) {
  // A tracer would record the allocation of the result, not the call.
  if (torch::jit::tracer::isTracing()) runtime_error(std::string(op) + " cannot be traced");
  if (!t.is_cuda()) runtime_error(std::string(op) + " runs on CUDA tensors only; there is no CPU fallback");
  if (!known(t.scalar_type())) type_error(std::string(name) + " must be bfloat16, float16 or float32");
}
// A small dense tensor of weights beside t, of any of the three types.
void check_weight(const Tensor& w, const Tensor& t, const char* name, at::IntArrayRef shape) {
  if (w.device() != t.device()) runtime_error(std::string(name) + " is on " + w.device().str() + ", not on " + t.device().str());
  if (!known(w.scalar_type())) type_error(std::string(name) + " must be bfloat16, float16 or float32");
  if (w.sizes() != shape) {
    std::string s = std::string(name) + " must have the shape [";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    value_error(s + "]");
  }
}
// Sizes are 32-bit in the C ABI: a view of many times the same values may have more along an axis.
void check_sizes(at::IntArrayRef sizes, int64_t most, const char* text) {
  for (const int64_t n : sizes)
    if (n > most) value_error(text);
}
float checked_eps(double eps) {
  if (!(eps >= 0.0) || std::isinf(eps)) value_error("eps must be a finite number that is not negative");
  return (float)eps;
}
// Derivatives in forward mode (dual tensors) are not worked out.  A dual tensor need not require a gradient, so a call that
// took it as an ordinary one would return a result whose derivative is zero; the same goes for a dual gradient.
bool is_dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
std::string no_forward_mode(const char* op) { return std::string(op) + " has no derivative in forward mode"; }
void no_duals(const char* op, std::initializer_list<const Maybe*> inputs) {
  for (const Maybe* t : inputs)
    if (*t && is_dual(**t)) runtime_error(no_forward_mode(op));
}
void once(const char* op, const Tensor& grad) {
  if (is_dual(grad)) throw std::runtime_error(no_forward_mode(op));
  if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(op) + " can be differentiated once; its gradient has no graph (create_graph)");
}
bool wants_grad(std::initializer_list<const Maybe*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Maybe* t : inputs)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}
const void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor dense(const Maybe& t) { return t ? t->contiguous() : Tensor(); }
Tensor last_axis_dense(const Tensor& t) { return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// The axes before the last one as three (or fewer) with strides; false where that takes more.
bool three_axes(const Tensor& t, int64_t* n, int64_t* st) {
  int used = 0;
  int64_t size[3] = {1, 1, 1}, stride[3] = {0, 0, 0};  // innermost first
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (used && t.stride(d) == stride[used - 1] * size[used - 1]) {
      size[used - 1] *= t.size(d);
      continue;
    }
    if (used == 3) return false;
    size[used] = t.size(d);
    stride[used++] = t.stride(d);
  }
  for (int i = 0; i < 3; ++i) n[2 - i] = size[i], st[2 - i] = stride[i];
  return true;
}
Tensor rows_in_place(const Tensor& t, int64_t* n, int64_t* st) {
  Tensor r = last_axis_dense(t);
  if (three_axes(r, n, st)) return r;
  r = r.contiguous();
  three_axes(r, n, st);
  return r;
}

// ---------------------------------------------------------------- layer norm

struct NormCall {
  Tensor x, w, b, stats, y;
  evoattn_layer_norm_params p{};
  NormCall(const Tensor& x_in, const Maybe& weight, const Maybe& bias, float eps) {
    x = rows_in_place(x_in, p.n, p.x_stride);
    w = dense(weight);
    b = dense(bias);
    fill(eps);
  }
  void fill(float eps) {
    p.dtype = dtype_code(x.scalar_type());
    p.C = (int32_t)x.size(-1);
    p.eps = eps;
    p.x = address(x);
    p.weight = address(w);
    p.bias = address(b);
    if (w.defined()) p.weight_dtype = dtype_code(w.scalar_type());
    if (b.defined()) p.bias_dtype = dtype_code(b.scalar_type());
  }
  void run(bool keep_stats) {
    y = at::empty(x.sizes(), x.options());
    p.y = y.data_ptr();
    if (keep_stats) {
      stats = at::empty({p.n[0] * p.n[1] * p.n[2], 2}, x.options().dtype(at::kFloat));
      p.stats = stats.data_ptr<float>();
    }
    check(evoattn_layer_norm_fwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_layer_norm_fwd");
  }
};

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    const c10::cuda::CUDAGuard guard(x.device());
    NormCall c(x, weight, bias, (float)eps);
    c.run(true);
    ctx->save_for_backward({c.x, c.w, c.b, c.stats});
    ctx->saved_data["eps"] = eps;
    return c.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("layer_norm", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    NormCall c(s[0], s[1].defined() ? Maybe(s[1]) : Maybe(), s[2].defined() ? Maybe(s[2]) : Maybe(), (float)ctx->saved_data["eps"].toDouble());
    Tensor dy = grads[0].scalar_type() == c.x.scalar_type() ? grads[0] : grads[0].to(c.x.scalar_type());
    // dy's rows in the axes of x: both as they lie where that works, else dy (and, failing that, x) dense
    int64_t n[3];
    evoattn_layer_norm_params& p = c.p;
    dy = rows_in_place(dy, n, p.d_y_stride);
    if (!std::equal(n, n + 3, p.n)) join(c, dy);
    p.d_y = address(dy);
    p.stats = s[3].data_ptr<float>();
    Tensor dx, dw, db;
    const size_t edge_w = 1, edge_b = c.w.defined() ? 2 : 1;
    if (ctx->needs_input_grad(0)) dx = at::empty(c.x.sizes(), c.x.options()), p.dx = dx.data_ptr();
    if (c.w.defined() && ctx->needs_input_grad(edge_w)) dw = at::empty(c.w.sizes(), c.w.options()), p.dweight = dw.data_ptr();
    if (c.b.defined() && ctx->needs_input_grad(edge_b)) db = at::empty(c.b.sizes(), c.b.options()), p.dbias = db.data_ptr();
    const size_t need = evoattn_layer_norm_bwd_workspace_bytes(&p);
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, c.x.options().dtype(at::kByte)), p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
    check(evoattn_layer_norm_bwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_layer_norm_bwd");
    return {dx, dw, db, Tensor()};
  }
  // x and dy whose rows fold into different axes: one set of up to three axes for both, by making one of them dense.
  static void join(NormCall& c, Tensor& dy) {
    evoattn_layer_norm_params& p = c.p;
    const auto split = [](const Tensor& dense, const int64_t* n, int64_t* st) {  // a dense tensor folds into any axes
      const int64_t C = dense.size(-1);
      st[2] = C; st[1] = n[2] * C; st[0] = n[1] * n[2] * C;
    };
    int64_t n[3];
    if (dy.is_contiguous()) {
      split(dy, p.n, p.d_y_stride);
    } else if (c.x.is_contiguous()) {
      dy = rows_in_place(dy, n, p.d_y_stride);
      std::copy(n, n + 3, p.n);
      split(c.x, p.n, p.x_stride);
    } else {
      dy = dy.contiguous();
      split(dy, p.n, p.d_y_stride);
    }
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  const Maybe xm(x);
  no_duals("layer_norm", {&xm, &weight, &bias});
  check_main(x, "layer_norm", "x");
  if (x.dim() < 1 || x.size(-1) < 1) value_error("x must have a last axis of at least one value");
  const int64_t C = x.size(-1);
  if (C > (1 << 24)) value_error("the last axis of x is too long");
  if (weight) check_weight(*weight, x, "weight", {C});
  if (bias) check_weight(*bias, x, "bias", {C});
  const float e = checked_eps(eps);
  if (wants_grad({&xm, &weight, &bias})) return LayerNorm::apply(x, weight, bias, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  NormCall c(x, weight, bias, e);
  c.run(false);
  return c.y;
}

// ---------------------------------------------------------------- relative position bias

struct RelativePlan {
  int64_t scheme, exact, buckets;
  std::vector<int32_t> edges;
};

// [B,1,H,Rq,Rk] whose rows begin on 16-byte boundaries, as the attention's tensor maps read a pair bias.
Tensor bias_rows(int64_t B, int64_t H, int64_t Rq, int64_t Rk, at::TensorOptions opt) {
  const int64_t per = 16 / (int64_t)c10::elementSize(c10::typeMetaToScalarType(opt.dtype())), ld = (Rk + per - 1) / per * per;
  return at::empty_strided({B, 1, H, Rq, Rk}, {H * Rq * ld, H * Rq * ld, Rq * ld, ld, 1}, opt);
}
void bias_strides(const Tensor& t, int64_t* st) {  // of (b, h, i) in [B,1,H,Rq,Rk]
  st[0] = t.stride(0); st[1] = t.stride(2); st[2] = t.stride(3);
}

struct RelativeCall {
  Tensor table, q, k, base;
  evoattn_relative_bias_params p{};
  RelativeCall(const Tensor& table_in, const Tensor& q_in, const Tensor& k_in, const RelativePlan& plan, int64_t B) {
    table = table_in.contiguous();
    // both in one type; rows contiguous
    const bool wide = q_in.scalar_type() == at::kLong || k_in.scalar_type() == at::kLong;
    q = last_axis_dense(q_in.to(wide ? at::kLong : at::kInt));
    k = last_axis_dense(k_in.to(wide ? at::kLong : at::kInt));
    p.table_dtype = dtype_code(table.scalar_type());
    p.B = (int32_t)B; p.H = (int32_t)table.size(1); p.Rq = (int32_t)q.size(-1); p.Rk = (int32_t)k.size(-1);
    p.buckets = (int32_t)plan.buckets; p.scheme = (int32_t)plan.scheme; p.exact = (int32_t)plan.exact;
    p.n_edges = (int32_t)plan.edges.size(); p.edges = plan.edges.data();
    p.positions64 = wide;
    p.table = address(table);
    p.q_pos = address(q); p.k_pos = address(k);
    p.q_pos_stride = q.dim() == 2 && q.size(0) > 1 ? q.stride(0) : 0;
    p.k_pos_stride = k.dim() == 2 && k.size(0) > 1 ? k.stride(0) : 0;
  }
  Tensor run(const Maybe& base_in, at::ScalarType type) {
    Tensor out = bias_rows(p.B, p.H, p.Rq, p.Rk, table.options().dtype(type));
    if (base_in) {
      base = last_axis_dense(*base_in);
      p.base = address(base);
      p.base_dtype = dtype_code(base.scalar_type());
      bias_strides(base, p.base_stride);
    }
    p.dtype = dtype_code(type);
    p.out = out.data_ptr();
    bias_strides(out, p.out_stride);
    check(evoattn_relative_bias_fwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_relative_bias_fwd");
    return out;
  }
};

struct RelativeBias : public torch::autograd::Function<RelativeBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Maybe& base, const Tensor& q, const Tensor& k,
                        const RelativePlan& plan, int64_t B, int64_t type) {
    const c10::cuda::CUDAGuard guard(table.device());
    RelativeCall c(table, q, k, plan, B);
    Tensor out = c.run(base, (at::ScalarType)type);
    ctx->save_for_backward({c.q, c.k});
    auto& sd = ctx->saved_data;
    sd["table"] = std::vector<int64_t>(table.sizes().vec());
    sd["table_t"] = (int64_t)table.scalar_type();
    sd["base_t"] = base ? (int64_t)base->scalar_type() : (int64_t)-1;
    sd["plan"] = std::vector<int64_t>{plan.scheme, plan.exact, plan.buckets, B};
    sd["edges"] = std::vector<int64_t>(plan.edges.begin(), plan.edges.end());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("relative_position_bias", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    auto& sd = ctx->saved_data;
    const Tensor& d_in = grads[0];
    const c10::cuda::CUDAGuard guard(d_in.device());
    const int64_t base_t = sd["base_t"].toInt();
    Tensor dtable, dbase;
    if (base_t >= 0 && ctx->needs_input_grad(1)) dbase = d_in.scalar_type() == (at::ScalarType)base_t ? d_in : d_in.to((at::ScalarType)base_t);
    if (ctx->needs_input_grad(0)) {
      const std::vector<int64_t> v = sd["plan"].toIntVector(), e = sd["edges"].toIntVector();
      const RelativePlan plan{v[0], v[1], v[2], std::vector<int32_t>(e.begin(), e.end())};
      dtable = at::empty(sd["table"].toIntVector(), d_in.options().dtype((at::ScalarType)sd["table_t"].toInt()));
      RelativeCall c(dtable, s[0], s[1], plan, v[3]);
      evoattn_relative_bias_params& p = c.p;
      p.table = nullptr;
      const Tensor d = last_axis_dense(d_in);
      p.dtype = dtype_code(d.scalar_type());
      p.d_out = address(d);
      bias_strides(d, p.d_out_stride);
      p.dtable = dtable.data_ptr();
      const size_t need = evoattn_relative_bias_bwd_workspace_bytes(&p);
      Tensor ws;
      if (need) ws = at::empty({(int64_t)need}, d.options().dtype(at::kByte)), p.workspace = ws.data_ptr();
      p.workspace_bytes = need;
      check(evoattn_relative_bias_bwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_relative_bias_bwd");
    }
    return {dtable, dbase, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_positions(const Tensor& t, const Tensor& table, const char* name) {
  if (t.device() != table.device()) runtime_error(std::string(name) + " is on " + t.device().str() + ", not on " + table.device().str());
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) type_error(std::string(name) + " must be int64 or int32");
  if (t.dim() != 1 && t.dim() != 2) value_error(std::string(name) + " must have the shape [N] or [B, N]");
}

Tensor relative_position_bias(const Tensor& table, const Tensor& q, const Maybe& keys, const Maybe& base, c10::optional<at::ScalarType> dtype,
                              int64_t scheme, int64_t exact, std::vector<int32_t> edges) {
  const Maybe tm(table);
  no_duals("relative_position_bias", {&tm, &base});
  check_main(table, "relative_position_bias", "table");
  if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1) value_error("table must have the shape [buckets, H]");
  const Tensor k = keys.value_or(q);
  check_positions(q, table, "positions");
  check_positions(k, table, "key_positions");
  const int64_t H = table.size(1), Rq = q.size(-1), Rk = k.size(-1);
  int64_t B = q.dim() == 2 ? q.size(0) : 1;
  const int64_t Bk = k.dim() == 2 ? k.size(0) : 1;
  if (B != Bk && B != 1 && Bk != 1) value_error("positions and key_positions differ in their batch");
  if (Bk != 1) B = Bk;
  if (base) {
    const Tensor& t = *base;
    if (t.device() != table.device()) runtime_error("pair_bias is on " + t.device().str() + ", not on " + table.device().str());
    if (!known(t.scalar_type())) type_error("pair_bias must be bfloat16, float16 or float32");
    if (t.dim() != 5 || t.size(1) != 1 || t.size(2) != H || t.size(3) != Rq || t.size(4) != Rk || (B != 1 && t.size(0) != B))
      value_error("pair_bias must have the shape [B, 1, H, N, N_keys] of the positions and the table");
    B = t.size(0);
  }
  check_sizes({B, H, Rq, Rk}, 1 << 23, "relative_position_bias takes up to 2^23 entries along an axis");
  const at::ScalarType type = dtype ? *dtype : base ? base->scalar_type() : table.scalar_type();
  if (!known(type)) type_error("dtype must be bfloat16, float16 or float32");
  const RelativePlan plan{scheme, exact, table.size(0), std::move(edges)};
  if (wants_grad({&tm, &base})) return RelativeBias::apply(table, base, q, k, plan, B, (int64_t)type);
  const c10::cuda::CUDAGuard guard(table.device());
  RelativeCall c(table, q, k, plan, B);
  return c.run(base, type);
}

// ---------------------------------------------------------------- pair-bias projection

struct ProjectionCall {
  Tensor z, w, g, b;
  evoattn_pair_projection_params p{};
  ProjectionCall(const Tensor& pair, const Tensor& weight, const Maybe& norm_weight, const Maybe& norm_bias, float eps) {
    z = last_axis_dense(pair);
    w = weight.contiguous();
    g = dense(norm_weight);
    b = dense(norm_bias);
    p.dtype = dtype_code(z.scalar_type());
    p.weight_dtype = dtype_code(w.scalar_type());
    if (g.defined()) p.norm_weight_dtype = dtype_code(g.scalar_type());
    if (b.defined()) p.norm_bias_dtype = dtype_code(b.scalar_type());
    p.eps = eps;
    p.B = (int32_t)z.size(0); p.Ri = (int32_t)z.size(1); p.Rj = (int32_t)z.size(2); p.C = (int32_t)z.size(3); p.H = (int32_t)w.size(0);
    p.pair = address(z);
    for (int i = 0; i < 3; ++i) p.pair_stride[i] = z.stride(i);
    p.weight = address(w); p.norm_weight = address(g); p.norm_bias = address(b);
  }
  Tensor run() {
    Tensor out = bias_rows(p.B, p.H, p.Ri, p.Rj, z.options());
    p.out = out.data_ptr();
    bias_strides(out, p.out_stride);
    check(evoattn_pair_projection_fwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_pair_projection_fwd");
    return out;
  }
};

struct PairProjection : public torch::autograd::Function<PairProjection> {
  static Tensor forward(AutogradContext* ctx, const Tensor& pair, const Tensor& weight, const Maybe& norm_weight, const Maybe& norm_bias, double eps) {
    const c10::cuda::CUDAGuard guard(pair.device());
    ProjectionCall c(pair, weight, norm_weight, norm_bias, (float)eps);
    Tensor out = c.run();
    ctx->save_for_backward({c.z, c.w, c.g, c.b});
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("pair_bias_projection", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    ProjectionCall c(s[0], s[1], s[2].defined() ? Maybe(s[2]) : Maybe(), s[3].defined() ? Maybe(s[3]) : Maybe(), (float)ctx->saved_data["eps"].toDouble());
    const Tensor d = last_axis_dense(grads[0].scalar_type() == c.z.scalar_type() ? grads[0] : grads[0].to(c.z.scalar_type()));
    evoattn_pair_projection_params& p = c.p;
    p.d_out = address(d);
    bias_strides(d, p.d_out_stride);
    Tensor dz, dw, dg, db;
    const size_t edge_g = 2, edge_b = c.g.defined() ? 3 : 2;
    if (ctx->needs_input_grad(0)) dz = at::empty(c.z.sizes(), c.z.options()), p.dpair = dz.data_ptr();
    if (ctx->needs_input_grad(1)) dw = at::empty(c.w.sizes(), c.w.options()), p.dweight = dw.data_ptr();
    if (c.g.defined() && ctx->needs_input_grad(edge_g)) dg = at::empty(c.g.sizes(), c.g.options()), p.dnorm_weight = dg.data_ptr();
    if (c.b.defined() && ctx->needs_input_grad(edge_b)) db = at::empty(c.b.sizes(), c.b.options()), p.dnorm_bias = db.data_ptr();
    const size_t need = evoattn_pair_projection_bwd_workspace_bytes(&p);
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, c.z.options().dtype(at::kByte)), p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
    check(evoattn_pair_projection_bwd(&p, at::cuda::getCurrentCUDAStream().stream()), "evoattn_pair_projection_bwd");
    return {dz, dw, dg, db, Tensor()};
  }
};

Tensor pair_bias_projection(const Tensor& pair, const Tensor& weight, const Maybe& norm_weight, const Maybe& norm_bias, double eps) {
  const Maybe zm(pair), wm(weight);
  no_duals("pair_bias_projection", {&zm, &wm, &norm_weight, &norm_bias});
  check_main(pair, "pair_bias_projection", "pair");
  if (pair.dim() != 4 || pair.size(3) < 1) value_error("pair must have the shape [B, N_res, N_res, C]");
  const int64_t C = pair.size(3);
  if (weight.dim() != 2 || weight.size(0) < 1) value_error("weight must have the shape [H, C]");
  check_weight(weight, pair, "weight", {weight.size(0), C});
  if (C > EVOATTN_PROJECTION_MAX_C || weight.size(0) > EVOATTN_PROJECTION_MAX_H)
    value_error("pair_bias_projection takes up to " + std::to_string(EVOATTN_PROJECTION_MAX_C) + " channels and " + std::to_string(EVOATTN_PROJECTION_MAX_H) + " heads");
  check_sizes(pair.sizes(), 1 << 20, "pair may have up to 2^20 entries along an axis");
  if (norm_weight) check_weight(*norm_weight, pair, "norm_weight", {C});
  if (norm_bias) check_weight(*norm_bias, pair, "norm_bias", {C});
  const float e = checked_eps(eps);
  if (wants_grad({&zm, &wm, &norm_weight, &norm_bias})) return PairProjection::apply(pair, weight, norm_weight, norm_bias, eps);
  const c10::cuda::CUDAGuard guard(pair.device());
  ProjectionCall c(pair, weight, norm_weight, norm_bias, e);
  return c.run();
}

}  // namespace

void register_inputs(py::module& m) {
  m.def("layer_norm", &layer_norm);
  m.def("relative_position_bias", &relative_position_bias);
  m.def("pair_bias_projection", &pair_bias_projection);
}

}  // namespace evohost
