// The autograd boundary of the operators of packed sequences (rotary positions, attention), in native code as that of the
// others is.
#include "host_common.h"

namespace evohost {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
void same_device(const Tensor& t, const Tensor& as, const char* name) {
  if (t.device() != as.device()) runtime_error(std::string(name) + " is on " + t.device().str() + ", not on " + as.device().str());
}
bool whole(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// ---------------------------------------------------------------- rotary positions

struct RotaryPlan {
  int64_t layout;
  double amplitude;
};

// x turned (both: q and k; either may be undefined) into fresh dense tensors.
variable_list rotate(const Tensor& q_in, const Tensor& k_in, const Tensor& positions, const Tensor& frequencies, const RotaryPlan& plan, bool inverse) {
  evoattn_rotary_params p{};
  const Tensor& any = q_in.defined() ? q_in : k_in;
  const Tensor q = q_in.defined() ? last_axis_dense(q_in) : q_in, k = k_in.defined() ? last_axis_dense(k_in) : k_in;
  const int64_t axes = any.dim() - 2;
  for (int64_t i = 0; i < 3; ++i) p.n[i] = 1;
  for (int64_t i = 0; i < axes; ++i) {
    p.n[3 - axes + i] = any.size(i);
    if (q.defined()) p.q_stride[3 - axes + i] = q.stride(i);
    if (k.defined()) p.k_stride[3 - axes + i] = k.stride(i);
    if (positions.dim() == axes) p.position_stride[3 - axes + i] = positions.size(i) == 1 ? 0 : positions.stride(i);
  }
  if (positions.dim() == 1) p.position_stride[2] = positions.stride(0);
  p.dtype = dtype_code(any.scalar_type());
  p.layout = (int32_t)plan.layout;
  p.inverse = inverse;
  p.positions64 = positions.scalar_type() == at::kLong;
  p.frequencies64 = frequencies.scalar_type() == at::kDouble;
  p.amplitude = (float)plan.amplitude;
  p.D = (int32_t)any.size(-1);
  p.rotary = (int32_t)(2 * frequencies.size(0));
  p.positions = positions.data_ptr();
  p.frequencies = frequencies.data_ptr();
  Tensor qo, ko;
  if (q.defined()) {
    qo = at::empty(q.sizes(), q.options());
    p.q = q.data_ptr(); p.q_out = qo.data_ptr(); p.H = (int32_t)q.size(-2); p.q_stride[3] = q.stride(-2);
  }
  if (k.defined()) {
    ko = at::empty(k.sizes(), k.options());
    p.k = k.data_ptr(); p.k_out = ko.data_ptr(); p.Hk = (int32_t)k.size(-2); p.k_stride[3] = k.stride(-2);
  }
  if (any.numel() > 0) check(evoattn_rotary(&p, stream()), "evoattn_rotary");
  return {qo, ko};
}

struct Rotary : public torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, const Tensor& positions, const Tensor& frequencies,
                               int64_t layout, double amplitude) {
    const c10::cuda::CUDAGuard guard(q.device());
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["layout"] = layout;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["type"] = (int64_t)q.scalar_type();
    ctx->set_materialize_grads(false);
    variable_list out = rotate(q, k ? *k : Tensor(), positions, frequencies, {layout, amplitude}, false);
    if (!k) out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool two = grads.size() > 1;
    for (const Tensor& g : grads) once("rotary_embedding", g);
    const variable_list s = ctx->get_saved_variables();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor d[2];
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && ctx->needs_input_grad(i)) d[i] = grads[i].scalar_type() == type ? grads[i] : grads[i].to(type);
    variable_list out{Tensor(), Tensor()};
    if (d[0].defined() || d[1].defined()) {
      const c10::cuda::CUDAGuard guard(s[0].device());
      out = rotate(d[0], two ? d[1] : Tensor(), s[0], s[1], {ctx->saved_data["layout"].toInt(), ctx->saved_data["amplitude"].toDouble()}, true);
    }
    return {out[0], out[1], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::object rotary_embedding(const Tensor& q, const Maybe& k, const Tensor& positions, const Tensor& frequencies, int64_t layout, double amplitude) {
  const char* op = "rotary_embedding";
  const Maybe qm(q), fm(frequencies);
  no_duals(op, {&qm, &k, &fm});
  check_main(q, op, "q");
  if (q.dim() < 3 || q.dim() > 5 || q.size(-1) < 1 || q.size(-2) < 1) value_error("q must have the shape [..., N, H, D] with up to two axes before N");
  const int64_t axes = q.dim() - 2, D = q.size(-1);
  if (D > EVOATTN_ROTARY_MAX_D || q.size(-2) > 65536) value_error("rotary_embedding takes head dimensions up to " + std::to_string(EVOATTN_ROTARY_MAX_D) + " and up to 65536 heads");
  if (k) {
    same_device(*k, q, "k");
    if (k->scalar_type() != q.scalar_type()) type_error("q and k must be of one type");
    if (k->dim() != q.dim() || k->size(-1) != D || k->size(-2) < 1 || k->size(-2) > 65536 || k->sizes().slice(0, axes) != q.sizes().slice(0, axes))
      value_error("k must have the shape of q but for the number of heads");
  }
  int64_t tokens = 1;
  for (int64_t i = 0; i < axes; ++i) {
    if (q.size(i) > 0x7fffffff || (tokens *= q.size(i)) > 0x7fffffff) value_error("q may have up to 2^31 - 1 tokens");
  }
  same_device(positions, q, "positions");
  if (!whole(positions)) type_error("positions must be int64 or int32");
  bool fits = positions.dim() == 1 ? positions.size(0) == q.size(axes - 1) : positions.dim() == axes;
  if (fits && positions.dim() > 1) {
    for (int64_t i = 0; i < axes; ++i) fits = fits && (positions.size(i) == q.size(i) || (i < axes - 1 && positions.size(i) == 1));
  }
  if (!fits) value_error("positions must have the shape [N], or that of the axes of q before its heads (1 for any but N)");
  same_device(frequencies, q, "frequencies");
  if (frequencies.scalar_type() != at::kDouble && frequencies.scalar_type() != at::kFloat) type_error("frequencies must be float64 or float32");
  if (frequencies.dim() != 1 || frequencies.size(0) < 1 || 2 * frequencies.size(0) > D) value_error("frequencies must have the shape [n] with 1 <= n <= D / 2");
  if (at::GradMode::is_enabled() && frequencies.requires_grad()) value_error("rotary_embedding has no gradient for the frequencies");
  if (!std::isfinite(amplitude) || !std::isfinite((float)amplitude)) value_error("amplitude must be a finite number");
  const Tensor f = dense(frequencies);
  variable_list out;
  if (wants_grad({&qm, &k})) {
    out = Rotary::apply(q, k, positions, f, layout, amplitude);
  } else {
    const c10::cuda::CUDAGuard guard(q.device());
    out = rotate(q, k ? *k : Tensor(), positions, f, {layout, amplitude}, false);
  }
  if (!k) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

// ---------------------------------------------------------------- attention over packed sequences

// Where the tensor-core kernels could take a call (16 bits, head dimensions in eights up to 128), an operand that a tensor
// map cannot read (rows off 16 bytes, steps of zero or backwards) is copied; elsewhere it is read as it lies.
Tensor mapped(const Tensor& t) {
  const Tensor r = last_axis_dense(t);
  if (r.scalar_type() == at::kFloat || r.size(2) % 8 || r.size(2) > 128 || r.numel() == 0) return r;
  const auto step = [](int64_t n, int64_t st) { return n == 1 || (st > 0 && st % 8 == 0); };
  return !((uintptr_t)r.data_ptr() & 15) && step(r.size(0), r.stride(0)) && step(r.size(1), r.stride(1)) ? r : r.clone(at::MemoryFormat::Contiguous);
}

struct PackedPlan {
  bool causal;
  double scale;
};
struct PackedCall {
  Tensor q, k, v, offsets, keys, o, lse, rest;
  evoattn_packed_params p{};
  PackedCall(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& off, const Tensor& key_off, const PackedPlan& plan)
      : q(mapped(q_in)), k(mapped(k_in)), v(mapped(v_in)), offsets(off), keys(key_off) {
    p.dtype = dtype_code(q.scalar_type());
    p.B = (int32_t)(offsets.size(0) - 1); p.H = (int32_t)q.size(1); p.Hk = (int32_t)k.size(1); p.D = (int32_t)q.size(2);
    p.causal = plan.causal;
    p.offsets64 = offsets.scalar_type() == at::kLong;
    p.key_form = keys.defined() && keys.dim() == 2 ? EVOATTN_PACKED_KEY_RANGES : EVOATTN_PACKED_KEY_OFFSETS;
    p.flags = generic_forced() ? EVOATTN_FLAG_FORCE_GENERIC : 0;
    p.scale = (float)plan.scale;
    p.Tq = q.size(0); p.Tk = k.size(0);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr();
    strides(q, p.q_stride); strides(k, p.k_stride); strides(v, p.v_stride);
    p.offsets = offsets.data_ptr();
    p.key_offsets = address(keys);
    p.status = status_ptr(q.device());
  }
  static void strides(const Tensor& t, int64_t* st) { st[0] = t.stride(0); st[1] = t.stride(1); }
  Tensor scratch(size_t need) {
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte)), p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
    return ws;
  }
  bool empty() const { return p.B < 1 || p.Tq < 1 || p.Tk < 1; }
  void run(bool keep_lse) {
    if (empty()) {
      o = at::zeros(q.sizes(), q.options());
      return;
    }
    o = at::empty(q.sizes(), q.options());
    p.o = o.data_ptr();
    if (keep_lse) {
      lse = at::empty({p.H, p.Tq}, q.options().dtype(at::kFloat));
      p.lse = lse.data_ptr<float>();
      if (p.dtype != EVOATTN_FP32) rest = at::empty(q.sizes(), q.options()), p.o_rest = rest.data_ptr();
    }
    const Tensor ws = scratch(evoattn_packed_fwd_workspace_bytes(&p));
    check(evoattn_packed_fwd(&p, stream()), "evoattn_packed_fwd");
    note_call(false);
  }
};

struct Packed : public torch::autograd::Function<Packed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, const Maybe& keys,
                        bool causal, double scale) {
    const c10::cuda::CUDAGuard guard(q.device());
    PackedCall c(q, k, v, offsets, keys ? *keys : Tensor(), {causal, scale});
    c.run(true);
    ctx->save_for_backward({c.q, c.k, c.v, c.offsets, c.keys, c.o, c.lse, c.rest});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return c.o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("packed_attention", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    PackedCall c(s[0], s[1], s[2], s[3], s[4], {ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble()});
    evoattn_packed_params& p = c.p;
    Tensor dq, dk, dv;
    const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    auto make = [&](const Tensor& t) { return c.empty() ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options()); };
    if (ctx->needs_input_grad(0)) dq = make(c.q), p.dq = address(dq) ? dq.data_ptr() : nullptr;
    if (keys) dk = make(c.k), dv = make(c.v), p.dk = dk.data_ptr(), p.dv = dv.data_ptr();
    if (!c.empty()) {
      const Tensor d = mapped(grads[0].scalar_type() == c.q.scalar_type() ? grads[0] : grads[0].to(c.q.scalar_type()));
      p.o = s[5].data_ptr();
      p.lse = s[6].data_ptr<float>();
      p.o_rest = s[7].defined() ? s[7].data_ptr() : nullptr;
      p.d_o = d.data_ptr();
      PackedCall::strides(d, p.do_stride);
      const Tensor ws = c.scratch(evoattn_packed_bwd_workspace_bytes(&p));
      check(evoattn_packed_bwd(&p, stream()), "evoattn_packed_bwd");
      note_call(true);
    }
    return {dq, ctx->needs_input_grad(1) ? dk : Tensor(), ctx->needs_input_grad(2) ? dv : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_rows(const Tensor& t, const Tensor& q, const char* name) {
  same_device(t, q, name);
  if (t.scalar_type() != q.scalar_type()) type_error("q, k and v must be of one type");
  if (t.dim() != 3) value_error(std::string(name) + " must have the shape [T, H, D]");
  if (t.size(0) > (1 << 30)) value_error(std::string(name) + " may have up to 2^30 rows");
}

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, const Maybe& key_offsets, bool causal,
                        c10::optional<double> scale_in) {
  const char* op = "packed_attention";
  const Maybe qm(q), km(k), vm(v);
  no_duals(op, {&qm, &km, &vm});
  check_main(q, op, "q");
  check_rows(q, q, "q");
  check_rows(k, q, "k");
  check_rows(v, q, "v");
  const int64_t H = q.size(1), D = q.size(2), Hk = k.size(1);
  if (H < 1 || D < 1 || Hk < 1 || H % Hk || H > 65535) value_error("q must have a multiple of the heads of k, at most 65535");
  if (q.size(0) * H > (1LL << 33)) value_error("q may have up to 2^33 rows over its heads");
  if (D > EVOATTN_PACKED_MAX_D) value_error("packed_attention takes head dimensions up to " + std::to_string(EVOATTN_PACKED_MAX_D));
  if (k.size(2) != D || v.sizes() != k.sizes()) value_error("k and v must have the shape [T, H_k, D] with the head dimension of q");
  same_device(offsets, q, "offsets");
  if (!whole(offsets)) type_error("offsets must be int64 or int32");
  if (offsets.dim() != 1 || offsets.size(0) < 1 || offsets.size(0) > (1 << 30)) value_error("offsets must have the shape [B + 1]");
  const int64_t B = offsets.size(0) - 1;
  Maybe keys;
  if (key_offsets) {
    same_device(*key_offsets, q, "key_offsets");
    if (!whole(*key_offsets)) type_error("key_offsets must be int64 or int32");
    const bool ranges = key_offsets->dim() == 2 && key_offsets->size(0) == B && key_offsets->size(1) == 2;
    if (!ranges && !(key_offsets->dim() == 1 && key_offsets->size(0) == B + 1)) value_error("key_offsets must have the shape [B + 1] or [B, 2]");
    keys = *key_offsets;
  } else if (q.size(0) != k.size(0)) {
    value_error("without key_offsets, k must have as many rows as q");
  }
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)D);
  if (!std::isfinite(scale) || !std::isfinite((float)scale)) value_error("scale must be a finite number");
  const bool grad = wants_grad({&qm, &km, &vm});
  if (grad && keys && keys->dim() == 2 && (k.requires_grad() || v.requires_grad()))
    value_error("keys in ranges have no gradient (two sequences may share them): detach k and v, or pass offsets");
  const c10::cuda::CUDAGuard guard(q.device());
  // both offsets dense and of one type (converted where they lie: nothing waits for the device)
  Tensor off = offsets.contiguous();
  if (keys) {
    if (keys->scalar_type() != off.scalar_type()) {
      if (off.scalar_type() == at::kInt) off = off.to(at::kLong);
      else keys = keys->to(at::kLong);
    }
    keys = keys->contiguous();
  }
  if (grad) return Packed::apply(q, k, v, off, keys, causal, scale);
  PackedCall c(q, k, v, off, keys ? *keys : Tensor(), {causal, scale});
  c.run(false);
  return c.o;
}

}  // namespace

void register_sequences(py::module& m) {
  m.def("rotary_embedding", &rotary_embedding);
  m.def("packed_attention", &packed_attention);
}

}  // namespace evohost
