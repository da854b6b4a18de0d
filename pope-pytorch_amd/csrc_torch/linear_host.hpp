// Eager calls of the linear attention, its step and the gated norm: included by pope_host.cpp, in its namespace.
#pragma once

// A call's operands in the caller's layout: rows (batch, heads, n, dim) or (batch, n, heads, dim).
struct LinearArgs {
  Tensor q, k, v, freqs, bias, log_decay, mask, cu, initial;
  double scale;
  bool with_state, head_first;
  bool o_f32 = false;   // o in fp32: the gated norm goes on from it

  int h() const { return head_first ? 1 : 2; }
  int n() const { return head_first ? 2 : 1; }
  int64_t sequences() const { return cu.defined() ? cu.size(0) - 1 : q.size(0); }

  void strides(int64_t* s, const Tensor& t) const { s[0] = t.stride(0), s[1] = t.stride(h()), s[2] = t.stride(n()); }
  at::ScalarType o_type() const { return o_f32 ? at::kFloat : q.scalar_type(); }
  Tensor rows(int64_t heads, int64_t cols, at::ScalarType dtype) const {
    const auto o = q.options().dtype(dtype).requires_grad(false);
    return head_first ? at::empty({q.size(0), heads, q.size(n()), cols}, o) : at::empty({q.size(0), q.size(n()), heads, cols}, o);
  }

  // Whether the call is as the kernels take it, up to conversions that convert() makes; otherwise the Python module converts, or
  // says what is wrong.
  bool fits() const {
    const auto here = [&](const Tensor& t) { return !t.defined() || t.device() == q.device(); };
    const auto type = [](const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; };
    if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || !type(q) ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
      return false;
    for (const Tensor* t : {&k, &v, &freqs, &bias, &log_decay, &mask, &cu, &initial})
      if (!here(*t)) return false;
    const int64_t B = q.size(0), N = q.size(n()), H = k.size(h()), D = q.size(3), Dv = v.size(3);
    if (B < 1 || N < 1 || H < 1 || q.size(h()) < 1 || q.size(h()) % H || k.size(0) != B || k.size(n()) != N || k.size(3) != D || D < 1 || D > 256 || v.size(0) != B ||
        v.size(h()) != H || v.size(n()) != N || Dv < 1 || Dv > 256)
      return false;
    if (freqs.defined() != bias.defined()) return false;
    if (freqs.defined()) {
      const int64_t R = freqs.size(-1);
      if (freqs.dim() < 2 || freqs.dim() > 3 || R < 1 || R > D || freqs.size(-2) != N || (freqs.dim() == 3 && freqs.size(0) != 1 && freqs.size(0) != B) || !type(freqs) ||
          !type(bias) || bias.dim() != 2 || bias.size(1) != R || (bias.size(0) != 1 && bias.size(0) != H))
        return false;
    }
    if (log_decay.defined() && (log_decay.scalar_type() != at::kFloat || log_decay.dim() != 1 || log_decay.size(0) != H || !log_decay.is_contiguous() || tracked(log_decay)))
      return false;
    if (mask.defined() && (mask.scalar_type() != at::kBool || mask.dim() != 2 || mask.size(0) != B || mask.size(1) != N)) return false;
    if (cu.defined() && (cu.scalar_type() != at::kInt || cu.dim() != 1 || cu.size(0) < 2 || !cu.is_contiguous() || B != 1)) return false;
    if (initial.defined() && (!type(initial) || initial.dim() != 4 || initial.size(0) != sequences() || initial.size(1) != H ||
                              initial.size(2) != D + (freqs.defined() ? freqs.size(-1) : 0) || initial.size(3) != Dv))
      return false;
    return true;
  }
  static bool tracked(const Tensor& t) { return t.defined() && ((t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined()); }

  // Rows as the kernels address them: unit feature stride, and not so far apart that a chunk's offsets pass 32 bits.
  static Tensor near_rows(const Tensor& t, int n) { return t.stride(-1) == 1 && t.stride(n) < POPE_LINEAR_ROW_STRIDE ? t : t.contiguous(); }

  // Rows near each other, fp32 angles and states; the bias is read as it is.
  LinearArgs convert() const {
    LinearArgs a = *this;
    for (Tensor* t : {&a.q, &a.k, &a.v}) *t = near_rows(*t, n());
    if (a.freqs.defined()) a.freqs = near_rows(a.freqs.to(at::kFloat), -2);
    if (a.bias.defined()) a.bias = unit_feature(a.bias);
    if (a.mask.defined() && a.mask.stride(1) != 1) a.mask = a.mask.contiguous();
    if (a.initial.defined()) a.initial = a.initial.to(at::kFloat).contiguous();
    return a;
  }

  pope_linear desc() const {
    pope_linear d{};
    const int64_t most = INT_MAX;
    TORCH_CHECK_VALUE(sequences() <= most && q.size(n()) <= most && q.size(h()) <= most, "pope_amd linear attention: too large");
    d.B = (int32_t)sequences();
    d.N = (int32_t)q.size(n());
    d.Hq = (int32_t)q.size(h());
    d.Hk = (int32_t)k.size(h());
    d.D = (int32_t)q.size(3);
    d.R = freqs.defined() ? (int32_t)freqs.size(-1) : 0;
    d.Dv = (int32_t)v.size(3);
    d.dtype = dtype_code(q);
    d.o_f32 = o_f32;
    d.scale = (float)scale;
    strides(d.q_s, q);
    strides(d.k_s, k);
    strides(d.v_s, v);
    if (freqs.defined()) {
      d.f_s[0] = freqs.dim() == 3 && freqs.size(0) > 1 ? freqs.stride(0) : 0;
      d.f_s[1] = freqs.stride(-2);
      d.bias_dtype = dtype_code(bias);
      d.bias_sh = bias.size(0) > 1 ? bias.stride(0) : 0;
    }
    if (mask.defined()) d.mask_sb = mask.stride(0);
    return d;
  }
  Tensor state() const { return fp32_like(q, {sequences(), k.size(h()), q.size(3) + (freqs.defined() ? freqs.size(-1) : 0), v.size(3)}); }
};

// Operands as the library reads them: what callers of the ops may have wrong.
void check_linear_operands(const LinearArgs& a) {
  check_device(a.q, {&a.k, &a.v, &a.freqs, &a.bias, &a.log_decay, &a.mask, &a.cu, &a.initial});
  TORCH_CHECK_VALUE(a.fits(), "pope_amd linear attention: operands do not fit (q ", a.q.sizes(), ", k ", a.k.sizes(), ", v ", a.v.sizes(), ")");
}

const uint8_t* bytes_of(const Tensor& t) { return static_cast<const uint8_t*>(data(t)); }
const int32_t* ints_of(const Tensor& t) { return static_cast<const int32_t*>(data(t)); }

struct LinearOut {
  Tensor o, last, kept;
};

LinearOut linear_forward(const LinearArgs& a) {   // converted operands
  pope_linear d = a.desc();
  const c10::DeviceGuard guard(a.q.device());
  LinearOut r;
  r.o = a.rows(d.Hq, d.Dv, a.o_type());
  a.strides(d.o_s, r.o);
  if (a.with_state) r.last = a.state();
  size_t n[2] = {0, 0};
  check(pope_linear_bytes(&d, a.cu.defined(), a.with_state, 0, n), "workspace query");
  r.kept = bytes_like(a.q, n[0]);
  check(pope_linear_fwd(&d, a.q.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), floats(a.freqs), data(a.bias), floats(a.log_decay), bytes_of(a.mask), ints_of(a.cu),
                        floats(a.initial), r.o.data_ptr(), static_cast<float*>(data(r.last)), data(r.kept), n[0], stream_of(a.q)),
        "linear attention");
  return r;
}

struct LinearGrads {
  Tensor dq, dk, dv, dfreqs, dbias, dinitial;
};

LinearGrads linear_backward(const LinearArgs& a, const Tensor& dout0, const Tensor& dlast0, const Tensor& kept, bool need_df, bool need_db, bool need_d0) {
  pope_linear d = a.desc();
  const c10::DeviceGuard guard(a.q.device());
  Tensor dout = dout0;
  if (!dout.defined()) dout = a.rows(d.Hq, d.Dv, a.o_type()).zero_();
  if (dout.scalar_type() != a.o_type()) dout = dout.to(a.o_type());
  dout = LinearArgs::near_rows(dout, dout.dim() == 4 ? a.n() : 0);
  const Tensor dlast = dlast0.defined() ? dlast0.to(at::kFloat).contiguous() : Tensor();
  check_device(a.q, {&dout, &dlast, &kept});
  TORCH_CHECK_VALUE(dout.dim() == 4 && dout.size(0) == a.q.size(0) && dout.size(a.h()) == d.Hq && dout.size(a.n()) == d.N && dout.size(3) == d.Dv, "dout ", dout.sizes(),
                    " does not fit the linear attention");
  a.strides(d.do_s, dout);
  LinearGrads r;
  r.dq = a.rows(d.Hq, d.D, a.q.scalar_type());
  r.dk = a.rows(d.Hk, d.D, a.q.scalar_type());
  r.dv = a.rows(d.Hk, d.Dv, a.q.scalar_type());
  a.strides(d.dq_s, r.dq);
  a.strides(d.dk_s, r.dk);
  a.strides(d.dv_s, r.dv);
  if (need_df) {
    r.dfreqs = fp32_like(a.q, a.freqs.sizes());
    d.df_s[0] = a.freqs.dim() == 3 && a.freqs.size(0) > 1 ? r.dfreqs.stride(0) : 0;
    d.df_s[1] = r.dfreqs.stride(-2);
  }
  // the library takes a stride of 0 for one bias row, and so for one gradient row: a row that a view repeats for the heads is copied
  Tensor bias = a.bias;
  if (need_db) {
    r.dbias = at::empty(bias.sizes(), bias.options().requires_grad(false));
    if (bias.size(0) > 1 && bias.stride(0) == 0) {
      bias = bias.contiguous();
      d.bias_sh = bias.stride(0);
    }
  }
  if (need_d0) r.dinitial = fp32_like(a.q, {d.B, d.Hk, d.D + d.R, d.Dv});
  TORCH_CHECK_VALUE(!dlast.defined() || dlast.numel() == (int64_t)d.B * d.Hk * (d.D + d.R) * d.Dv, "the states' gradient ", dlast.sizes(), " does not fit");
  size_t n[2] = {0, 0};
  check(pope_linear_bytes(&d, a.cu.defined(), 0, need_df, n), "workspace query");
  const Tensor ws = bytes_like(a.q, n[1]);
  check(pope_linear_bwd(&d, dout.data_ptr(), floats(dlast), a.q.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), floats(a.freqs), data(bias), floats(a.log_decay),
                        bytes_of(a.mask), ints_of(a.cu), floats(a.initial), data(kept), kept.defined() ? kept.nbytes() : 0, r.dq.data_ptr(), r.dk.data_ptr(),
                        r.dv.data_ptr(), static_cast<float*>(data(r.dfreqs)), data(r.dbias), static_cast<float*>(data(r.dinitial)), data(ws), n[1],
                        stream_of(a.q)),
        "linear attention backward");
  return r;
}

using Grads6 = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

struct LinearFn : torch::autograd::Function<LinearFn> {
  // every tensor is passed, undefined where there is none, so that inputs keep their numbers
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias, OptTensor initial,
                               OptTensor log_decay, OptTensor mask, OptTensor cu, double scale, bool with_state, bool head_first, bool o_f32) {
    const LinearArgs raw{q, k, v, opt(freqs), opt(bias), opt(log_decay), opt(mask), opt(cu), opt(initial), scale, with_state, head_first, o_f32};
    const LinearArgs a = raw.convert();
    const LinearOut r = linear_forward(a);
    ctx->save_for_backward({q, k, v, raw.freqs, raw.bias, raw.initial, a.log_decay, a.mask, a.cu, r.kept});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["with_state"] = with_state;
    ctx->saved_data["head_first"] = head_first;
    ctx->saved_data["o_f32"] = o_f32;
    // which gradients an undefined input would shift: positions of the optional inputs among the node's
    int64_t at = 3;
    for (const auto& [name, t] : {std::pair<const char*, Tensor>{"freqs", raw.freqs}, {"bias", raw.bias}, {"initial", raw.initial}}) {
      ctx->saved_data[name] = t.defined() ? at : (int64_t)-1;
      if (t.defined()) ++at;
    }
    ctx->set_materialize_grads(false);
    return with_state ? variable_list{r.o, r.last} : variable_list{r.o};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list sv = ctx->get_saved_variables();
    const bool hf = ctx->saved_data["head_first"].toBool();
    const LinearArgs raw{sv[0], sv[1], sv[2], sv[3], sv[4], sv[6], sv[7], sv[8], sv[5], ctx->saved_data["scale"].toDouble(), ctx->saved_data["with_state"].toBool(), hf, ctx->saved_data["o_f32"].toBool()};
    const auto need = [&](const char* name) {
      const int64_t at = ctx->saved_data[name].toInt();
      return at >= 0 && ctx->needs_input_grad(at);
    };
    const bool ndf = need("freqs"), ndb = need("bias"), nd0 = need("initial");
    const Tensor dlast = grads.size() > 1 ? grads[1] : Tensor();
    LinearGrads r;
    if (on_ops(grads)) {
      const auto front = [&](const Tensor& t) { return hf || !t.defined() ? t : t.transpose(1, 2); };
      const auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      const auto f32 = [](const Tensor& t) { return t.defined() ? t.to(at::kFloat) : t; };
      const Tensor dout = grads[0].defined() ? front(grads[0]) : at::zeros({sv[0].size(0), front(sv[0]).size(1), front(sv[0]).size(2), sv[2].size(3)}, sv[0].options().dtype(raw.o_type()).requires_grad(false));
      using O = OptTensor;
      std::tie(r.dq, r.dk, r.dv, r.dfreqs, r.dbias, r.dinitial) =
          op<Grads6(const Tensor&, O, const Tensor&, const Tensor&, const Tensor&, O, O, O, O, O, O, O, double, bool, bool, bool, bool)>("pope_amd::linear_bwd")
              .call(dout, maybe(dlast), front(sv[0]), front(sv[1]), front(sv[2]), maybe(f32(sv[3])), maybe(sv[4]), maybe(sv[6]), maybe(sv[7]), maybe(sv[8]),
                    maybe(f32(sv[5])), maybe(sv[9]), raw.scale, raw.o_f32, ndf, ndb, nd0);
      r.dq = front(r.dq), r.dk = front(r.dk), r.dv = front(r.dv);
    } else {
      r = linear_backward(raw.convert(), grads[0], dlast, sv[9], ndf, ndb, nd0);
    }
    const auto like = [](const Tensor& g, const Tensor& t, bool want) { return want ? (g.scalar_type() == t.scalar_type() ? g : g.to(t.scalar_type())) : Tensor(); };
    variable_list out{r.dq, r.dk, r.dv, like(r.dfreqs, sv[3], ndf), ndb ? r.dbias : Tensor(), like(r.dinitial, sv[5], nd0)};
    out.resize(13);
    return on_ops(grads) ? out : once_differentiable(std::move(out), "linear attention");
  }
};

// (o, last or nothing); nothing at all where the call is not as the kernels take it.
std::optional<std::pair<Tensor, std::optional<Tensor>>> linear_eager(const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias,
                                                                     OptTensor log_decay, OptTensor mask, OptTensor cu, OptTensor initial, double scale,
                                                                     bool with_state, bool head_first, bool o_f32) {
  const LinearArgs a{q, k, v, opt(freqs), opt(bias), opt(log_decay), opt(mask), opt(cu), opt(initial), scale, with_state, head_first, o_f32};
  if (!a.fits()) return std::nullopt;
  const auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  if (tracked({a.q, a.k, a.v, a.freqs, a.bias, a.initial})) {
    const variable_list r = LinearFn::apply(q, k, v, freqs, bias, initial, log_decay, mask, cu, scale, with_state, head_first, o_f32);
    return std::make_pair(r[0], with_state ? maybe(r[1]) : std::nullopt);
  }
  const LinearOut r = linear_forward(a.convert());
  return std::make_pair(r.o, maybe(r.last));
}

// The ops' implementations: head-first rows.  Nothing is undefined in what an op returns.
std::tuple<Tensor, Tensor, Tensor> linear_fwd_impl(const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias, OptTensor log_decay, OptTensor mask,
                                                   OptTensor cu, OptTensor initial, double scale, bool with_state, bool o_f32) {
  const LinearArgs a{q, k, v, opt(freqs), opt(bias), opt(log_decay), opt(mask), opt(cu), opt(initial), scale, with_state, true, o_f32};
  check_linear_operands(a);
  const LinearOut r = linear_forward(a.convert());
  return {r.o, r.last.defined() ? r.last : fp32_like(q, {0}), r.kept};
}

Grads6 linear_bwd_impl(const Tensor& dout, OptTensor dlast, const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias, OptTensor log_decay,
                       OptTensor mask, OptTensor cu, OptTensor initial, OptTensor kept, double scale, bool o_f32, bool need_df, bool need_db, bool need_d0) {
  const LinearArgs a{q, k, v, opt(freqs), opt(bias), opt(log_decay), opt(mask), opt(cu), opt(initial), scale, false, true, o_f32};
  check_linear_operands(a);
  const LinearGrads r = linear_backward(a.convert(), dout, opt(dlast), opt(kept), need_df, need_db, need_d0);
  const auto some = [&](const Tensor& t) { return t.defined() ? t : fp32_like(q, {0}); };
  return {r.dq, r.dk, r.dv, some(r.dfreqs), some(r.dbias), some(r.dinitial)};
}

// ---------------------------------------------------------------- the step

// The norm's weight as the kernels read it: (1 or heads, cols), unit stride.
pope_gated_norm norm_desc(const Tensor& weight, int64_t cols, double eps, int dtype) {
  pope_gated_norm d{};
  d.cols = (int32_t)cols;
  d.dtype = dtype;
  d.eps = (float)eps;
  d.weight_rows = 1;
  if (weight.defined()) {
    d.weight_f32 = weight.scalar_type() == at::kFloat;
    if (weight.dim() == 2) {
      d.weight_rows = (int32_t)weight.size(0);
      d.weight_sh = weight.stride(0);
    }
  }
  return d;
}
bool weight_fits(const Tensor& w, const Tensor& x, int64_t heads, int64_t cols) {
  return !w.defined() || (w.device() == x.device() && (w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat) && (w.dim() == 1 || w.dim() == 2) &&
                          w.size(-1) == cols && (w.dim() == 1 || w.size(0) == 1 || w.size(0) == heads) && w.stride(-1) == 1);
}

struct StepArgs {
  LinearArgs a;
  Tensor state, from, to, gate, weight;
  double eps;

  bool fits() const {
    if (!a.fits() || a.q.size(a.n()) != 1) return false;
    const auto tr = LinearArgs::tracked;
    for (const Tensor* t : {&a.q, &a.k, &a.v, &a.freqs, &a.bias, &state, &gate, &weight})
      if (tr(*t)) return false;
    const int64_t H = a.k.size(a.h()), E = a.q.size(3) + (a.freqs.defined() ? a.freqs.size(-1) : 0), Dv = a.v.size(3), B = a.q.size(0);
    if (state.device() != a.q.device() || state.scalar_type() != at::kFloat || state.dim() != 4 || state.size(0) < 1 || state.size(1) != H || state.size(2) != E || state.size(3) != Dv ||
        state.stride(3) != 1 || state.stride(2) != Dv || state.stride(1) != E * Dv || (state.size(0) > 1 && state.stride(0) < H * E * Dv) || state.size(0) > INT_MAX)
      return false;
    if (!from.defined() && B > state.size(0)) return false;
    for (const Tensor* t : {&from, &to})
      if (t->defined() && (t->scalar_type() != at::kInt || t->device() != a.q.device() || t->dim() != 1 || t->size(0) != B || !t->is_contiguous())) return false;
    if (gate.defined() && (gate.scalar_type() != a.q.scalar_type() || gate.device() != a.q.device() || gate.dim() != 4 || gate.size(0) != B || gate.size(a.h()) != a.q.size(a.h()) ||
                           gate.size(a.n()) != 1 || gate.size(3) != Dv || gate.stride(3) != 1))
      return false;
    return gate.defined() ? weight_fits(weight, a.q, a.q.size(a.h()), Dv) : !weight.defined();
  }

  Tensor run() const {
    const LinearArgs c = a.convert();
    pope_linear d = c.desc();
    const c10::DeviceGuard guard(a.q.device());
    const Tensor o = c.rows(d.Hq, d.Dv, c.o_type());
    c.strides(d.o_s, o);
    pope_gated_norm n{};
    if (gate.defined()) {
      n = norm_desc(weight, d.Dv, eps, d.dtype);
      n.B = d.B, n.H = d.Hq, n.N = 1;
      c.strides(n.gate_s, gate);
    }
    const int64_t slot = state.size(0) > 1 ? state.stride(0) : state.size(1) * state.size(2) * state.size(3);
    check(pope_linear_step(&d, c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), floats(c.freqs), data(c.bias), floats(c.log_decay), static_cast<float*>(state.data_ptr()),
                           (int32_t)state.size(0), slot, ints_of(from), ints_of(to), gate.defined() ? &n : nullptr, data(gate), data(weight), o.data_ptr(), stream_of(a.q)),
          "linear attention step");
    return o;
  }
};

std::optional<Tensor> linear_step_eager(const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias, OptTensor log_decay, const Tensor& state,
                                        OptTensor from, OptTensor to, OptTensor gate, OptTensor weight, double eps, double scale, bool head_first) {
  const StepArgs s{{q, k, v, opt(freqs), opt(bias), opt(log_decay), Tensor(), Tensor(), Tensor(), scale, false, head_first}, state, opt(from), opt(to), opt(gate), opt(weight), eps};
  if (!s.fits()) return std::nullopt;
  const Tensor o = s.run();
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return o;
}

Tensor linear_step_impl(const Tensor& q, const Tensor& k, const Tensor& v, OptTensor freqs, OptTensor bias, OptTensor log_decay, const Tensor& state, OptTensor from, OptTensor to,
                        OptTensor gate, OptTensor weight, double eps, double scale) {
  const StepArgs s{{q, k, v, opt(freqs), opt(bias), opt(log_decay), Tensor(), Tensor(), Tensor(), scale, false, true}, state, opt(from), opt(to), opt(gate), opt(weight), eps};
  TORCH_CHECK_VALUE(s.fits(), "pope_amd linear attention step: operands do not fit (q ", q.sizes(), ", state ", state.sizes(), ")");
  return s.run();
}

// ---------------------------------------------------------------- the gated norm

struct NormArgs {
  Tensor x, gate, weight;
  double eps;
  bool head_first;
  int h() const { return head_first ? 1 : 2; }
  int n() const { return head_first ? 2 : 1; }
  bool fits() const {
    const at::ScalarType t = gate.scalar_type();
    if (!x.is_cuda() || x.dim() != 4 || (t != at::kFloat && t != at::kHalf && t != at::kBFloat16) || gate.device() != x.device() ||
        (x.scalar_type() != t && x.scalar_type() != at::kFloat) || gate.sizes() != x.sizes() || x.size(3) < 1 || x.size(3) > 512 || x.size(h()) < 1)
      return false;
    return weight_fits(weight, gate, x.size(h()), x.size(3));
  }
  void strides(int64_t* s, const Tensor& t) const { s[0] = t.stride(0), s[1] = t.stride(h()), s[2] = t.stride(n()); }
  pope_gated_norm desc() const {   // x and gate of unit feature stride
    TORCH_CHECK_VALUE(x.size(0) <= INT_MAX && x.size(1) <= INT_MAX && x.size(2) <= INT_MAX, "pope_amd gated norm: too large");
    pope_gated_norm d = norm_desc(weight, x.size(3), eps, dtype_code(gate));
    d.x_f32 = x.scalar_type() == at::kFloat;
    d.B = (int32_t)x.size(0), d.H = (int32_t)x.size(h()), d.N = (int32_t)x.size(n());
    strides(d.x_s, x);
    strides(d.gate_s, gate);
    return d;
  }
  NormArgs convert() const { return {unit_feature(x), unit_feature(gate), weight, eps, head_first}; }
};

Tensor norm_forward(const NormArgs& a) {
  pope_gated_norm d = a.desc();
  const c10::DeviceGuard guard(a.x.device());
  const Tensor y = rows_like(a.x, a.gate.scalar_type());
  a.strides(d.y_s, y);
  check(pope_gated_norm_fwd(&d, a.x.data_ptr(), a.gate.data_ptr(), data(a.weight), y.data_ptr(), stream_of(a.x)), "gated norm");
  return y;
}

variable_list norm_backward(const NormArgs& a, Tensor dy, bool need_dw) {
  pope_gated_norm d = a.desc();
  const c10::DeviceGuard guard(a.x.device());
  if (dy.scalar_type() != a.gate.scalar_type()) dy = dy.to(a.gate.scalar_type());
  dy = unit_feature(dy);
  check_device(a.x, {&dy});
  TORCH_CHECK_VALUE(dy.sizes() == a.x.sizes(), "dy ", dy.sizes(), " must match x ", a.x.sizes());
  const Tensor dx = rows_like(a.x), dg = rows_like(a.gate);
  a.strides(d.dy_s, dy);
  a.strides(d.dx_s, dx);
  a.strides(d.dgate_s, dg);
  Tensor dw, ws;
  size_t n = 0;
  if (need_dw) {
    const auto o = a.weight.options().requires_grad(false);
    dw = a.x.numel() ? at::empty(a.weight.sizes(), o) : at::zeros(a.weight.sizes(), o);
    check(pope_gated_norm_bytes(&d, &n), "workspace query");
    ws = bytes_like(a.x, n);
  }
  check(pope_gated_norm_bwd(&d, dy.data_ptr(), a.x.data_ptr(), a.gate.data_ptr(), data(a.weight), dx.data_ptr(), dg.data_ptr(), data(dw), data(ws), n, stream_of(a.x)),
        "gated norm backward");
  return {dx, dg, dw};
}

struct GatedNormFn : torch::autograd::Function<GatedNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, OptTensor weight, double eps, bool head_first) {
    ctx->save_for_backward({x, gate, opt(weight)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["head_first"] = head_first;
    return norm_forward(NormArgs{x, gate, opt(weight), eps, head_first}.convert());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list sv = ctx->get_saved_variables();
    const bool ndw = sv[2].defined() && ctx->needs_input_grad(2), hf = ctx->saved_data["head_first"].toBool();
    const double eps = ctx->saved_data["eps"].toDouble();
    if (on_ops(grads)) {
      const auto [dx, dg, dw] = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, OptTensor, double, bool, bool)>("pope_amd::gated_norm_bwd")
                                    .call(grads[0], sv[0], sv[1], sv[2].defined() ? std::optional<Tensor>(sv[2]) : std::nullopt, eps, hf, ndw);
      return {dx, dg, ndw ? dw : Tensor(), Tensor(), Tensor()};
    }
    variable_list r = norm_backward(NormArgs{sv[0], sv[1], sv[2], eps, hf}.convert(), grads[0], ndw);
    r.resize(5);
    return once_differentiable(std::move(r), "gated norm");
  }
};

std::optional<Tensor> gated_norm_eager(const Tensor& x, const Tensor& gate, OptTensor weight, double eps, bool head_first) {
  const NormArgs a{x, gate, opt(weight), eps, head_first};
  if (!a.fits()) return std::nullopt;
  if (tracked({x, gate, a.weight})) return GatedNormFn::apply(x, gate, weight, eps, head_first);
  return norm_forward(a.convert());
}

Tensor gated_norm_fwd_impl(const Tensor& x, const Tensor& gate, OptTensor weight, double eps, bool head_first) {
  const NormArgs a{x, gate, opt(weight), eps, head_first};
  TORCH_CHECK_VALUE(a.fits(), "pope_amd gated norm: operands do not fit (x ", x.sizes(), ", gate ", gate.sizes(), ")");
  return norm_forward(a.convert());
}

std::tuple<Tensor, Tensor, Tensor> gated_norm_bwd_impl(const Tensor& dy, const Tensor& x, const Tensor& gate, OptTensor weight, double eps, bool head_first, bool need_dw) {
  const NormArgs a{x, gate, opt(weight), eps, head_first};
  TORCH_CHECK_VALUE(a.fits(), "pope_amd gated norm: operands do not fit (x ", x.sizes(), ", gate ", gate.sizes(), ")");
  const variable_list r = norm_backward(a.convert(), dy, need_dw);
  return {r[0], r[1], r[2].defined() ? r[2] : fp32_like(x, {0})};
}
