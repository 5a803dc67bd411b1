// The short causal convolution and the selective scan as autograd operators; part of ops.cpp.
#pragma once
#include "../cuda/selective_scan.h"

extern "C" {
int esgd_causal_conv_fwd(const void* x, int64_t xb, int64_t xt, const void* state, const float* weight, const float* bias,
                         const int64_t* lengths, void* y, void* state_out, int is_bf16, int64_t batch, int64_t length, int channels, int taps,
                         int act, void* stream);
int64_t esgd_causal_conv_parts(int64_t batch, int64_t length, int channels);
int esgd_causal_conv_bwd(const void* x, int64_t xb, int64_t xt, const void* state, const float* weight, const float* bias,
                         const int64_t* lengths, const void* dy, void* dx, float* sums, int64_t* parts, int is_bf16, int64_t batch,
                         int64_t length, int channels, int taps, int act, void* stream);
int esgd_causal_conv_step(const void* x, int64_t xb, const void* state, void* state_out, const float* weight, const float* bias, void* y,
                          int is_bf16, int64_t batch, int channels, int taps, int act, void* stream);
int64_t esgd_selective_scan_local(const esgd_scan* e, int backward);
int64_t esgd_selective_scan_keep(const esgd_scan* e);
int64_t esgd_selective_scan_narrow(const esgd_scan* e);
int64_t esgd_selective_scan_parts(const esgd_scan* e);
int esgd_selective_scan_fwd(const esgd_scan* e, void* out, float* state_out, float* keep, float* local, void* stream);
int esgd_selective_scan_bwd(const esgd_scan* e, const void* dout, const float* keep, void* du, void* ddelta, void* dz, void* dB, void* dC,
                            float* narrow, float* sums, float* local, void* stream);
int esgd_selective_scan_step(const esgd_scan* e, float* state_out, void* out, void* stream);
}

namespace {

using Opt = c10::optional<Tensor>;

// Rows are read where they lie, whatever is between them; the values of a row have to be next to each other.
Tensor rows_dense(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
const int64_t* lengths_of(const Tensor& t) { return t.defined() ? t.data_ptr<int64_t>() : nullptr; }
void check_lengths(const char* op, const Opt& lengths, const Tensor& x) {
  if (!lengths.has_value()) return;
  TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == x.size(0) && lengths->is_contiguous(), op, ": lengths ", lengths->sizes(), " for ",
              x.size(0), " sequences");
  check_operand(op, "lengths", *lengths, x, at::kLong);
}
// A state carries no gradient: a sequence that is trained over its whole length has none.
void check_state(const char* op, const Opt& state, const Tensor& x, at::IntArrayRef shape, at::ScalarType type) {
  if (!state.has_value()) return;
  TORCH_CHECK(state->sizes() == shape && state->is_contiguous(), op, ": a state of ", state->sizes(), ", not ", shape, " in a row");
  check_operand(op, "the state", *state, x, type);
  TORCH_CHECK(!differentiable(*state), op, ": no gradient goes through a state: detach it");
}
// Where a step leaves the new state: a tensor of its own, or the caller's (which may be the old state itself, not a part of it).
Tensor state_for(const char* op, const Opt& out, const Tensor& state) {
  if (!out.has_value()) return at::empty_like(state);
  TORCH_CHECK(out->sizes() == state.sizes() && out->is_contiguous(), op, ": out ", out->sizes(), " is no room for a state of ", state.sizes());
  check_operand(op, "out", *out, state, state.scalar_type());
  TORCH_CHECK(!differentiable(*out), op, ": no gradient goes through out: detach it");
  const char *a = (const char*)state.data_ptr(), *b = (const char*)out->data_ptr();
  TORCH_CHECK(a == b || a + state.nbytes() <= b || b + out->nbytes() <= a, op, ": out overlaps the state without being it");
  return *out;
}
Tensor room(int64_t floats, const Tensor& like) { return floats > 0 ? fresh_floats({floats}, like) : Tensor(); }
void written(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// ---------------------------------------------------------------- causal convolution
struct CausalConvFn : public Function<CausalConvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_in, const Opt& weight_in, const Opt& bias_in, const Held& weight,
                               const Held& bias, const Held& state, const Held& lengths, int64_t act, bool want_state, const Sink& ws,
                               const Sink& bs, const Opt& anchor) {
    const Tensor x = rows_dense(x_in);
    variable_list out = run(x, weight.t, bias.t, state.t, lengths.t, act, want_state);
    ctx->save_for_backward({x, weight.t, bias.t, state.t, lengths.t});
    ctx->saved_data["act"] = act;
    ctx->saved_data["need"] = (int64_t)x_in.requires_grad() | wants(weight_in) << 1 | wants(bias_in) << 2;
    save_sink(ctx, "w", ws);
    save_sink(ctx, "b", bs);
    if (want_state) ctx->mark_non_differentiable({out[1]});
    return out;
  }
  static variable_list run(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, const Tensor& lengths, int64_t act,
                           bool want_state) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t b = x.size(0), t = x.size(1), d = x.size(2), taps = weight.size(1);
    variable_list out = {fresh({b, t, d}, x.scalar_type(), x)};
    if (want_state) out.push_back(fresh({b, taps - 1, d}, x.scalar_type(), x));
    ck(esgd_causal_conv_fwd(ptr(x), x.stride(0), x.stride(1), ptr(state), fptr(weight), fptr(bias), lengths_of(lengths), mut(out[0]),
                            want_state ? mut(out[1]) : nullptr, x.scalar_type() == at::kBFloat16, b, t, (int)d, (int)taps, (int)act, stream_of(x)),
       "causal_conv");
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(12);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &state = saved[3], &lengths = saved[4];
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t b = x.size(0), t = x.size(1), d = x.size(2), taps = weight.size(1);
    const bool is_bf16 = x.scalar_type() == at::kBFloat16;
    const Tensor dy = dense(grads[0]);
    const ParamGrad dw(ctx, "w", need & 2, {d, taps}, x), db(ctx, "b", need & 4, {d}, x);
    Tensor dx, sums;
    if (need & 1) dx = fresh({b, t, d}, x.scalar_type(), x);
    const bool any = dw.out() != nullptr || db.out() != nullptr;
    if (any) sums = fresh_floats({esgd_causal_conv_parts(b, t, (int)d), d * (taps + 1)}, x);
    int64_t parts = 0;
    ck(esgd_causal_conv_bwd(ptr(x), x.stride(0), x.stride(1), ptr(state), fptr(weight), fptr(bias), lengths_of(lengths), ptr(dy), mut(dx),
                            fptr(sums), &parts, is_bf16, b, t, (int)d, (int)taps, (int)ctx->saved_data["act"].toInt(), stream_of(x)),
       "causal_conv backward");
    if (any)
      ck(esgd_sum_parts(fptr(sums), parts, dw.out(), d * taps, dw.add(), db.out(), d, db.add(), nullptr, 0, 0, stream_of(x)),
         "causal_conv parameter gradients");
    dw.done();
    db.done();
    out[0] = dx; out[1] = dw.grad; out[2] = db.grad;
    return once("causal_conv", grads, std::move(out));
  }
};

void check_conv_operands(const char* op, const Tensor& x, const Tensor& weight, const Opt& bias, int64_t act) {
  check_float(op, "the input", x);
  const int64_t d = x.size(-1);
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) == d && weight.size(1) >= 2 && weight.size(1) <= 4 && weight.is_contiguous(), op,
              ": a weight of ", weight.sizes(), " for ", d, " channels; takes two to four taps a channel, in a row");
  check_operand(op, "the weight", weight, x, at::kFloat);
  if (bias.has_value()) check_vector(op, "the bias", *bias, x, d);
  TORCH_CHECK(act == 0 || act == 2, op, ": no such activation");
  TORCH_CHECK(d >= 1 && d < ((int64_t)1 << 27), op, ": ", d, " channels");
}

// x [B, T, D] bf16 or fp32, weight [D, K] fp32 -> y [B, T, D] and, if wanted, the last K - 1 inputs [B, K - 1, D].
variable_list causal_conv(const Tensor& x, const Tensor& weight, const Opt& bias_in, int64_t act, const Opt& state, const Opt& lengths,
                          bool want_state) {
  const char* op = "causal_conv";
  TORCH_CHECK(x.dim() == 3, op, ": takes a 3-D input, not ", x.sizes());
  check_conv_operands(op, x, weight, bias_in, act);
  check_lengths(op, lengths, x);
  check_state(op, state, x, {x.size(0), weight.size(1) - 1, x.size(2)}, x.scalar_type());
  TORCH_CHECK(x.size(0) * ((x.size(1) + 31) / 32) * ((x.size(2) + 31) / 32) < ((int64_t)1 << 30), op, ": an input of ", x.sizes(), " is too large");
  refuse_tangents(op, x, weight, bias_in, state);
  check_gpu(op, x);
  const Tensor bias = value_of(bias_in);
  if (!differentiable(x) && !differentiable(weight) && !differentiable(bias))
    return CausalConvFn::run(rows_dense(x), weight, bias, value_of(state), value_of(lengths), act, want_state);
  Sink ws = find_sink(weight), bs = find_sink(bias);
  check_capture(op, {&x, ws ? &x : &weight, bs ? &x : &bias});
  sink_use(ws);
  sink_use(bs);
  return CausalConvFn::apply(x, graph_only(weight, ws), bias.defined() ? graph_only(bias, bs) : Opt(), Held{weight}, Held{bias},
                             Held{value_of(state)}, Held{value_of(lengths)}, act, want_state, ws, bs, anchor_for(x, ws || bs));
}

// One input [B, D] more.
std::pair<Tensor, Tensor> causal_conv_step(const Tensor& x_in, const Tensor& state, const Tensor& weight, const Opt& bias, int64_t act,
                                           const Opt& out) {
  const char* op = "causal_conv_step";
  TORCH_CHECK(x_in.dim() == 2, op, ": takes a 2-D input, not ", x_in.sizes());
  check_conv_operands(op, x_in, weight, bias, act);
  check_state(op, state, x_in, {x_in.size(0), weight.size(1) - 1, x_in.size(1)}, x_in.scalar_type());
  TORCH_CHECK(!differentiable(x_in) && !differentiable(weight) && !(bias.has_value() && differentiable(*bias)), op,
              ": no gradient goes through a step; call it under torch.no_grad()");
  const Tensor next = state_for(op, out, state);
  refuse_tangents(op, x_in, state, weight, bias);
  check_gpu(op, x_in);
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = rows_dense(x_in);
  const int64_t b = x.size(0), d = x.size(1);
  TORCH_CHECK(b * d < ((int64_t)1 << 37), op, ": an input of ", x.sizes(), " is too large");
  Tensor y = fresh({b, d}, x.scalar_type(), x);
  ck(esgd_causal_conv_step(ptr(x), x.stride(0), ptr(state), mut(next), fptr(weight), fptr(value_of(bias)), mut(y),
                           x.scalar_type() == at::kBFloat16, b, (int)d, (int)weight.size(1), (int)act, stream_of(x)), op);
  written(next);
  return {y, next};
}

// ---------------------------------------------------------------- selective scan
struct ScanInputs {
  Tensor u, delta, z, B, C, A, D, bias, state, lengths;
  bool softplus;
  esgd_scan args() const {
    esgd_scan e = {};
    const Tensor* seq[5] = {&u, &delta, &z, &B, &C};
    const bool step = u.dim() == 2;
    for (int i = 0; i < 5; ++i) {
      e.p[i] = ptr(*seq[i]);
      if (!seq[i]->defined()) continue;
      e.b[i] = seq[i]->stride(0);
      e.t[i] = step ? 0 : seq[i]->stride(1);
    }
    e.A = fptr(A); e.D = fptr(D); e.bias = fptr(bias);
    e.lengths = lengths_of(lengths);
    e.state = fptr(state);
    e.batch = u.size(0);
    e.length = step ? 1 : u.size(1);
    e.channels = (int)u.size(-1);
    e.states = (int)A.size(1);
    e.softplus = softplus;
    e.is_bf16 = u.scalar_type() == at::kBFloat16;
    return e;
  }
};

struct SelectiveScanFn : public Function<SelectiveScanFn> {
  // The parameters that a step's accumulators take come as Held, and not as A_in, D_in, bias_in.
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Opt& A_in, const Tensor& B, const Tensor& C,
                               const Opt& D_in, const Opt& z, const Opt& bias_in, const Held& A, const Held& D, const Held& bias,
                               const Held& state, const Held& lengths, bool softplus, bool want_state, const Sink& as, const Sink& ds,
                               const Sink& bs, const Opt& anchor) {
    const ScanInputs in = {rows_dense(u), rows_dense(delta), z.has_value() ? rows_dense(*z) : Tensor(), rows_dense(B), rows_dense(C), A.t, D.t,
                           bias.t, state.t, lengths.t, softplus};
    Tensor keep;
    variable_list out = run(in, want_state, &keep);
    ctx->save_for_backward({in.u, in.delta, in.z, in.B, in.C, A.t, D.t, bias.t, lengths.t, keep});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["need"] = wants(A_in) | wants(D_in) << 1 | wants(bias_in) << 2;
    save_sink(ctx, "A", as);
    save_sink(ctx, "D", ds);
    save_sink(ctx, "b", bs);
    if (want_state) ctx->mark_non_differentiable({out[1]});
    return out;
  }
  static variable_list run(const ScanInputs& in, bool want_state, Tensor* keep) {
    c10::cuda::CUDAGuard guard(in.u.device());
    const esgd_scan e = in.args();
    variable_list out = {fresh(in.u.sizes(), in.u.scalar_type(), in.u)};
    if (want_state) out.push_back(fresh_floats({e.batch, e.channels, e.states}, in.u));
    if (keep != nullptr) *keep = fresh_floats({esgd_selective_scan_keep(&e)}, in.u);
    const Tensor local = room(esgd_selective_scan_local(&e, 0), in.u);
    ck(esgd_selective_scan_fwd(&e, mut(out[0]), want_state ? fptr(out[1]) : nullptr, keep != nullptr ? fptr(*keep) : nullptr, fptr(local),
                               stream_of(in.u)), "selective_scan");
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(19);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const ScanInputs in = {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], Tensor(), saved[8],
                           ctx->saved_data["softplus"].toBool()};
    const Tensor& keep = saved[9];
    c10::cuda::CUDAGuard guard(in.u.device());
    const esgd_scan e = in.args();
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t d = e.channels, n = e.states;
    const auto type = in.u.scalar_type();
    const Tensor dout = dense(grads[0]);
    Tensor du = fresh(in.u.sizes(), type, in.u), ddelta = fresh(in.u.sizes(), type, in.u), dz = in.z.defined() ? fresh(in.u.sizes(), type, in.u) : Tensor();
    Tensor dB = fresh({e.batch, e.length, n}, type, in.u), dC = fresh({e.batch, e.length, n}, type, in.u);
    const ParamGrad dA(ctx, "A", need & 1, {d, n}, in.u), dD(ctx, "D", need & 2, {d}, in.u), db(ctx, "b", need & 4, {d}, in.u);
    // one workspace: the shares of dB and dC, those of the parameters, and the chunks' states; each on 16 bytes
    const int64_t parts = esgd_selective_scan_parts(&e), n_narrow = esgd_selective_scan_narrow(&e), n_sums = (parts * d * (n + 2) + 3) / 4 * 4;
    const Tensor work = room(n_narrow + n_sums + esgd_selective_scan_local(&e, 1), in.u);
    float *narrow = fptr(work), *sums = narrow + n_narrow, *local = sums + n_sums;
    ck(esgd_selective_scan_bwd(&e, ptr(dout), fptr(keep), mut(du), mut(ddelta), mut(dz), mut(dB), mut(dC), narrow, sums, local,
                               stream_of(in.u)), "selective_scan backward");
    ck(esgd_sum_parts(sums, parts, dA.out(), d * n, dA.add(), dD.out(), d, dD.add(), db.out(), d, db.add(), stream_of(in.u)),
       "selective_scan parameter gradients");
    dA.done();
    dD.done();
    db.done();
    out[0] = du; out[1] = ddelta; out[2] = dA.grad; out[3] = dB; out[4] = dC; out[5] = dD.grad; out[6] = dz; out[7] = db.grad;
    return once("selective_scan", grads, std::move(out));
  }
};

// What a scan and its step have in common: u [..., D], delta, z like it, B and C [..., N], A [D, N].
void check_scan_operands(const char* op, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
                         const Opt& z, const Opt& bias) {
  check_float(op, "u", u);
  const int64_t d = u.size(-1);
  TORCH_CHECK(A.dim() == 2 && A.size(0) == d && A.size(1) >= 1 && A.size(1) <= 64 && A.is_contiguous(), op, ": A is ", A.sizes(), " for ", d,
              " channels; takes one to 64 states a channel, in a row");
  check_operand(op, "A", A, u, at::kFloat);
  auto narrow = u.sizes().vec();
  narrow.back() = A.size(1);
  TORCH_CHECK(delta.sizes() == u.sizes() && B.sizes() == at::IntArrayRef(narrow) && C.sizes() == at::IntArrayRef(narrow), op, ": delta ",
              delta.sizes(), ", B ", B.sizes(), " and C ", C.sizes(), " for u ", u.sizes(), " and ", A.size(1), " states");
  check_operand(op, "delta", delta, u, u.scalar_type());
  check_operand(op, "B", B, u, u.scalar_type());
  check_operand(op, "C", C, u, u.scalar_type());
  if (z.has_value()) {
    TORCH_CHECK(z->sizes() == u.sizes(), op, ": z ", z->sizes(), " is not of u's size ", u.sizes());
    check_operand(op, "z", *z, u, u.scalar_type());
  }
  if (D.has_value()) check_vector(op, "D", *D, u, d);
  if (bias.has_value()) check_vector(op, "delta_bias", *bias, u, d);
  TORCH_CHECK(d >= 1 && d < ((int64_t)1 << 25) && u.size(0) * ((d + 7) / 8) < ((int64_t)1 << 31), op, ": u of ", u.sizes(), " is too large");
}

// -> out [B, T, D] and, if wanted, the last state [B, D, N] (fp32).
variable_list selective_scan(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D_in,
                             const Opt& z, const Opt& bias_in, bool softplus, const Opt& state, const Opt& lengths, bool want_state) {
  const char* op = "selective_scan";
  TORCH_CHECK(u.dim() == 3, op, ": takes a 3-D u, not ", u.sizes());
  check_scan_operands(op, u, delta, A, B, C, D_in, z, bias_in);
  check_lengths(op, lengths, u);
  check_state(op, state, u, {u.size(0), u.size(2), A.size(1)}, at::kFloat);
  refuse_tangents(op, u, delta, A, B, C, D_in, z, bias_in, state);
  check_gpu(op, u);
  const Tensor D = value_of(D_in), bias = value_of(bias_in), gate = value_of(z);
  if (!differentiable(u) && !differentiable(delta) && !differentiable(A) && !differentiable(B) && !differentiable(C) && !differentiable(D) &&
      !differentiable(gate) && !differentiable(bias))
    return SelectiveScanFn::run({rows_dense(u), rows_dense(delta), gate.defined() ? rows_dense(gate) : Tensor(), rows_dense(B), rows_dense(C), A,
                                 D, bias, value_of(state), value_of(lengths), softplus}, want_state, nullptr);
  Sink as = find_sink(A), ds = find_sink(D), bs = find_sink(bias);
  check_capture(op, {&u, &delta, &B, &C, &gate, as ? &u : &A, ds ? &u : &D, bs ? &u : &bias});
  sink_use(as);
  sink_use(ds);
  sink_use(bs);
  return SelectiveScanFn::apply(u, delta, graph_only(A, as), B, C, D.defined() ? graph_only(D, ds) : Opt(), z,
                                bias.defined() ? graph_only(bias, bs) : Opt(), Held{A}, Held{D}, Held{bias}, Held{value_of(state)},
                                Held{value_of(lengths)}, softplus, want_state, as, ds, bs, anchor_for(u, as || ds || bs));
}

// One step more: u, delta, z [B, D], B and C [B, N], state [B, D, N].
std::pair<Tensor, Tensor> selective_scan_step(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                                              const Tensor& state, const Opt& D, const Opt& z, const Opt& bias, bool softplus, const Opt& out) {
  const char* op = "selective_scan_step";
  TORCH_CHECK(u.dim() == 2, op, ": takes a 2-D u, not ", u.sizes());
  check_scan_operands(op, u, delta, A, B, C, D, z, bias);
  check_state(op, state, u, {u.size(0), u.size(1), A.size(1)}, at::kFloat);
  for (const Tensor* t : {&u, &delta, &A, &B, &C})
    TORCH_CHECK(!differentiable(*t), op, ": no gradient goes through a step; call it under torch.no_grad()");
  for (const Opt* t : {&D, &z, &bias})
    TORCH_CHECK(!t->has_value() || !differentiable(**t), op, ": no gradient goes through a step; call it under torch.no_grad()");
  const Tensor next = state_for(op, out, state);
  refuse_tangents(op, u, delta, A, B, C, state, D, z, bias);
  check_gpu(op, u);
  c10::cuda::CUDAGuard guard(u.device());
  const ScanInputs in = {rows_dense(u), rows_dense(delta), z.has_value() ? rows_dense(*z) : Tensor(), rows_dense(B), rows_dense(C), A,
                         value_of(D), value_of(bias), state, Tensor(), softplus};
  const esgd_scan e = in.args();
  Tensor y = fresh(u.sizes(), u.scalar_type(), u);
  ck(esgd_selective_scan_step(&e, fptr(next), mut(y), stream_of(u)), op);
  written(next);
  return {y, next};
}

}  // namespace
