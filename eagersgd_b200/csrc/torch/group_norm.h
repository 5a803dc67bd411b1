// Group norm (+ residual) (+ activation) as an autograd operator; part of ops.cpp.
#pragma once
#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

extern "C" {
int esgd_group_norm_max_group();
int esgd_group_norm_fits(int64_t samples, int64_t rows, int channels, int groups, int is_bf16);
int esgd_group_norm_fwd(const void* x, const void* residual, void* z, const float* gamma, const float* beta, float* stats, int is_bf16,
                        int64_t samples, int64_t rows, int channels, int groups, int act, float eps, void* stream);
int esgd_group_norm_bwd(const void* x, const void* residual, const void* dz, void* dx, void* dres, const float* gamma, const float* beta,
                        const float* stats, float* sums, int is_bf16, int64_t samples, int64_t rows, int channels, int groups, int act,
                        void* stream);
int esgd_sum_parts(const float* ws, int64_t parts, float* a, int64_t na, int add_a, float* b, int64_t nb, int add_b, float* c, int64_t nc,
                   int add_c, void* stream);
}

namespace {

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// at::empty without its way through the dispatcher: an operator's backward pass has up to ten of them, two microseconds each.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
Tensor fresh_floats(at::IntArrayRef sizes, const Tensor& like) { return fresh(sizes, at::kFloat, like); }
Tensor fresh_image(const Tensor& like) { return at::detail::empty_cuda(like.sizes(), like.scalar_type(), like.device(), kCL); }
Tensor value_of(const c10::optional<Tensor>& o) { return o.has_value() ? *o : Tensor(); }
bool differentiable(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

int64_t wants(const c10::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }

// bf16 or fp32.
void check_float(const char* op, const char* name, const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, op, ": ", name, " is ", t.scalar_type(),
              ", neither bfloat16 nor float32");
}
// A forward-mode derivative, which none of these operators makes: without it the result would read as a derivative of zero.
void refuse_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK(!t.defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), op,
              ": no forward-mode derivative goes through it");
}
void refuse_tangent(const char* op, const c10::optional<Tensor>& t) {
  if (t.has_value()) refuse_tangent(op, *t);
}
template <class... T> void refuse_tangents(const char* op, const T&... tensors) { (refuse_tangent(op, tensors), ...); }
// The last check: what came before it needs no GPU.
void check_gpu(const char* op, const Tensor& t) { TORCH_CHECK(t.is_cuda(), op, ": the input is on ", t.device(), ", not on a GPU"); }

bool capturing(const Tensor& t) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(t.get_device()).stream(), &status) == cudaSuccess &&
         status != cudaStreamCaptureStatusNone;
}
// The capture that the current stream is part of, 0: none.
int64_t capture_of(const Tensor& t) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  return cudaStreamGetCaptureInfo(c10::cuda::getCurrentCUDAStream(t.get_device()).stream(), &status, &id) == cudaSuccess &&
         status != cudaStreamCaptureStatusNone ? (int64_t)id : 0;
}

// A gradient that goes to `t` ends in the node that adds it to t.grad, on the stream that node was made on.  In a capture that has
// to be the capturing stream: a node left by an eager graph that is still alive is on another one, and the engine's waiting for it
// would break the capture off from inside the backward pass.
void check_capture(const char* op, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors) {
    if (!t->defined() || !t->is_leaf() || !t->requires_grad()) continue;
    if (!capturing(*t)) return;
    const auto stream = c10::cuda::getCurrentCUDAStream(t->get_device());
    const auto* meta = torch::autograd::impl::get_autograd_meta(*t);
    const auto node = meta != nullptr ? meta->grad_accumulator_.lock() : nullptr;
    if (!node) continue;
    const auto made = node->stream();
    TORCH_CHECK(!made.has_value() || *made == stream.unwrap(), op, ": a graph from outside the capture still holds a parameter's gradient "
                "on another stream; let go of it (its loss, its outputs) before the capture");
  }
}

// Where a parameter's fp32 gradient goes: the step's accumulator, a new tensor, or nowhere.
struct ParamGrad {
  Sink sink;
  Tensor grad;
  ParamGrad(AutogradContext* ctx, const char* key, bool wanted, at::IntArrayRef shape, const Tensor& like) : sink(load_sink(ctx, key)) {
    if (!sink && wanted) grad = fresh_floats(shape, like);
  }
  float* out() const { return sink ? sink->acc : fptr(grad); }
  int add() const { return sink ? 1 : 0; }
  void done() const {
    if (sink) sink_done(sink);
  }
};

// The gradients of a backward pass that is to be differentiated itself (create_graph): they can be used, and refuse to be differentiated.
// As they come out of the kernels they would read as constants.  The refusal lies on the way to whatever the operator was made of, and
// to the gradients that arrived.
variable_list once(const char* op, const variable_list& arrived, variable_list&& grads) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(arrived);
  if (const auto node = torch::autograd::get_current_node()) edges.insert(edges.end(), node->next_edges().begin(), node->next_edges().end());
  const auto error = std::make_shared<torch::autograd::Error>(c10::str(op, ": there is no second derivative"), std::move(edges));
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    torch::autograd::impl::set_gradient_edge(g, {error, error->add_input_metadata(g)});
  }
  return std::move(grads);
}

// Floats of room for the samples' shares of dgamma and dbeta: 64 MB, which L2 holds between the kernels that write and read them.
constexpr int64_t kShares = 16 << 20;

struct GroupNormFn : public Function<GroupNormFn> {
  using Opt = c10::optional<Tensor>;
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Opt& gamma_in, const Opt& beta_in, const Opt& res_in, int64_t groups,
                        int64_t act, double eps, const Held& gamma, const Held& beta, const Sink& gs, const Sink& bs, const Opt& anchor) {
    Tensor stats;
    const Tensor x = nhwc(x_in), res = res_in.has_value() ? nhwc(*res_in) : Tensor();
    Tensor z = run(x, gamma.t, beta.t, res, groups, act, eps, &stats);
    ctx->save_for_backward({x, act != 0 ? res : Tensor(), gamma.t, beta.t, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["need"] = (int64_t)x_in.requires_grad() | wants(gamma_in) << 1 | wants(beta_in) << 2 | wants(res_in) << 3;
    save_sink(ctx, "g", gs);
    save_sink(ctx, "b", bs);
    return z;
  }
  // stats: also leave the statistics there.
  static Tensor run(const Tensor& x, const Tensor& gamma, const Tensor& beta, const Tensor& res, int64_t groups, int64_t act, double eps,
                    Tensor* stats) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t n = x.size(0), c = x.size(1), rows = x.size(2) * x.size(3);
    Tensor z = fresh_image(x);
    if (stats != nullptr) *stats = fresh_floats({n, groups, 2}, x);
    ck(esgd_group_norm_fwd(ptr(x), ptr(res), mut(z), fptr(gamma), fptr(beta), stats != nullptr ? fptr(*stats) : nullptr,
                           x.scalar_type() == at::kBFloat16, n, rows, (int)c, (int)groups, (int)act, (float)eps, stream_of(x)), "group_norm_act");
    return z;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &res = saved[1], &gamma = saved[2], &beta = saved[3], &stats = saved[4];
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["act"].toInt();
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t n = x.size(0), c = x.size(1), rows = x.size(2) * x.size(3);
    const Tensor dz = nhwc(grads[0]);
    Tensor dx, dres;
    if (need & 1) dx = fresh_image(x);
    if (need & 8) dres = act == 0 ? dz : fresh_image(x);
    const ParamGrad dgamma(ctx, "g", need & 2, {c}, x), dbeta(ctx, "b", need & 4, {c}, x);
    void* st = stream_of(x);
    // Every sample has its share of dgamma and dbeta.  Where those of all would take more room than kShares -- samples of few pixels, whose
    // shares are larger than they are -- the samples are worked on a portion at a time, and the gradients added up in their order.
    const int64_t all = rows > 0 ? n : 0, portion = std::max<int64_t>(1, std::min(all, kShares / (2 * c)));
    const Tensor sums = fresh_floats({std::min(all, portion), 2, c}, x);
    for (int64_t first = 0; first == 0 || first < all; first += portion) {
      const int64_t parts = std::min(portion, all - first), at = first * rows * c * x.element_size();
      auto from = [at](const Tensor& t) -> void* { return t.defined() ? (char*)t.data_ptr() + at : nullptr; };
      ck(esgd_group_norm_bwd(from(x), from(res), from(dz), from(dx), act == 0 ? nullptr : from(dres), fptr(gamma), fptr(beta),
                             fptr(stats) + first * groups * 2, fptr(sums), x.scalar_type() == at::kBFloat16, parts, rows, (int)c, (int)groups,
                             (int)act, st), "group_norm_act backward");
      ck(esgd_sum_parts(fptr(sums), parts, dbeta.out(), c, dbeta.add() || first > 0, dgamma.out(), c, dgamma.add() || first > 0, nullptr, 0, 0,
                        st), "group_norm_act parameter gradients");
    }
    dgamma.done();
    dbeta.done();
    variable_list out(12);
    out[0] = dx; out[1] = dgamma.grad; out[2] = dbeta.grad;
    if (act != 0) out[3] = dres;
    out = once("group_norm_act", grads, std::move(out));
    if (act == 0) out[3] = dres;         // what arrived, with a derivative of its own
    return out;
  }
};

// x [N, C, H, W] bf16 or fp32; gamma, beta fp32 [C]; act: 0 none, 1 ReLU, 2 SiLU.
Tensor group_norm_act(const Tensor& x, int64_t groups, const Tensor& gamma, const Tensor& beta, int64_t act, const c10::optional<Tensor>& res,
                      double eps) {
  TORCH_CHECK(x.dim() == 4, "group_norm_act: takes a 4-D input, not ", x.sizes());
  check_float("group_norm_act", "the input", x);
  const int64_t c = x.size(1);
  TORCH_CHECK(groups >= 1 && c >= 1 && c % groups == 0, "group_norm_act: ", c, " channels do not make ", groups, " groups");
  TORCH_CHECK(c / groups <= esgd_group_norm_max_group(), "group_norm_act: takes up to ", esgd_group_norm_max_group(), " channels a group, not ",
              c / groups);
  TORCH_CHECK(act >= 0 && act <= 2 && eps >= 0, "group_norm_act: no such activation, or an eps below zero");
  // what the grids hold; of fewer channels in all there are not so many CTAs
  TORCH_CHECK(c < ((int64_t)1 << 31) && x.size(2) * x.size(3) < ((int64_t)1 << 30) &&
                  (x.size(0) <= ((int64_t)1 << 27) / c ||
                   esgd_group_norm_fits(x.size(0), x.size(2) * x.size(3), (int)c, (int)groups, x.scalar_type() == at::kBFloat16)),
              "group_norm_act: an input of ", x.sizes(), " is too large");
  check_vector("group_norm_act", "gamma", gamma, x, c);
  check_vector("group_norm_act", "beta", beta, x, c);
  if (res.has_value()) {
    TORCH_CHECK(res->sizes() == x.sizes(), "group_norm_act: the residual ", res->sizes(), " is not of the input's size ", x.sizes());
    check_operand("group_norm_act", "the residual", *res, x, x.scalar_type());
  }
  refuse_tangents("group_norm_act", x, gamma, beta, res);
  check_gpu("group_norm_act", x);
  const Tensor residual = value_of(res);
  if (!differentiable(x) && !differentiable(gamma) && !differentiable(beta) && !differentiable(residual))
    return GroupNormFn::run(nhwc(x), gamma, beta, residual.defined() ? nhwc(residual) : Tensor(), groups, act, eps, nullptr);
  Sink gs = find_sink(gamma), bs = find_sink(beta);
  check_capture("group_norm_act", {&x, gs ? &x : &gamma, bs ? &x : &beta, &residual});
  sink_use(gs);
  sink_use(bs);
  return GroupNormFn::apply(x, graph_only(gamma, gs), graph_only(beta, bs), res, groups, act, eps, Held{gamma}, Held{beta}, gs, bs,
                            anchor_for(x, gs || bs));
}

}  // namespace
