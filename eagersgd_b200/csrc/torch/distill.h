// Distillation from a teacher's top logits as an autograd operator; part of ops.cpp.
#pragma once

extern "C" {
int esgd_distill_max_top();
int esgd_distill(const void* logits, void* grad, int is_bf16, const void* values, int values_bf16, const int64_t* classes_of,
                 const int64_t* labels, int rows, int classes, int ld, int top, float temperature, float hard_weight, float* row_loss,
                 float* loss, void* stream);
int esgd_distill_scale(const void* in, void* out, int is_bf16, const float* factor, int64_t n, void* stream);
}

namespace {

struct DistillFn : public Function<DistillFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Held& values, const Held& classes, const Held& labels,
                        double temperature, double hard_weight) {
    Tensor grad;
    Tensor loss = run(logits, values.t, classes.t, labels.t, temperature, hard_weight, &grad);
    ctx->save_for_backward({grad});
    ctx->saved_data["capture"] = capture_of(logits);
    return loss;
  }
  // grad: also the gradient for a factor of one, rows as far apart as those of the logits where these are the dense layer's padded
  // ones, else dense.
  static Tensor run(const Tensor& logits_in, const Tensor& values_in, const Tensor& classes_in, const Tensor& labels_in, double temperature,
                    double hard_weight, Tensor* grad) {
    c10::cuda::CUDAGuard guard(logits_in.device());
    const int64_t rows = logits_in.size(0), classes = logits_in.size(1), top = values_in.size(1), ld = logits_in.stride(0);
    const Tensor logits = aligned(logits_in.stride(1) == 1 && ld >= classes && ld < classes + 8 ? logits_in : logits_in.contiguous());
    const Tensor values = values_in.contiguous(), named = classes_in.contiguous(), labels = labels_in.defined() ? labels_in.contiguous() : Tensor();
    if (grad != nullptr) *grad = at::empty_strided({rows, classes}, {logits.stride(0), 1}, logits.options());
    Tensor loss = fresh_floats({}, logits);
    const Tensor row_loss = fresh_floats({rows}, logits);
    ck(esgd_distill(ptr(logits), grad != nullptr ? mut(*grad) : nullptr, logits.scalar_type() == at::kBFloat16, ptr(values),
                    values.scalar_type() == at::kBFloat16, named.data_ptr<int64_t>(), labels.defined() ? labels.data_ptr<int64_t>() : nullptr,
                    (int)rows, (int)classes, (int)logits.stride(0), (int)top, (float)temperature, (float)hard_weight, fptr(row_loss), fptr(loss),
                    stream_of(logits)), "distillation_loss");
    return loss;
  }
  // The gradient is there; times the factor that arrives.  Where this is its only use it is scaled where it lies, and the kernel
  // returns at once for a factor of one (loss.backward()).  A graph that is kept gets a product of its own, and so does one whose
  // backward pass is captured without its forward pass, or apart from it: every replay of that alone would scale the buffer once
  // more.  Another factor rounds a bf16 gradient a second time: the price of not reading the logits again.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor grad = ctx->get_saved_variables()[0];
    c10::cuda::CUDAGuard guard(grad.device());
    const Tensor factor = grads[0].to(at::kFloat).contiguous();
    const bool kept = torch::autograd::get_current_graph_task_keep_graph() || ctx->saved_data["capture"].toInt() != capture_of(grad);
    Tensor out = kept ? at::empty_strided(grad.sizes(), grad.strides(), grad.options()) : grad;
    const int64_t n = (grad.size(0) - 1) * grad.stride(0) + grad.size(1);
    ck(esgd_distill_scale(ptr(grad), mut(out), grad.scalar_type() == at::kBFloat16, fptr(factor), n, stream_of(grad)),
       "distillation_loss backward");
    return once("distillation_loss", grads, {out, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// logits [rows, classes] bf16 or fp32; teacher_logits [rows, top] bf16 or fp32, teacher_classes [rows, top] int64; labels [rows] int64.
Tensor distillation_loss(const Tensor& logits, const Tensor& values, const Tensor& classes, double temperature,
                         const c10::optional<Tensor>& labels, double hard_weight) {
  const char* op = "distillation_loss";
  TORCH_CHECK(logits.dim() == 2 && values.dim() == 2, op, ": takes 2-D logits, not ", logits.sizes(), " and ", values.sizes());
  check_float(op, "logits", logits);
  check_float(op, "teacher_logits", values);
  check_operand(op, "teacher_logits", values, logits, values.scalar_type());
  check_operand(op, "teacher_classes", classes, logits, at::kLong);
  TORCH_CHECK(logits.size(0) >= 1 && logits.size(1) >= 1, op, ": there is no mean over logits of ", logits.sizes());
  TORCH_CHECK(values.size(0) == logits.size(0) && classes.sizes() == values.sizes(), op, ": a teacher of ", values.sizes(), " logits and ",
              classes.sizes(), " classes for ", logits.size(0), " rows");
  TORCH_CHECK(values.size(1) <= esgd_distill_max_top(), op, ": takes up to ", esgd_distill_max_top(), " of a teacher's logits, not ", values.size(1));
  TORCH_CHECK(logits.size(0) <= ((int64_t)1 << 27) && logits.size(1) < ((int64_t)1 << 31) - 8, op, ": logits of ", logits.sizes(), " are too many");
  // the kernel has T, 1 / T and T^2 in fp32
  const float t = (float)temperature;
  TORCH_CHECK(t > 0 && std::isnormal(t * t) && hard_weight >= 0 && hard_weight <= 1, op, ": a temperature of ",
              temperature, " and a hard weight of ", hard_weight);
  TORCH_CHECK(!values.requires_grad() || !at::GradMode::is_enabled(), op, ": the teacher's logits get no gradient: detach them");
  if (labels.has_value()) {
    TORCH_CHECK(labels->numel() == logits.size(0), op, ": ", labels->numel(), " labels for ", logits.size(0), " rows");
    check_operand(op, "the labels", *labels, logits, at::kLong);
  }
  TORCH_CHECK(hard_weight == 0 || labels.has_value(), op, ": a hard weight without labels");
  refuse_tangents(op, logits, values);
  check_gpu(op, logits);
  if (!differentiable(logits)) return DistillFn::run(logits, values, classes, value_of(labels), temperature, hard_weight, nullptr);
  check_capture(op, {&logits});
  return DistillFn::apply(logits, Held{values}, Held{classes}, Held{value_of(labels)}, temperature, hard_weight);
}

}  // namespace
