// Scored routing and the 4-bit products as native autograd nodes, and the whole layer of 4-bit
// experts as one call: route -> quantise into expert order -> linear + activation + quantisation
// -> linear -> combine.  Part of the extension (fmoe_cuda_ext.cpp), on the operators there.
//
// Why native: these calls are a few microseconds of GPU work each (64 tokens: 4.8 us for the
// router), and a torch.autograd.Function in Python costs the host 40 us more than its kernels.
#pragma once
#include <torch/extension.h>

#include <ATen/core/grad_mode.h>

namespace {

// The operators here have no second derivative; a backward that is itself to be differentiated,
// or that runs for a batch of gradients at once (torch's vmap), is refused.
Tensor only_once(const Tensor& grad, const char* what) {
  need(!at::GradMode::is_enabled() && grad.has_storage(),
       std::string(what) + ": the gradient is that of one backward pass, and cannot be "
                           "differentiated again");
  return grad.contiguous();
}

struct ScoreTopkNode : public torch::autograd::Function<ScoreTopkNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& bias,
                               int64_t top_k, int64_t n_group, int64_t top_group,
                               int64_t group_best, int64_t score, bool renormalize, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor l = logits.contiguous();
    auto r = score_topk_fwd(l, bias, top_k, n_group, top_group, group_best, score, renormalize,
                            scale);
    ctx->save_for_backward({l, std::get<0>(r)});
    ctx->saved_data["args"] = std::vector<int64_t>{score, renormalize};
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({std::get<0>(r)});
    ctx->set_materialize_grads(false);
    return {std::get<0>(r), std::get<1>(r)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(9);
    if (!grads[1].defined()) return none;
    const variable_list v = ctx->get_saved_variables();
    c10::DeviceGuard guard(v[0].device());
    const auto args = ctx->saved_data["args"].toIntVector();
    none[0] = score_topk_bwd(only_once(grads[1], "score_topk"), v[0], v[1], args[0], args[1] != 0,
                             ctx->saved_data["scale"].toDouble());
    return none;
  }
};

// functions.score_topk: logits [..., E]
std::tuple<Tensor, Tensor> score_topk(const Tensor& logits, const OptTensor& bias, int64_t top_k,
                                      int64_t n_group, int64_t top_group, int64_t group_best,
                                      int64_t score, bool renormalize, double scale) {
  need(logits.is_cuda() && logits.dim() >= 1, "logits must be a CUDA tensor");
  c10::DeviceGuard guard(logits.device());
  const Tensor flat = logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)});
  OptTensor b;
  if (bias.has_value() && bias->defined()) b = bias->detach().to(at::kFloat).contiguous();
  variable_list r = ScoreTopkNode::apply(flat, b, top_k, n_group, top_group, group_best, score,
                                         renormalize, scale);
  return {r[0], r[1]};
}

// mx.quantize: x [..., features], codes and scales with its leading dimensions
std::tuple<Tensor, Tensor> mx_quantize_rows(const Tensor& x) {
  at::AutoDispatchBelowADInplaceOrView below;
  need(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1, "x must be a CUDA tensor [..., features]");
  if (x.dim() == 2) return mx_quantize(x.contiguous(), c10::nullopt);
  auto q = mx_quantize(x.reshape({-1, x.size(-1)}).contiguous(), c10::nullopt);
  auto shaped = [&](const Tensor& t) {
    auto sizes = x.sizes().vec();
    sizes.back() = t.size(1);
    return t.view(sizes);
  };
  return {shaped(std::get<0>(q)), shaped(std::get<1>(q))};
}

// MXTensor.dequantize
Tensor mx_dequantize_rows(const Tensor& codes, const Tensor& scales, int64_t features,
                          at::ScalarType dtype) {
  mx_check(codes, scales, features, "mx_dequantize");
  c10::DeviceGuard guard(codes.device());
  auto sizes = codes.sizes().vec();
  sizes.back() = features;
  Tensor out = torch::empty(sizes, codes.options().dtype(dtype));
  if (out.numel() == 0) return out;
  check(fmoe_mx_dequantize(codes.data_ptr(), scales.data_ptr(), out.numel() / features, features,
                           out.data_ptr(), dt(out, "out"), stream_of(out)),
        "mx_dequantize");
  return out;
}

// x in MXFP4 and the segment table of `counts` (int64 row counts on x's device, or on the host),
// unless that is at hand: then rows behind its end, those of dropped slots, are left out.
struct MxRows {
  Tensor codes, scales, seg;
  MxRows(const Tensor& x, const Tensor& counts_or_seg) {
    const bool counts = counts_or_seg.scalar_type() == at::kLong;
    if (counts && counts_or_seg.is_cuda()) {
      auto q = mx_quantize_counted(x, counts_or_seg.contiguous());
      std::tie(codes, scales, seg) = q;
      return;
    }
    seg = counts ? seg_off_from_counts(counts_or_seg, x, x.size(0)) : counts_or_seg;
    OptTensor live;
    if (!counts && seg.dim() == 1 && seg.numel() > 0) live = seg.narrow(0, seg.numel() - 1, 1);
    std::tie(codes, scales) = mx_quantize(x, live);
  }
};

struct MxLinearNode : public torch::autograd::Function<MxLinearNode> {
  static Tensor run(const Tensor& x, const MxRows& rows, const Tensor& wc, const Tensor& ws,
                    const OptTensor& bias) {
    Tensor y = torch::empty({x.size(0), wc.size(1)}, x.options());
    return mx_linear_fwd(rows.codes, rows.scales, wc, ws, x.size(1), bias, rows.seg, y);
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& counts_or_seg,
                        const Tensor& wc, const Tensor& ws, const OptTensor& bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    const MxRows rows(x.contiguous(), counts_or_seg);
    ctx->save_for_backward({rows.seg, wc, ws});
    ctx->saved_data["in"] = x.size(1);
    ctx->saved_data["bias"] = bias.has_value();   // (an absent one is no input of the node)
    return run(x, rows, wc, ws, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    c10::DeviceGuard guard(v[0].device());
    auto r = mx_linear_bwd(only_once(grads[0], "mx.linear"), v[0], v[1], v[2],
                           ctx->saved_data["in"].toInt(), ctx->needs_input_grad(0),
                           ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(4));
    auto got = [](const OptTensor& t) { return t.has_value() ? *t : Tensor(); };
    return {got(std::get<0>(r)), Tensor(), Tensor(), Tensor(), got(std::get<1>(r))};
  }
};

// mx.linear
Tensor mx_linear(const Tensor& x, const Tensor& counts_or_seg, const Tensor& wc, const Tensor& ws,
                 int64_t in_f, const OptTensor& bias) {
  need(x.is_cuda() && x.dim() == 2 && x.size(1) == in_f,
       "x must be a CUDA tensor [rows, " + std::to_string(in_f) + "]");
  need(wc.dim() == 3, "the weight must be [E, out, in]");
  c10::DeviceGuard guard(x.device());
  OptTensor b;
  if (bias.has_value() && bias->defined()) b = bias->contiguous();
  if (at::GradMode::is_enabled() && (x.requires_grad() || (b.has_value() && b->requires_grad())))
    return MxLinearNode::apply(x, counts_or_seg, wc, ws, b);
  const Tensor rows = x.contiguous();
  return MxLinearNode::run(rows, MxRows(rows, counts_or_seg), wc, ws, b);
}

// mx.expert_layer without gradients, for an activation the library has: gate_idx and score
// [tokens, top_k]
Tensor mx_expert_layer(const Tensor& x_in, const Tensor& gate_idx, const Tensor& score_in,
                       const Tensor& w1c, const Tensor& w1s, int64_t in_f, const OptTensor& b1,
                       const Tensor& w2c, const Tensor& w2s, int64_t hidden, const OptTensor& b2,
                       int64_t act) {
  at::AutoDispatchBelowADInplaceOrView below;
  need(x_in.is_cuda() && x_in.dim() == 2, "x must be a 2-d CUDA tensor");
  need(gate_idx.dim() == 2 && gate_idx.size(0) == x_in.size(0), "gate_idx must be [tokens, top_k]");
  need(score_in.numel() == gate_idx.numel(), "score must be [tokens, top_k]");
  need(w1c.dim() == 3 && w2c.dim() == 3 && w1c.size(0) == w2c.size(0) && w1c.size(1) == hidden,
       "w1 must be [E, hidden, in] and w2 [E, out, hidden]");
  c10::DeviceGuard guard(x_in.device());
  const Tensor x = x_in.contiguous();
  const int64_t t = x.size(0), k = gate_idx.size(1);
  auto contiguous = [](const OptTensor& b) {
    return b.has_value() && b->defined() ? OptTensor(b->contiguous()) : OptTensor();
  };
  auto r = route(gate_idx.contiguous(), w1c.size(0), true);
  const Tensor &seg = std::get<2>(r), &inv = *std::get<3>(r);
  auto q = mx_quantize_tokens(x, inv, k);
  auto h = mx_linear_act_fwd(std::get<0>(q), std::get<1>(q), w1c, w1s, in_f, contiguous(b1), seg, act);
  // The experts' rows have x's type on their way to the combine, as those of the 16-bit experts
  // do.  Kept in f32 the result's error against 64 bits would be one rounding's, not 1.4 times
  // that; 8192 tokens x top-2 of 1024 features in f16 would take 9 us more of 155 (product 53 ->
  // 54, combine 8 -> 16), 2047 x top-8 of 2048 in bf16 14 of 181 (63 -> 67, 12 -> 22).
  Tensor y = torch::empty({t * k, w2c.size(1)}, x.options());
  mx_linear_fwd(std::get<0>(h), std::get<1>(h), w2c, w2s, hidden, contiguous(b2), seg, y);
  return gather_combine_fwd(y, inv, score_in.reshape({t, k}).contiguous().to(x.scalar_type()), t, k);
}

}  // namespace
