// Rows and expert weights in 8-bit integers: the operators, their product as a native autograd node,
// and the whole layer of 8-bit experts without gradients as one call.  Part of the extension
// (fmoe_cuda_ext.cpp); csrc/mx_layer.h says why such nodes are native.
#pragma once
#include <torch/extension.h>

#include <ATen/core/grad_mode.h>

namespace {

int64_t i8_bytes(int64_t features) {
  const int64_t n = fmoe_i8_row_bytes(features);
  check(n < 0 ? (int)n : 0, "i8_row_bytes");
  return n;
}

// codes [rows, row bytes] and scales [rows] of rows of `features` values
std::tuple<Tensor, Tensor> i8_empty(int64_t rows, int64_t features, const Tensor& like) {
  return {torch::empty({rows, i8_bytes(features)}, like.options().dtype(at::kChar)),
          torch::empty({rows}, like.options().dtype(at::kFloat))};
}

void i8_check(const Tensor& codes, const Tensor& scales, int64_t features, const char* name) {
  dev(codes, name, at::kChar);
  dev(scales, name, at::kFloat);
  need(features >= 1, std::string(name) + ": features must be positive");
  need(codes.dim() >= 1 && scales.dim() == codes.dim() - 1 &&
           codes.sizes().slice(0, codes.dim() - 1) == scales.sizes() &&
           codes.size(-1) == i8_bytes(features) && codes.device() == scales.device(),
       std::string(name) + ": codes and scales do not hold rows of that many features");
}

std::tuple<Tensor, Tensor> i8_quantize(Tensor x, OptTensor n_rows_dev) {
  dev(x, "x");
  need(x.dim() == 2 && x.size(1) >= 1, "x must be [rows, features]");
  if (n_rows_dev.has_value() && n_rows_dev->defined()) {
    dev(*n_rows_dev, "n_rows_dev", at::kInt);
    need(n_rows_dev->numel() >= 1 && n_rows_dev->device() == x.device(),
         "n_rows_dev must be an int32 on x's device");
  }
  c10::DeviceGuard guard(x.device());
  auto q = i8_empty(x.size(0), x.size(1), x);
  check(fmoe_i8_quantize(x.data_ptr(), x.size(0), x.size(1), (const int32_t*)ptr(n_rows_dev),
                         std::get<0>(q).data_ptr(), std::get<1>(q).data_ptr<float>(), dt(x, "x"),
                         stream_of(x)),
        "i8_quantize");
  return q;
}

// i8_quantize and, in the same launch, the segment table of the rows' device counts (of none: all
// rows are one expert's)
std::tuple<Tensor, Tensor, Tensor> i8_quantize_counted(Tensor x, OptTensor expert_count) {
  dev(x, "x");
  need(x.dim() == 2 && x.size(1) >= 1, "x must be [rows, features]");
  const bool counted = expert_count.has_value() && expert_count->defined();
  if (counted) {
    dev(*expert_count, "expert_count", at::kLong);
    need(expert_count->numel() >= 1 && expert_count->device() == x.device(),
         "expert_count must lie on x's device");
  }
  const int64_t e = counted ? expert_count->numel() : 1;
  c10::DeviceGuard guard(x.device());
  auto q = i8_empty(x.size(0), x.size(1), x);
  Tensor seg = torch::empty({e + 1}, x.options().dtype(at::kInt));
  check(fmoe_i8_quantize_counted(x.data_ptr(), x.size(0), x.size(1), (const int64_t*)ptr(expert_count),
                                 e, seg.data_ptr<int32_t>(), std::get<0>(q).data_ptr(),
                                 std::get<1>(q).data_ptr<float>(), dt(x, "x"), stream_of(x)),
        "i8_quantize_counted");
  return {std::get<0>(q), std::get<1>(q), seg};
}

std::tuple<Tensor, Tensor> i8_quantize_tokens(Tensor x, Tensor inv, int64_t top_k) {
  dev(x, "x");
  dev(inv, "inv", at::kInt);
  need(x.dim() == 2 && x.size(1) >= 1, "x must be [tokens, features]");
  need(top_k >= 1 && inv.numel() == x.size(0) * top_k && inv.device() == x.device(),
       "inv must have tokens * top_k entries on x's device");
  c10::DeviceGuard guard(x.device());
  auto q = i8_empty(x.size(0) * top_k, x.size(1), x);
  check(fmoe_i8_quantize_tokens(x.data_ptr(), inv.data_ptr<int32_t>(), x.size(0), top_k, x.size(1),
                                std::get<0>(q).data_ptr(), std::get<1>(q).data_ptr<float>(),
                                dt(x, "x"), stream_of(x)),
        "i8_quantize_tokens");
  return q;
}

Tensor i8_dequantize(Tensor codes, Tensor scales, Tensor out) {
  dev(out, "out");
  need(out.dim() == 2 && out.size(1) >= 1, "out must be [rows, features]");
  i8_check(codes, scales, out.size(1), "i8_dequantize");
  need(codes.dim() == 2 && codes.size(0) == out.size(0) && codes.device() == out.device(),
       "i8_dequantize: out has other rows");
  c10::DeviceGuard guard(out.device());
  check(fmoe_i8_dequantize(codes.data_ptr(), scales.data_ptr<float>(), out.size(0), out.size(1),
                           out.data_ptr(), dt(out, "out"), stream_of(out)),
        "i8_dequantize");
  return out;
}

Tensor i8_linear_fwd(Tensor xc, Tensor xs, Tensor wc, Tensor ws, int64_t in_f, OptTensor bias,
                     Tensor seg_off, Tensor out) {
  i8_check(xc, xs, in_f, "x");
  i8_check(wc, ws, in_f, "weight");
  dev(seg_off, "seg_off", at::kInt);
  dev(out, "out");
  need(xc.dim() == 2 && wc.dim() == 3, "x must be 2-d and weight 3-d");
  need(xc.device() == wc.device() && xc.device() == seg_off.device() && xc.device() == out.device(),
       "x, weight, seg_off and out must share a device");
  need(seg_off.numel() == wc.size(0) + 1, "seg_off must have E+1 entries");
  need(out.dim() == 2 && out.size(0) == xc.size(0) && out.size(1) == wc.size(1),
       "out must be [rows, out]");
  if (bias.has_value() && bias->defined()) {
    dev(*bias, "bias", out.scalar_type());
    need(bias->dim() == 2 && bias->size(0) == wc.size(0) && bias->size(1) == wc.size(1) &&
             bias->device() == out.device(),
         "bias must be [E, out]");
  }
  c10::DeviceGuard guard(out.device());
  check(fmoe_i8_linear_fwd(xc.data_ptr(), xs.data_ptr<float>(), wc.data_ptr(), ws.data_ptr<float>(),
                           ptr(bias), seg_off.data_ptr<int32_t>(), out.data_ptr(), xc.size(0), in_f,
                           wc.size(1), wc.size(0), dt(out, "out"), stream_of(out)),
        "i8_linear_fwd");
  return out;
}

// Gradients of the rows and of the bias in front of frozen 8-bit weights, the former by the faster of
// two ways (csrc/i8_grad.hip).  Rows that no expert owns get zeros.
std::tuple<OptTensor, OptTensor> i8_linear_bwd(Tensor dy, Tensor seg_off, Tensor wc, Tensor ws,
                                               int64_t in_f, bool need_dx, bool need_bias) {
  dev(dy, "dy");
  i8_check(wc, ws, in_f, "weight");
  dev(seg_off, "seg_off", at::kInt);
  need(dy.dim() == 2 && wc.dim() == 3 && dy.size(1) == wc.size(1), "dy must be [rows, out]");
  need(dy.device() == wc.device() && dy.device() == seg_off.device(),
       "dy, weight and seg_off must share a device");
  need(seg_off.numel() == wc.size(0) + 1, "seg_off must have E+1 entries");
  c10::DeviceGuard guard(dy.device());
  const int64_t e = wc.size(0), out_f = wc.size(1);
  const int64_t rows = dy.size(0);
  const int type = dt(dy, "dy");
  OptTensor dx, db;
  if (need_dx) {
    const bool few = fmoe_i8_few_rows(rows, e, type);
    const int64_t bytes = few ? fmoe_i8_dx_workspace_bytes(rows, in_f, out_f, e, type)
                              : fmoe_i8_dx_many_workspace_bytes(rows, in_f, out_f, e, type);
    check(bytes < 0 ? (int)bytes : 0, "i8_linear_dx");
    dx = torch::empty({rows, in_f}, dy.options());
    // (a tensor of its own: a backward pass does not hold the interpreter lock)
    Tensor work = torch::empty({bytes}, dy.options().dtype(at::kByte));
    check((few ? fmoe_i8_linear_dx : fmoe_i8_linear_dx_many)(
              dy.data_ptr(), wc.data_ptr(), ws.data_ptr<float>(), seg_off.data_ptr<int32_t>(),
              dx->data_ptr(), rows, in_f, out_f, e, work.data_ptr(), bytes, type, stream_of(dy)),
          "i8_linear_dx");
  }
  if (need_bias) {   // (the weights and the layer's input have no part in it)
    db = torch::empty({e, out_f}, dy.options());
    check(fmoe_grouped_linear_bwd(dy.data_ptr(), dy.data_ptr(), nullptr, seg_off.data_ptr<int32_t>(),
                                  nullptr, nullptr, db->data_ptr(), rows, in_f, out_f, e, type,
                                  stream_of(dy)),
          "i8_linear_bwd");
  }
  return {dx, db};
}

// i8.quantize: x [..., features], codes and scales with its leading dimensions
std::tuple<Tensor, Tensor> i8_quantize_rows(const Tensor& x) {
  at::AutoDispatchBelowADInplaceOrView below;
  need(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1, "x must be a CUDA tensor [..., features]");
  auto q = i8_quantize(x.reshape({-1, x.size(-1)}).contiguous(), c10::nullopt);
  if (x.dim() == 2) return q;
  auto sizes = x.sizes().vec();
  sizes.back() = std::get<0>(q).size(1);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  return {std::get<0>(q).view(sizes), std::get<1>(q).view(lead)};
}

// I8Tensor.dequantize
Tensor i8_dequantize_rows(const Tensor& codes, const Tensor& scales, int64_t features,
                          at::ScalarType dtype) {
  i8_check(codes, scales, features, "i8_dequantize");
  c10::DeviceGuard guard(codes.device());
  auto sizes = codes.sizes().vec();
  sizes.back() = features;
  Tensor out = torch::empty(sizes, codes.options().dtype(dtype));
  if (out.numel() == 0) return out;
  check(fmoe_i8_dequantize(codes.data_ptr(), scales.data_ptr<float>(), out.numel() / features,
                           features, out.data_ptr(), dt(out, "out"), stream_of(out)),
        "i8_dequantize");
  return out;
}

// x in 8 bits and the segment table of `counts` (int64 row counts on x's device or on the host, or
// none), unless that is at hand: then rows behind its end, those of dropped slots, are left out.
struct I8Rows {
  Tensor codes, scales, seg;
  I8Rows(const Tensor& x, const OptTensor& counts_or_seg) {
    const bool given = counts_or_seg.has_value() && counts_or_seg->defined();
    const bool counts = given && counts_or_seg->scalar_type() == at::kLong;
    if (!given || (counts && counts_or_seg->is_cuda())) {
      auto q = i8_quantize_counted(x, given ? OptTensor(counts_or_seg->contiguous()) : OptTensor());
      std::tie(codes, scales, seg) = q;
      return;
    }
    seg = counts ? seg_off_from_counts(*counts_or_seg, x, x.size(0)) : *counts_or_seg;
    OptTensor live;
    if (!counts && seg.dim() == 1 && seg.numel() > 0) live = seg.narrow(0, seg.numel() - 1, 1);
    std::tie(codes, scales) = i8_quantize(x, live);
  }
};

struct I8LinearNode : public torch::autograd::Function<I8LinearNode> {
  static Tensor run(const Tensor& x, const I8Rows& rows, const Tensor& wc, const Tensor& ws,
                    const OptTensor& bias) {
    Tensor y = torch::empty({x.size(0), wc.size(1)}, x.options());
    return i8_linear_fwd(rows.codes, rows.scales, wc, ws, x.size(1), bias, rows.seg, y);
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& counts_or_seg,
                        const Tensor& wc, const Tensor& ws, const OptTensor& bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    const I8Rows rows(x.contiguous(), counts_or_seg);
    ctx->save_for_backward({rows.seg, wc, ws});
    ctx->saved_data["in"] = x.size(1);
    // (absent tensors are no inputs of the node)
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["counts"] = counts_or_seg.has_value() && counts_or_seg->defined();
    return run(x, rows, wc, ws, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    c10::DeviceGuard guard(v[0].device());
    const int at_bias = ctx->saved_data["counts"].toBool() ? 4 : 3;
    auto r = i8_linear_bwd(only_once(grads[0], "i8.linear"), v[0], v[1], v[2],
                           ctx->saved_data["in"].toInt(), ctx->needs_input_grad(0),
                           ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(at_bias));
    auto got = [](const OptTensor& t) { return t.has_value() ? *t : Tensor(); };
    return {got(std::get<0>(r)), Tensor(), Tensor(), Tensor(), got(std::get<1>(r))};
  }
};

// i8.linear: weight [E, out, in]; without counts all rows are one expert's
Tensor i8_linear(const Tensor& x, const OptTensor& counts_or_seg, const Tensor& wc, const Tensor& ws,
                 int64_t in_f, const OptTensor& bias) {
  need(x.is_cuda() && x.dim() == 2 && x.size(1) == in_f,
       "x must be a CUDA tensor [rows, " + std::to_string(in_f) + "]");
  need(wc.dim() == 3, "the weight must be [E, out, in]");
  const bool given = counts_or_seg.has_value() && counts_or_seg->defined();
  need(given || wc.size(0) == 1, "the rows of several experts need counts");
  c10::DeviceGuard guard(x.device());
  OptTensor b;
  if (bias.has_value() && bias->defined()) b = bias->contiguous();
  if (at::GradMode::is_enabled() && (x.requires_grad() || (b.has_value() && b->requires_grad())))
    return I8LinearNode::apply(x, given ? counts_or_seg : OptTensor(), wc, ws, b);
  const Tensor rows = x.contiguous();
  return I8LinearNode::run(rows, I8Rows(rows, counts_or_seg), wc, ws, b);
}

// i8.expert_layer without gradients, for an activation the library has: gate_idx and score
// [tokens, top_k].  The hidden layer is rounded to x's type in front of its quantisation, as in the
// chain of single operators, whose bits these are.
Tensor i8_expert_layer(const Tensor& x_in, const Tensor& gate_idx, const Tensor& score_in,
                       const Tensor& w1c, const Tensor& w1s, int64_t in_f, const OptTensor& b1,
                       const Tensor& w2c, const Tensor& w2s, int64_t hidden, const OptTensor& b2,
                       int64_t act) {
  at::AutoDispatchBelowADInplaceOrView below;
  need(x_in.is_cuda() && x_in.dim() == 2, "x must be a 2-d CUDA tensor");
  need(gate_idx.dim() == 2 && gate_idx.size(0) == x_in.size(0), "gate_idx must be [tokens, top_k]");
  need(score_in.numel() == gate_idx.numel(), "score must be [tokens, top_k]");
  need(w1c.dim() == 3 && w2c.dim() == 3 && w1c.size(0) == w2c.size(0) && w1c.size(1) == hidden,
       "w1 must be [E, hidden, in] and w2 [E, out, hidden]");
  need(act == FMOE_ACT_GELU || act == FMOE_ACT_RELU, "unknown activation");
  c10::DeviceGuard guard(x_in.device());
  const Tensor x = x_in.contiguous();
  const int64_t t = x.size(0), k = gate_idx.size(1);
  auto bias = [&](const OptTensor& b) {
    return b.has_value() && b->defined() ? OptTensor(b->to(x.scalar_type()).contiguous()) : OptTensor();
  };
  auto r = route(gate_idx.contiguous(), w1c.size(0), true);
  const Tensor &seg = std::get<2>(r), &inv = *std::get<3>(r);
  const Tensor live = seg.narrow(0, seg.numel() - 1, 1);
  auto q = i8_quantize_tokens(x, inv, k);
  Tensor h = torch::empty({t * k, hidden}, x.options());
  i8_linear_fwd(std::get<0>(q), std::get<1>(q), w1c, w1s, in_f, bias(b1), seg, h);
  h = act == FMOE_ACT_GELU ? gelu_fwd(h, live) : h.relu_();
  q = i8_quantize(h, live);
  Tensor y = torch::empty({t * k, w2c.size(1)}, x.options());
  i8_linear_fwd(std::get<0>(q), std::get<1>(q), w2c, w2s, hidden, bias(b2), seg, y);
  return gather_combine_fwd(y, inv, score_in.reshape({t, k}).contiguous().to(x.scalar_type()), t, k);
}

}  // namespace
