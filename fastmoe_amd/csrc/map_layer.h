// Tokens sorted by expert and back along a map of truth values: the operators, and each as a native
// autograd node whose gradient is the other.  Part of the extension (fmoe_cuda_ext.cpp);
// csrc/mx_layer.h says why such nodes are native.
#pragma once
#include <torch/extension.h>

#include <ATen/core/grad_mode.h>

namespace {

// `sizes` of a tensor's values from `offset` on, as a tensor of its own on the same memory.
Tensor part_of(const Tensor& whole, int64_t offset, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                      whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// (counts int64 [E], seg_off int32 [E + 1], token_off int32 [T + 1], pairs int32 [max_rows, 2])
std::tuple<Tensor, Tensor, Tensor, Tensor> map_plan(Tensor map, int64_t max_rows) {
  dev(map, "routing_map", at::kBool);
  need(map.dim() == 2 && map.size(1) >= 1, "routing_map must be [tokens, experts]");
  need(max_rows >= 0, "max_rows must not be negative");
  c10::DeviceGuard guard(map.device());
  const int64_t t = map.size(0), e = map.size(1);
  const auto ints = map.options().dtype(at::kInt);
  // (one allocation, the host's share of a decode step's plan; what a user may keep, the counts, apart)
  const int64_t at_off = (e + 2) & ~1, at_pairs = at_off + ((t + 2) & ~1);
  Tensor whole = torch::empty({at_pairs + 2 * max_rows}, ints);
  Tensor pairs = part_of(whole, at_pairs, {max_rows, 2});
  if (t == 0)
    return {torch::zeros({e}, map.options().dtype(at::kLong)), torch::zeros({e + 1}, ints),
            torch::zeros({1}, ints), pairs};
  Tensor counts = torch::empty({e}, map.options().dtype(at::kLong));
  Tensor seg = part_of(whole, 0, {e + 1}), off = part_of(whole, at_off, {t + 1});
  need(e <= FMOE_MAP_MAX_EXPERTS, "routing_map has too many experts");
  const int64_t bytes = fmoe_map_workspace_bytes(t, (int32_t)e);
  check(bytes < 0 ? (int)bytes : 0, "map_plan");
  Tensor ws;                           // (few tokens need none)
  if (bytes > 0) ws = workspace_of(bytes, map);
  check(fmoe_map_plan((const uint8_t*)map.data_ptr(), t, (int32_t)e, max_rows,
                      counts.data_ptr<int64_t>(), seg.data_ptr<int32_t>(), off.data_ptr<int32_t>(),
                      pairs.data_ptr<int32_t>(), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                      stream_of(map)),
        "map_plan");
  return {counts, seg, off, pairs};
}

// What both directions check: rows [max_rows, d] and tokens [T, d] against a plan, and the weight.
void map_check(const Tensor& given, const char* name, int64_t count, const OptTensor& weight,
               const Tensor& seg_off, const Tensor& token_off, const Tensor& pairs) {
  dev(given, name);
  dev(seg_off, "seg_off", at::kInt);
  dev(token_off, "token_off", at::kInt);
  dev(pairs, "pairs", at::kInt);
  need(pairs.dim() == 2 && pairs.size(1) == 2 && token_off.numel() >= 1 && seg_off.numel() >= 2,
       "the plan's tensors do not belong together");
  // (texts are put together where they are wanted: a decode step's calls are all host time)
  if (!(given.dim() == 2 && given.size(0) == count && given.size(1) >= 1))
    need(false, std::string(name) + " must be [" + std::to_string(count) + ", features]");
  if (!(given.device() == seg_off.device() && given.device() == token_off.device() &&
        given.device() == pairs.device()))
    need(false, std::string(name) + " and the plan must share a device");
  if (weight.has_value() && weight->defined()) {
    dev(*weight, "weight");
    need(weight->dim() == 2 && weight->size(0) == token_off.numel() - 1 &&
             weight->size(1) == seg_off.numel() - 1 && weight->device() == given.device(),
         "weight must be [tokens, experts] on the plan's device");
    need(weight->scalar_type() == at::kFloat || weight->scalar_type() == given.scalar_type(),
         "weight must be float32 or of the rows' dtype");
  }
}
int weight_dtype(const OptTensor& weight) {
  return weight.has_value() && weight->defined() ? dt(*weight, "weight") : FMOE_F32;
}
const Tensor* defined(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }

// (rows [max_rows, d], unless they are not `wanted`, the weights' gradient if `given` rows are handed
// over)
std::tuple<Tensor, OptTensor> map_expand(Tensor tokens, OptTensor weight, Tensor seg_off,
                                         Tensor token_off, Tensor pairs, OptTensor given, bool clear,
                                         bool wanted = true) {
  map_check(tokens, "tokens", token_off.numel() - 1, weight, seg_off, token_off, pairs);
  OptTensor dw;
  if (const Tensor* g = defined(given)) {
    map_check(*g, "rows", pairs.size(0), weight, seg_off, token_off, pairs);
    need(defined(weight) && g->sizes()[1] == tokens.size(1) && g->scalar_type() == tokens.scalar_type(),
         "a gradient of weights needs them, and rows like the tokens");
  }
  c10::DeviceGuard guard(tokens.device());
  need(wanted || defined(given), "nothing to do without rows and without a gradient of weights");
  Tensor rows;
  if (wanted) rows = torch::empty({pairs.size(0), tokens.size(1)}, tokens.options());
  if (defined(given)) dw = torch::empty_like(*weight);
  if (tokens.size(0) == 0) {
    if (wanted && clear) rows.zero_();
    return {rows, dw};
  }
  check(fmoe_map_expand(tokens.data_ptr(), ptr(given), ptr(weight), token_off.data_ptr<int32_t>(),
                        pairs.data_ptr<int32_t>(),
                        clear ? seg_off.data_ptr<int32_t>() + seg_off.numel() - 1 : nullptr,
                        wanted ? rows.data_ptr() : nullptr, ptr(dw), tokens.size(0), tokens.size(1),
                        (int32_t)(seg_off.numel() - 1), pairs.size(0), dt(tokens, "tokens"),
                        weight_dtype(weight), stream_of(tokens)),
        "map_expand");
  return {rows, dw};
}

// (tokens [T, d], unless they are not `wanted`, the weights' gradient if `given` tokens are handed over)
std::tuple<Tensor, OptTensor> map_reduce(Tensor rows, OptTensor weight, Tensor seg_off,
                                         Tensor token_off, Tensor pairs, OptTensor given,
                                         bool wanted = true) {
  map_check(rows, "rows", pairs.size(0), weight, seg_off, token_off, pairs);
  if (const Tensor* g = defined(given)) {
    map_check(*g, "tokens", token_off.numel() - 1, weight, seg_off, token_off, pairs);
    need(defined(weight) && g->sizes()[1] == rows.size(1) && g->scalar_type() == rows.scalar_type(),
         "a gradient of weights needs them, and tokens like the rows");
  }
  c10::DeviceGuard guard(rows.device());
  need(wanted || defined(given), "nothing to do without tokens and without a gradient of weights");
  const int64_t t = token_off.numel() - 1;
  OptTensor dw;
  Tensor tokens;
  if (wanted) tokens = torch::empty({t, rows.size(1)}, rows.options());
  if (defined(given)) dw = torch::empty_like(*weight);
  if (t == 0) return {tokens, dw};
  check(fmoe_map_reduce(rows.data_ptr(), ptr(given), ptr(weight), token_off.data_ptr<int32_t>(),
                        pairs.data_ptr<int32_t>(), wanted ? tokens.data_ptr() : nullptr, ptr(dw), t,
                        rows.size(1), (int32_t)(seg_off.numel() - 1), pairs.size(0),
                        dt(rows, "rows"), weight_dtype(weight), stream_of(rows)),
        "map_reduce");
  return {tokens, dw};
}

// EXPAND: functions.sort_tokens; otherwise functions.unsort_tokens
template <bool EXPAND> struct MapNode : public torch::autograd::Function<MapNode<EXPAND>> {
  static Tensor run(const Tensor& from, const OptTensor& weight, const Tensor& seg_off,
                    const Tensor& token_off, const Tensor& pairs) {
    return EXPAND ? std::get<0>(map_expand(from, weight, seg_off, token_off, pairs, c10::nullopt, false))
                  : std::get<0>(map_reduce(from, weight, seg_off, token_off, pairs, c10::nullopt));
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& from_in, const Tensor& seg_off,
                        const Tensor& token_off, const Tensor& pairs, const OptTensor& weight_in) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor from = from_in.contiguous();
    OptTensor weight;
    if (defined(weight_in)) weight = weight_in->contiguous();
    const bool dot = weight.has_value() && weight_in->requires_grad();
    ctx->save_for_backward({seg_off, token_off, pairs, weight.has_value() ? *weight : Tensor(),
                            dot ? from : Tensor()});
    return run(from, weight, seg_off, token_off, pairs);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    c10::DeviceGuard guard(v[0].device());
    const Tensor g = only_once(grads[0], EXPAND ? "sort_tokens" : "unsort_tokens");
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const bool wanted = ctx->needs_input_grad(0);
    // (an absent weight is no input of the node; v[4] is there for one that has a gradient alone)
    const OptTensor dot = v[4].defined() && ctx->needs_input_grad(4) ? OptTensor(v[4]) : OptTensor();
    if (!wanted && !dot.has_value()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    auto r = EXPAND ? map_reduce(g, opt(v[3]), v[0], v[1], v[2], dot, wanted)
                    : map_expand(g, opt(v[3]), v[0], v[1], v[2], dot, true, wanted);
    const OptTensor& dw = std::get<1>(r);
    return {std::get<0>(r), Tensor(), Tensor(), Tensor(), dw.has_value() ? *dw : Tensor()};
  }
};

template <bool EXPAND>
Tensor map_move(const Tensor& from, const OptTensor& weight, const Tensor& seg_off,
                const Tensor& token_off, const Tensor& pairs) {
  need(from.is_cuda(), "the input must be a CUDA tensor");
  c10::DeviceGuard guard(from.device());
  if (at::GradMode::is_enabled() &&
      (from.requires_grad() || (defined(weight) && weight->requires_grad())))
    return MapNode<EXPAND>::apply(from, seg_off, token_off, pairs, weight);
  OptTensor w;
  if (defined(weight)) w = weight->contiguous();
  return MapNode<EXPAND>::run(from.contiguous(), w, seg_off, token_off, pairs);
}
Tensor sort_tokens(const Tensor& x, const OptTensor& weight, const Tensor& seg_off,
                   const Tensor& token_off, const Tensor& pairs) {
  return map_move<true>(x, weight, seg_off, token_off, pairs);
}
Tensor unsort_tokens(const Tensor& rows, const OptTensor& weight, const Tensor& seg_off,
                     const Tensor& token_off, const Tensor& pairs) {
  return map_move<false>(rows, weight, seg_off, token_off, pairs);
}

}  // namespace
