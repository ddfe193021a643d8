r"""Experts with 4-bit weights: rows in microscaled floating point (MXFP4 of the OCP
Microscaling Formats specification), their products on the matrix cores, and an expert
module for `FMoE` layers that holds nothing else.

A block of 32 features shares a power of two (one byte, exponent + 127; 255 is NaN), every
value is a 4-bit E2M1 code (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign).  Weights are quantised
once and stay frozen; rows of activations are quantised on the way into a product, their
gradient passes straight through that rounding.

The reference has no such experts; they stand in the place of the fused `_Expert` of
fmoe/transformer.py:11-31.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.nn.modules.module import _has_any_global_hook

from . import fmoe_cuda
from .functions import (FusedGatherCombine, FusedScatter, RoutePlan, SegmentTable,
                        apply_activation)
from .linear import FMoELinear, _segments, is_exact_gelu, native_act
from .transformer import _Expert, _watched

BLOCK = 32      # features that share a scale


class MXTensor:
    r"""Rows of `features` values in MXFP4: `codes` uint8 [..., rows, 64 ceil(features / 128)],
    the even feature of a pair in the low half of its byte, and `scales` uint8
    [..., rows, 16 ceil(features / 512)].  Codes behind the last feature are zero."""

    __slots__ = ("codes", "scales", "features")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, features: int):
        self.codes, self.scales, self.features = codes, scales, int(features)

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.features))

    @property
    def device(self):
        return self.codes.device

    def to(self, device) -> "MXTensor":
        return MXTensor(self.codes.to(device), self.scales.to(device), self.features)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        r"""The values [..., rows, features] as `dtype` (float32, float16 or bfloat16)."""
        native = fmoe_cuda.native()
        if native is not None:
            return native.mx_dequantize_rows(self.codes.contiguous(), self.scales.contiguous(),
                                             self.features, dtype)
        return _Dequantize.apply(self.codes, self.scales, self.features, dtype)

    @classmethod
    def from_blocks(cls, codes: torch.Tensor, scales: torch.Tensor) -> "MXTensor":
        r"""From the tight layout of MXFP4 checkpoints: codes uint8 [..., rows, K / 2] and
        scales uint8 [..., rows, K / 32], K a multiple of 32."""
        k = 2 * codes.shape[-1]
        if (k % BLOCK or k == 0 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8
                or scales.shape != (*codes.shape[:-1], k // BLOCK)):
            raise ValueError("codes must be uint8 [..., K / 2] and scales uint8 [..., K / 32]")
        pad = nn.functional.pad
        return cls(pad(codes, (0, -(-k // 128) * 64 - codes.shape[-1])),
                   pad(scales, (0, -(-k // 512) * 16 - scales.shape[-1])), k)


# Where the extension's own nodes do not apply (fmoe_cuda.native()), somebody may be looking at
# torch operations: tracing records these functions where an operator called directly would leave
# the example's results behind as constants, and forward-mode differentiation is refused by them
# where such an operator would drop the tangents.
class _Quantize(Function):
    @staticmethod
    def forward(ctx, x):
        k = x.shape[-1]
        codes, scales = fmoe_cuda.mx_quantize(x.reshape(-1, k).contiguous())
        codes = codes.view(*x.shape[:-1], codes.shape[-1])
        scales = scales.view(*x.shape[:-1], scales.shape[-1])
        ctx.mark_non_differentiable(codes, scales)
        return codes, scales

    @staticmethod
    def backward(ctx, *_grads):
        return None


class _Dequantize(Function):
    @staticmethod
    def forward(ctx, codes, scales, features, dtype):
        out = torch.empty((*codes.shape[:-1], features), dtype=dtype, device=codes.device)
        if out.numel():
            fmoe_cuda.mx_dequantize(codes.reshape(-1, codes.shape[-1]).contiguous(),
                                    scales.reshape(-1, scales.shape[-1]).contiguous(),
                                    out.view(-1, features))
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, _grad):
        return None, None, None, None


def quantize(x: torch.Tensor) -> MXTensor:
    r"""x [..., features] (float32, float16 or bfloat16, on the GPU) in MXFP4.  The scale of a
    block is 2^(floor(log2(max |x|)) - 2); values are rounded to nearest, ties to the even
    code, and saturate at 6 times the scale.  A block with an infinity or a NaN is NaN."""
    k = x.shape[-1]
    native = fmoe_cuda.native()
    if native is not None:
        return MXTensor(*native.mx_quantize_rows(x), k)
    return MXTensor(*_Quantize.apply(x.detach()), k)


class MXLinear(Function):
    r"""All experts' linear maps on 4-bit weights in one grouped product; the gradient of the
    rows is that of the weights' values, straight through the rounding of the rows."""

    @staticmethod
    def forward(ctx, x, counts, w_codes, w_scales, bias):
        r"""`counts`: a SegmentTable, int64 counts on the host or on the device, or the segment
        bounds themselves (int32 on the device)."""
        in_feat = x.shape[1]
        x = x.contiguous()
        bias = None if bias is None else bias.contiguous()
        on_device = isinstance(counts, torch.Tensor) and counts.is_cuda
        if on_device and counts.dtype == torch.int64:
            codes, scales, seg_off = fmoe_cuda.mx_quantize_counted(x, counts.contiguous())
        else:
            if isinstance(counts, torch.Tensor) and not on_device and (
                    bool((counts < 0).any()) or int(counts.sum()) > x.shape[0]):
                raise RuntimeError("expert counts are negative or claim more rows than x holds")
            seg_off = counts.contiguous() if on_device else _segments(counts, x.device)
            # (rows behind a segment table's end, those of dropped slots, are left out)
            host = isinstance(counts, torch.Tensor) and not on_device
            codes, scales = fmoe_cuda.mx_quantize(x, None if host else seg_off[-1:])
        out = torch.empty((x.shape[0], w_codes.shape[1]), dtype=x.dtype, device=x.device)
        fmoe_cuda.mx_linear_fwd(codes, scales, w_codes, w_scales, in_feat, bias, seg_off, out)
        ctx.in_feat = in_feat
        ctx.save_for_backward(seg_off, w_codes, w_scales)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        seg_off, w_codes, w_scales = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, db = fmoe_cuda.mx_linear_bwd(grad_out.contiguous(), seg_off, w_codes, w_scales,
                                         ctx.in_feat, need[0], need[4])
        return dx, None, None, None, db


def linear(x: torch.Tensor, fwd_expert_count, weight: MXTensor, bias=None) -> torch.Tensor:
    r"""y[rows of e] = x[rows of e] @ weight[e].T + bias[e]: the grouped linear layer of
    `FMoELinear` with 4-bit weights [E, out, in].  x [rows, in] holds the rows in expert
    order and is quantised on the way; `fwd_expert_count` is an int64 tensor of row counts
    (host or device) or a SegmentTable; bias [E, out] has x's dtype, as has the result.  Rows of
    x that the counts do not cover are in no product: their rows of y are left as they were
    allocated, their gradient is zero."""
    native = fmoe_cuda.native()
    if native is not None:
        segments = (fwd_expert_count.seg_off if isinstance(fwd_expert_count, SegmentTable)
                    else fwd_expert_count)
        return native.mx_linear(x, segments, weight.codes, weight.scales, weight.features, bias)
    if isinstance(fwd_expert_count, SegmentTable) and torch._C._get_tracing_state() is not None:
        raise RuntimeError("a SegmentTable would be a constant of the trace: trace the layer or "
                           "mx.expert_layer, or hand over counts")
    if x.dim() != 2 or x.shape[1] != weight.features or not x.is_cuda:
        raise RuntimeError(f"x must be a CUDA tensor [rows, {weight.features}]")
    return MXLinear.apply(x, fwd_expert_count, weight.codes, weight.scales, bias)


def _activate(activation, x, n_rows_dev):
    r"""`activation(x)`, called as the module it is where somebody watches it."""
    return activation(x) if _watched(activation) else apply_activation(activation, x, n_rows_dev)


def _as(x, bias):
    return x if bias is None else x.type_as(bias)


class _Route(Function):
    r"""fmoe_cuda.route as an operation that tracing records."""

    @staticmethod
    def forward(ctx, gate_idx, n_expert):
        routed = fmoe_cuda.route(gate_idx.contiguous(), n_expert)
        ctx.mark_non_differentiable(*routed)
        return tuple(routed)

    @staticmethod
    def backward(ctx, *_grads):
        return None, None


class _Scatter(Function):
    r"""FusedScatter on the tensors of its plan, for tracing (a plan would be a constant)."""

    @staticmethod
    def forward(ctx, x, gate_idx, n_expert, *routed):
        return FusedScatter.forward(ctx, x, RoutePlan(gate_idx, n_expert, routed))

    @staticmethod
    def backward(ctx, grad_buf):
        return (FusedScatter.backward(ctx, grad_buf)[0],) + (None,) * 6


class _Combine(Function):
    r"""FusedGatherCombine on the tensors of its plan, for tracing."""

    @staticmethod
    def forward(ctx, buf, score, gate_idx, n_expert, *routed):
        return FusedGatherCombine.forward(ctx, buf, score, RoutePlan(gate_idx, n_expert, routed))

    @staticmethod
    def backward(ctx, grad_y):
        return FusedGatherCombine.backward(ctx, grad_y)[:2] + (None,) * 6


class MXExpertLayer(Function):
    r"""The layer without gradients (see expert_layer) operator by operator."""

    @staticmethod
    def forward(ctx, x, gate_idx, score, w1_codes, w1_scales, in_feat, b1, w2_codes, w2_scales,
                hidden, b2, act):
        n_tokens, top_k = gate_idx.shape
        x = x.contiguous()
        _pos, _counts, seg_off, inv = fmoe_cuda.route(gate_idx.contiguous(), w1_codes.shape[0])
        codes, scales = fmoe_cuda.mx_quantize_tokens(x, inv, top_k)
        codes, scales = fmoe_cuda.mx_linear_act_fwd(
            codes, scales, w1_codes, w1_scales, in_feat, None if b1 is None else b1.contiguous(),
            seg_off, act)
        # (in x's dtype, not in f32: csrc/mx_layer.h says why)
        out = torch.empty((n_tokens * top_k, w2_codes.shape[1]), dtype=x.dtype, device=x.device)
        fmoe_cuda.mx_linear_fwd(codes, scales, w2_codes, w2_scales, hidden,
                                None if b2 is None else b2.contiguous(), seg_off, out)
        score = score.reshape(n_tokens, top_k).contiguous().to(x.dtype)
        return fmoe_cuda.gather_combine_fwd(out, inv, score, n_tokens, top_k)

    @staticmethod
    def backward(ctx, _grad):
        raise RuntimeError("mx.expert_layer was called (or traced) without gradients")


def expert_layer(x: torch.Tensor, gate_idx: torch.Tensor, score: torch.Tensor, w1: MXTensor, b1,
                 w2: MXTensor, b2, activation) -> torch.Tensor:
    r"""sum_j score[t, j] * expert_{gate_idx[t, j]}(x[t]) over the live slots (index >= 0), the
    experts being `linear -> activation -> linear` with 4-bit weights w1 [E, hidden, in] and
    w2 [E, out, hidden].  Without gradients and for GELU and ReLU: routing, one pass that
    quantises the tokens into expert order, the first product with bias, activation and
    quantisation in its epilogue, the second product, the weighted combine.  Otherwise the
    chain of single operators, in which the hidden layer is rounded to x's dtype on its way.
    An activation module with hooks, or a `forward` set on it, is called (the chain, too).
    The result has x's dtype; biases of another are taken in it (b1, without gradients, as it is)."""
    top_k = gate_idx.shape[-1] if gate_idx.dim() >= 2 else 1
    if x.dim() != 2 or x.shape[1] != w1.features or w1.codes.shape[-2] != w2.features:
        raise RuntimeError("x [tokens, in], w1 [E, hidden, in] and w2 [E, out, hidden] disagree")
    n_expert = w1.codes.shape[0]
    act = 0 if _watched(activation) else native_act(activation, x)
    grads = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, score, b1, b2))
    gate_idx = gate_idx.reshape(-1, top_k)
    b2 = None if b2 is None else b2.to(x.dtype)
    if grads or not act or x.dtype == torch.float64:
        # (the hidden layer in x's dtype: any activation takes it so, and what its gradient keeps
        # until the backward pass is half of f32's size)
        score = score.reshape(-1, top_k)
        if torch._C._get_tracing_state() is not None:
            routed = _Route.apply(gate_idx, n_expert)
            segments, live = routed[2], routed[2][-1:]
            h = _Scatter.apply(x, gate_idx, n_expert, *routed)
        else:
            plan = RoutePlan(gate_idx, n_expert)
            segments, live = plan.segments, plan.n_rows_dev
            h = FusedScatter.apply(x, plan)
        b1 = None if b1 is None else b1.to(x.dtype)
        h = _activate(activation, linear(h, segments, w1, b1), live)
        y = linear(h, segments, w2, b2)
        if torch._C._get_tracing_state() is not None:
            return _Combine.apply(y, score, gate_idx, n_expert, *routed)
        return FusedGatherCombine.apply(y, score, plan)
    native = fmoe_cuda.native()
    run = MXExpertLayer.apply if native is None else native.mx_expert_layer
    return run(x, gate_idx, score, w1.codes, w1.scales, w1.features, b1, w2.codes, w2.scales,
               w2.features, b2, act)


def _experts(inp, counts, w1, b1, w2, b2, activation):
    r"""The experts on rows in expert order, operator by operator."""
    x = linear(_as(inp, b1), counts, w1, b1)
    live = counts.seg_off[-1:] if isinstance(counts, SegmentTable) else None
    x = _activate(activation, x, live)
    return linear(_as(x, b2), counts, w2, b2)


class _MXExpertView:
    r"""`experts[i]` of an MXExpert: called like an MXExpert of one expert, on views of the
    weights `w1`, `w2` (MXTensor [1, out, in]) and of the biases `b1`, `b2` (gradients flow into
    the parameters)."""

    def __init__(self, parent: "MXExpert", i: int):
        def one(w):
            return MXTensor(w.codes[i:i + 1], w.scales[i:i + 1], w.features)
        self.w1, self.w2 = one(parent.w1), one(parent.w2)
        self.b1, self.b2 = (None if b is None else b[i:i + 1] for b in (parent.b1, parent.b2))
        self.activation = parent.activation

    def __call__(self, inp, fwd_expert_count):
        return _experts(inp, fwd_expert_count, self.w1, self.b1, self.w2, self.b2,
                        self.activation)

    def parameters(self):
        return (b for b in (self.b1, self.b2) if b is not None)


class MXExpert(nn.Module):
    r"""The experts of a layer (`linear -> activation -> linear`) with 4-bit weights, in the
    place of the fused `_Expert`: `layer.experts = MXExpert.from_expert(layer.experts)`, or
    `quantize_experts(layer)`.  Weights are uint8 buffers and frozen; the biases stay
    parameters.  Accepts host counts or a device-side SegmentTable, casts its rows to its
    parameters' dtype, and gives views of single experts, as `_Expert` does."""

    accepts_segment_table = True

    def __init__(self, w1: MXTensor, b1, w2: MXTensor, b2, activation):
        super().__init__()
        if w1.codes.dim() != 3 or w2.codes.dim() != 3 or w1.shape[0] != w2.shape[0] or \
                w1.shape[1] != w2.features:
            raise ValueError(f"w1 [E, hidden, in] and w2 [E, out, hidden] disagree: "
                             f"{tuple(w1.shape)}, {tuple(w2.shape)}")
        for name, w in (("w1", w1), ("w2", w2)):
            self.register_buffer(name + "_codes", w.codes.contiguous())
            self.register_buffer(name + "_scales", w.scales.contiguous())
        self.in_features, self.hidden_features = w1.features, w2.features
        self.num_expert = w1.shape[0]
        for name, b in (("b1", b1), ("b2", b2)):
            b = None if b is None else nn.Parameter(b.detach().clone(),
                                                    requires_grad=b.requires_grad)
            self.register_parameter(name, b)
        self.activation = activation

    @classmethod
    def from_expert(cls, expert) -> "MXExpert":
        r"""From a fused `_Expert` on the GPU, its weights quantised.  The biases keep their
        `dp_comm` tags and what else was set on them, the module its training flag; hooks on
        the expert module and on its two linear layers do not come along.  An expert with a
        `forward` other than `_Expert`'s, in itself or a linear layer, is refused."""
        l1, l2 = expert.htoh4, expert.h4toh
        for module, kind in ((expert, _Expert), (l1, FMoELinear), (l2, FMoELinear)):
            if type(module).forward is not kind.forward or "forward" in module.__dict__:
                raise TypeError(f"{type(module).__name__} computes something of its own and "
                                "cannot be quantised")
        new = cls(quantize(l1.weight), l1.bias, quantize(l2.weight), l2.bias, expert.activation)
        for old, b in ((l1.bias, new.b1), (l2.bias, new.b2)):
            if b is not None:
                b.__dict__.update(old.__dict__)
        # (not train(): the activation is shared)
        new.training = expert.training
        return new

    @property
    def w1(self) -> MXTensor:
        return MXTensor(self.w1_codes, self.w1_scales, self.in_features)

    @property
    def w2(self) -> MXTensor:
        return MXTensor(self.w2_codes, self.w2_scales, self.hidden_features)

    def forward(self, inp, fwd_expert_count):
        return _experts(inp, fwd_expert_count, self.w1, self.b1, self.w2, self.b2,
                        self.activation)

    # what FMoE.forward asks of a module that can run the whole dispatch
    def can_run_layer(self, inp, top_k) -> bool:
        return (torch.is_tensor(inp) and inp.dim() == 2 and inp.is_cuda and 1 <= top_k <= 64
                and all(b is None or b.dtype == inp.dtype for b in (self.b1, self.b2))
                and "forward" not in self.__dict__ and type(self).forward is MXExpert.forward
                # (hooks on all modules see experts called where they see `_Expert` called)
                and (is_exact_gelu(self.activation, inp) or not _has_any_global_hook())
                and not (self._forward_hooks or self._forward_pre_hooks or self._backward_hooks
                         or self._backward_pre_hooks))

    def run_layer(self, inp, gate_idx, score):
        return expert_layer(inp, gate_idx, score, self.w1, self.b1, self.w2, self.b2,
                            self.activation)

    def run_gated_layer(self, gate, inp):
        return None      # (the gate always runs as the module it is)

    def __len__(self):
        return self.num_expert

    def __getitem__(self, i):
        if not -self.num_expert <= i < self.num_expert:
            raise IndexError(f"expert {i} of {self.num_expert}")
        return _MXExpertView(self, i % self.num_expert)

    def __iter__(self):
        return (_MXExpertView(self, i) for i in range(self.num_expert))


def quantize_experts(layer):
    r"""Puts the fused experts of an `FMoE` layer on the GPU into 4 bits, in place; returns the
    layer.  Its state dict then holds `experts.w1_codes` and so on.  The gate stays, and hooks
    on the layer, the gate and the activation; see MXExpert.from_expert for the experts."""
    if not isinstance(layer.experts, _Expert):
        raise TypeError("only a layer whose experts are one fused module can be quantised")
    layer.experts = MXExpert.from_expert(layer.experts)
    return layer
