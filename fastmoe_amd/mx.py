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

from . import fmoe_cuda
from .frozen import FrozenExpert, layer_chain
from .functions import SegmentTable, bounds_within, segments_for
from .linear import _segments, native_act
from .transformer import _watched

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
            seg_off = (bounds_within(counts, x.shape[0]).contiguous() if on_device
                       else _segments(counts, x))
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
        segments = segments_for(fwd_expert_count, x)
        return native.mx_linear(x, segments, weight.codes, weight.scales, weight.features, bias)
    if isinstance(fwd_expert_count, SegmentTable) and torch._C._get_tracing_state() is not None:
        raise RuntimeError("a SegmentTable would be a constant of the trace: trace the layer or "
                           "mx.expert_layer, or hand over counts")
    if x.dim() != 2 or x.shape[1] != weight.features or not x.is_cuda:
        raise RuntimeError(f"x must be a CUDA tensor [rows, {weight.features}]")
    return MXLinear.apply(x, fwd_expert_count, weight.codes, weight.scales, bias)


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
        return layer_chain(linear, x, gate_idx, score, w1, b1, w2, b2, activation)
    native = fmoe_cuda.native()
    run = MXExpertLayer.apply if native is None else native.mx_expert_layer
    return run(x, gate_idx, score, w1.codes, w1.scales, w1.features, b1, w2.codes, w2.scales,
               w2.features, b2, act)


class MXExpert(FrozenExpert):
    r"""The experts of a layer (`linear -> activation -> linear`) with 4-bit weights, in the
    place of the fused `_Expert`: `layer.experts = MXExpert.from_expert(layer.experts)`, or
    `quantize_experts(layer)`.  Weights are uint8 buffers and frozen; the biases stay
    parameters.  Accepts host counts or a device-side SegmentTable, casts its rows to its
    parameters' dtype, and gives views of single experts, as `_Expert` does."""

    tensor = MXTensor

    @staticmethod
    def quantize(weight):
        return quantize(weight)

    @staticmethod
    def linear(x, counts, weight, bias):
        return linear(x, counts, weight, bias)

    @staticmethod
    def layer(*args):
        return expert_layer(*args)


def quantize_experts(layer):
    r"""Puts the fused experts of an `FMoE` layer on the GPU into 4 bits, in place; returns the
    layer.  Its state dict then holds `experts.w1_codes` and so on.  The gate stays, and hooks
    on the layer, the gate and the activation; see MXExpert.from_expert for the experts."""
    return MXExpert.replace_in(layer)
