r"""Experts with 8-bit weights: rows in integers with one scale each, their products on the matrix
cores (a scale for each token and each output channel), and the quantisation of checkpoints.

With a = max |x| over a row, its scale is a / 127 and the code of x the integer nearest to
127 x / a.  Weights are quantised once, a scale per output feature, and stay frozen; rows of
activations are quantised on the way into a product, their gradient passes straight through that
rounding.  Sums of products are exact integers.

The reference has no such experts; the products stand in the place of the ones of
fmoe/linear.py:12-52.
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

STEP = 128      # rows of codes are padded with zeros to multiples of this


class I8Tensor:
    r"""Rows of `features` values in 8 bits: `codes` int8 [..., rows, 128 ceil(features / 128)],
    zeros behind the last feature, and `scales` float32 [..., rows]."""

    __slots__ = ("codes", "scales", "features")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, features: int):
        self.codes, self.scales, self.features = codes, scales, int(features)

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.features))

    @property
    def device(self):
        return self.codes.device

    def to(self, device) -> "I8Tensor":
        return I8Tensor(self.codes.to(device), self.scales.to(device), self.features)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        r"""The values [..., rows, features] as `dtype` (float32, float16 or bfloat16)."""
        native = fmoe_cuda.native()
        if native is not None:
            return native.i8_dequantize_rows(self.codes.contiguous(), self.scales.contiguous(),
                                             self.features, dtype)
        return _Dequantize.apply(self.codes, self.scales, self.features, dtype)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "I8Tensor":
        r"""From the tight layout of 8-bit checkpoints: codes int8 [..., rows, K] and scales
        [..., rows] or [..., rows, 1]."""
        if scales.dim() == codes.dim() and scales.shape[-1:] == (1,):
            scales = scales[..., 0]
        k = codes.shape[-1]
        if k == 0 or codes.dtype != torch.int8 or scales.shape != codes.shape[:-1]:
            raise ValueError("codes must be int8 [..., K] and scales [...]")
        return cls(nn.functional.pad(codes, (0, -k % STEP)), scales.float(), k)


# (as in mx.py: where the extension's own nodes do not apply, tracing has to see these)
class _Quantize(Function):
    @staticmethod
    def forward(ctx, x):
        k = x.shape[-1]
        codes, scales = fmoe_cuda.i8_quantize(x.reshape(-1, k).contiguous())
        codes = codes.view(*x.shape[:-1], codes.shape[-1])
        scales = scales.view(x.shape[:-1])
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
            fmoe_cuda.i8_dequantize(codes.reshape(-1, codes.shape[-1]).contiguous(),
                                    scales.reshape(-1).contiguous(), out.view(-1, features))
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, _grad):
        return None, None, None, None


def quantize(x: torch.Tensor) -> I8Tensor:
    r"""x [..., features] (float32, float16 or bfloat16, on the GPU) in 8 bits, a scale per row:
    max |x| / 127, codes rounded to nearest, ties to even.  A row of zeros has scale zero; a row
    with an infinity or a NaN is NaN."""
    k = x.shape[-1]
    native = fmoe_cuda.native()
    if native is not None:
        return I8Tensor(*native.i8_quantize_rows(x), k)
    return I8Tensor(*_Quantize.apply(x.detach()), k)


class I8Linear(Function):
    r"""All experts' linear maps on 8-bit weights in one grouped product; the gradient of the rows
    is that of the weights' values, straight through the rounding of the rows."""

    @staticmethod
    def forward(ctx, x, counts, w_codes, w_scales, bias):
        r"""`counts`: a SegmentTable, int64 counts on the host or on the device, the segment bounds
        themselves (int32 on the device), or None (one expert has all rows)."""
        in_feat = x.shape[1]
        x = x.contiguous()
        bias = None if bias is None else bias.contiguous()
        on_device = isinstance(counts, torch.Tensor) and counts.is_cuda
        if counts is None or (on_device and counts.dtype == torch.int64):
            codes, scales, seg_off = fmoe_cuda.i8_quantize_counted(
                x, None if counts is None else counts.contiguous())
        else:
            if isinstance(counts, torch.Tensor) and not on_device and (
                    bool((counts < 0).any()) or int(counts.sum()) > x.shape[0]):
                raise RuntimeError("expert counts are negative or claim more rows than x holds")
            seg_off = (bounds_within(counts, x.shape[0]).contiguous() if on_device
                       else _segments(counts, x))
            # (rows behind a segment table's end, those of dropped slots, are left out)
            host = isinstance(counts, torch.Tensor) and not on_device
            codes, scales = fmoe_cuda.i8_quantize(x, None if host else seg_off[-1:])
        out = torch.empty((x.shape[0], w_codes.shape[1]), dtype=x.dtype, device=x.device)
        fmoe_cuda.i8_linear_fwd(codes, scales, w_codes, w_scales, in_feat, bias, seg_off, out)
        ctx.in_feat = in_feat
        ctx.save_for_backward(seg_off, w_codes, w_scales)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        seg_off, w_codes, w_scales = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, db = fmoe_cuda.i8_linear_bwd(grad_out.contiguous(), seg_off, w_codes, w_scales,
                                         ctx.in_feat, need[0], need[4])
        return dx, None, None, None, db


def linear(x: torch.Tensor, fwd_expert_count, weight: I8Tensor, bias=None) -> torch.Tensor:
    r"""y[rows of e] = x[rows of e] @ weight[e].T + bias[e]: the grouped linear layer of
    `FMoELinear` with 8-bit weights [E, out, in].  x [rows, in] holds the rows in expert order and
    is quantised on the way; `fwd_expert_count` is an int64 tensor of row counts (host or device) or
    a SegmentTable; bias [E, out] has x's dtype, as has the result.  Rows of x that the counts do
    not cover are in no product: their rows of y are left as they were allocated, their gradient is
    zero.  With a weight [out, in] and a bias [out], all rows go through that one weight, and
    `fwd_expert_count` is None."""
    codes, scales = weight.codes, weight.scales
    if codes.dim() == 2:
        if fwd_expert_count is not None:
            raise RuntimeError("one weight [out, in] takes all rows: fwd_expert_count must be None")
        codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
        bias = None if bias is None else bias.unsqueeze(0)
    native = fmoe_cuda.native()
    if native is not None:
        segments = segments_for(fwd_expert_count, x)
        return native.i8_linear(x, segments, codes, scales, weight.features, bias)
    if isinstance(fwd_expert_count, SegmentTable) and torch._C._get_tracing_state() is not None:
        raise RuntimeError("a SegmentTable would be a constant of the trace: hand over counts")
    if x.dim() != 2 or x.shape[1] != weight.features or not x.is_cuda:
        raise RuntimeError(f"x must be a CUDA tensor [rows, {weight.features}]")
    if fwd_expert_count is None and (codes.dim() != 3 or codes.shape[0] != 1):
        raise RuntimeError("the rows of several experts need counts")
    return I8Linear.apply(x, fwd_expert_count, codes, scales, bias)


def expert_layer(x: torch.Tensor, gate_idx: torch.Tensor, score: torch.Tensor, w1: I8Tensor, b1,
                 w2: I8Tensor, b2, activation) -> torch.Tensor:
    r"""sum_j score[t, j] * expert_{gate_idx[t, j]}(x[t]) over the live slots (index >= 0), the
    experts being `linear -> activation -> linear` with 8-bit weights w1 [E, hidden, in] and
    w2 [E, out, hidden].  Without gradients and for GELU and ReLU tokens are quantised into expert
    order in one pass; the bits are those of the chain of single operators, which runs otherwise.
    An activation module with hooks, or a `forward` set on it, is called.  The hidden layer and the
    result have x's dtype; biases of another are taken in it."""
    top_k = gate_idx.shape[-1] if gate_idx.dim() >= 2 else 1
    if x.dim() != 2 or x.shape[1] != w1.features or w1.codes.shape[-2] != w2.features:
        raise RuntimeError("x [tokens, in], w1 [E, hidden, in] and w2 [E, out, hidden] disagree")
    act = 0 if _watched(activation) else native_act(activation, x)
    grads = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, score, b1, b2))
    gate_idx = gate_idx.reshape(-1, top_k)
    native = None if grads or not act or x.dtype == torch.float64 else fmoe_cuda.native()
    if native is None:
        return layer_chain(linear, x, gate_idx, score, w1, b1, w2, b2, activation)
    return native.i8_expert_layer(x, gate_idx, score, w1.codes, w1.scales, w1.features, b1,
                                  w2.codes, w2.scales, w2.features, b2, act)


class I8Expert(FrozenExpert):
    r"""The experts of a layer (`linear -> activation -> linear`) with 8-bit weights, in the place
    of the fused `_Expert`: `layer.experts = I8Expert.from_expert(layer.experts)`, or
    `quantize_experts(layer)`.  Codes and scales are buffers and frozen; the biases stay parameters.
    Scales stay in float32 whatever dtype the module is cast to."""

    tensor = I8Tensor

    def _apply(self, fn, *args, **kwargs):
        kept = {name: getattr(self, name) for name in ("w1_scales", "w2_scales")}
        super()._apply(fn, *args, **kwargs)
        for name, scales in kept.items():
            now = getattr(self, name)
            if now.dtype != scales.dtype:
                setattr(self, name, scales.to(now.device))
        return self

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
    r"""Puts the fused experts of an `FMoE` layer on the GPU into 8 bits, in place; returns the
    layer.  Its state dict then holds `experts.w1_codes`, `experts.w1_scales` and so on.  The gate
    stays, and hooks on the layer, the gate and the activation; see FrozenExpert.from_expert for the
    experts."""
    return I8Expert.replace_in(layer)
