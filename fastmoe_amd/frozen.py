r"""Experts with quantised, frozen weights in the place of the fused `_Expert` of
fmoe/transformer.py:11-31: what 4-bit (mx.py) and 8-bit ones (i8.py) share."""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.nn.modules.module import _has_any_global_hook

from . import fmoe_cuda
from .functions import (FusedGatherCombine, FusedScatter, RoutePlan, SegmentTable,
                        apply_activation)
from .linear import FMoELinear, is_exact_gelu
from .transformer import _Expert, _watched


def activate(activation, x, n_rows_dev):
    r"""`activation(x)`, called as the module it is where somebody watches it."""
    return activation(x) if _watched(activation) else apply_activation(activation, x, n_rows_dev)


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


def layer_chain(linear, x, gate_idx, score, w1, b1, w2, b2, activation):
    r"""A layer of quantised experts operator by operator, from gate_idx [tokens, top_k] to combined
    rows; `linear(rows, segments, weight, bias)` multiplies."""
    n_expert = w1.codes.shape[0]
    tracing = torch._C._get_tracing_state() is not None
    score = score.reshape(-1, gate_idx.shape[-1])
    if tracing:
        routed = _Route.apply(gate_idx, n_expert)
        segments, live = routed[2], routed[2][-1:]
        h = _Scatter.apply(x, gate_idx, n_expert, *routed)
    else:
        plan = RoutePlan(gate_idx, n_expert)
        segments, live = plan.segments, plan.n_rows_dev
        h = FusedScatter.apply(x, plan)
    b1, b2 = (None if b is None else b.to(x.dtype) for b in (b1, b2))
    h = activate(activation, linear(h, segments, w1, b1), live)
    y = linear(h, segments, w2, b2)
    if tracing:
        return _Combine.apply(y, score, gate_idx, n_expert, *routed)
    return FusedGatherCombine.apply(y, score, plan)


def _as(x, bias):
    return x if bias is None else x.type_as(bias)


def _experts(kind, inp, counts, w1, b1, w2, b2, activation):
    r"""The experts on rows in expert order, operator by operator."""
    x = kind.linear(_as(inp, b1), counts, w1, b1)
    live = counts.seg_off[-1:] if isinstance(counts, SegmentTable) else None
    x = activate(activation, x, live)
    return kind.linear(_as(x, b2), counts, w2, b2)


class _View:
    r"""`experts[i]` of a FrozenExpert: called like one of a single expert, on views of the weights
    `w1`, `w2` ([1, out, in]) and of the biases `b1`, `b2` (gradients flow into the parameters)."""

    def __init__(self, parent: "FrozenExpert", i: int):
        def one(w):
            return type(w)(w.codes[i:i + 1], w.scales[i:i + 1], w.features)
        self.kind = type(parent)
        self.w1, self.w2 = one(parent.w1), one(parent.w2)
        self.b1, self.b2 = (None if b is None else b[i:i + 1] for b in (parent.b1, parent.b2))
        self.activation = parent.activation

    def __call__(self, inp, fwd_expert_count):
        return _experts(self.kind, inp, fwd_expert_count, self.w1, self.b1, self.w2, self.b2,
                        self.activation)

    def parameters(self):
        return (b for b in (self.b1, self.b2) if b is not None)


class FrozenExpert(nn.Module):
    r"""A kind of quantised experts says how weights are held (`tensor`, with codes, scales and
    features), made (`quantize`) and multiplied (`linear`), and how a whole layer runs (`layer`)."""

    accepts_segment_table = True
    tensor = None

    def __init__(self, w1, b1, w2, b2, activation):
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
    def from_expert(cls, expert):
        r"""From a fused `_Expert` on the GPU, its weights quantised.  The biases keep their
        `dp_comm` tags and what else was set on them, the module its training flag; hooks on
        the expert module and on its two linear layers do not come along.  An expert with a
        `forward` other than `_Expert`'s, in itself or a linear layer, is refused."""
        l1, l2 = expert.htoh4, expert.h4toh
        for module, kind in ((expert, _Expert), (l1, FMoELinear), (l2, FMoELinear)):
            if type(module).forward is not kind.forward or "forward" in module.__dict__:
                raise TypeError(f"{type(module).__name__} computes something of its own and "
                                "cannot be quantised")
        new = cls(cls.quantize(l1.weight), l1.bias, cls.quantize(l2.weight), l2.bias,
                  expert.activation)
        for old, b in ((l1.bias, new.b1), (l2.bias, new.b2)):
            if b is not None:
                b.__dict__.update(old.__dict__)
        # (not train(): the activation is shared)
        new.training = expert.training
        return new

    @classmethod
    def replace_in(cls, layer):
        r"""Puts these in the place of a layer's fused experts; returns the layer."""
        if not isinstance(layer.experts, _Expert):
            raise TypeError("only a layer whose experts are one fused module can be quantised")
        layer.experts = cls.from_expert(layer.experts)
        return layer

    @property
    def w1(self):
        return self.tensor(self.w1_codes, self.w1_scales, self.in_features)

    @property
    def w2(self):
        return self.tensor(self.w2_codes, self.w2_scales, self.hidden_features)

    def forward(self, inp, fwd_expert_count):
        return _experts(type(self), inp, fwd_expert_count, self.w1, self.b1, self.w2, self.b2,
                        self.activation)

    # what FMoE.forward asks of a module that can run the whole dispatch
    def can_run_layer(self, inp, top_k) -> bool:
        return (torch.is_tensor(inp) and inp.dim() == 2 and inp.is_cuda and 1 <= top_k <= 64
                and all(b is None or b.dtype == inp.dtype for b in (self.b1, self.b2))
                and "forward" not in self.__dict__ and type(self).forward is FrozenExpert.forward
                # (hooks on all modules see experts called where they see `_Expert` called)
                and (is_exact_gelu(self.activation, inp) or not _has_any_global_hook())
                and not (self._forward_hooks or self._forward_pre_hooks or self._backward_hooks
                         or self._backward_pre_hooks))

    def run_layer(self, inp, gate_idx, score):
        return self.layer(inp, gate_idx, score, self.w1, self.b1, self.w2, self.b2,
                          self.activation)

    def run_gated_layer(self, gate, inp):
        return None      # (the gate always runs as the module it is)

    def __len__(self):
        return self.num_expert

    def __getitem__(self, i):
        if not -self.num_expert <= i < self.num_expert:
            raise IndexError(f"expert {i} of {self.num_expert}")
        return _View(self, i % self.num_expert)

    def __iter__(self):
        return (_View(self, i) for i in range(self.num_expert))
