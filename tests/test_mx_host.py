"""4-bit experts, what needs no GPU: how the layer is called, not what its kernels compute.  The
operators are opaque stand-ins that autograd and tracing cannot look into, like the real ones."""
import os
import re

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from conftest import ROOT

E, D, H = 3, 32, 64


def _weight(out, features, seed):
    from fastmoe_amd import mx

    rng = np.random.default_rng(seed)
    return mx.MXTensor(
        torch.from_numpy(rng.integers(0, 256, (E, out, -(-features // 128) * 64)).astype(np.uint8)),
        torch.from_numpy(rng.integers(120, 130, (E, out, -(-features // 512) * 16)).astype(np.uint8)),
        features)


@pytest.fixture
def operators(monkeypatch):
    """Operators on the CPU whose results depend on their inputs; the list of their calls."""
    from fastmoe_amd import fmoe_cuda

    calls = []

    def stand_in(name, fn):
        def op(*args, **kwargs):
            calls.append(name)
            with torch.no_grad():
                return fn(*args, **kwargs)
        monkeypatch.setattr(fmoe_cuda, name, op)

    def opaque(a):
        return torch.from_numpy(a.detach().float().numpy().copy())

    def route(gate, n_expert, want_inv=True):
        g = gate.numpy().reshape(-1)
        order = np.argsort(np.where(g < 0, n_expert, g), kind="stable")
        live = int((g >= 0).sum())
        inv = np.full(g.size, -1, dtype=np.int32)
        inv[order[:live]] = np.arange(live)
        counts = np.bincount(g[g >= 0], minlength=n_expert)
        seg = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        return tuple(torch.from_numpy(a.copy()) for a in (order, counts, seg, inv))

    def quantize_tokens(x, inv, top_k):
        rows = torch.zeros(x.shape[0] * top_k, x.shape[1])
        keep = inv >= 0
        rows[inv[keep].long()] = opaque(x).repeat_interleave(top_k, 0)[keep]
        return rows, torch.zeros(rows.shape[0], 16)

    def linear_act(codes, scales, wc, ws, k, bias, seg, act):
        return codes.mean(1, keepdim=True).repeat(1, wc.shape[1]), scales

    def linear_fwd(codes, scales, wc, ws, k, bias, seg, out):
        return out.copy_(codes.mean(1, keepdim=True).to(out.dtype))

    def combine(buf, inv, score, n_tokens, top_k):
        rows = buf[inv.clamp(min=0).long()].view(n_tokens, top_k, -1)
        return (rows * (opaque(score) * (inv >= 0).view(n_tokens, top_k))[..., None]).sum(1)

    for name, fn in (("route", route), ("mx_quantize_tokens", quantize_tokens),
                     ("mx_linear_act_fwd", linear_act), ("mx_linear_fwd", linear_fwd),
                     ("gather_combine_fwd", combine)):
        stand_in(name, fn)
    monkeypatch.setattr(fmoe_cuda, "_compiled", None)      # (the other binding's way)
    return calls


def _inputs(seed, tokens=5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, D, generator=g)
    idx = torch.randint(-1, E, (tokens, 2), generator=g)
    return x, idx, torch.rand(tokens, 2, generator=g) + 0.5


def test_traced_expert_layer_follows_its_inputs(operators):
    from fastmoe_amd import mx

    w1, w2 = _weight(H, D, 1), _weight(D, H, 2)

    def layer(x, idx, score):
        return mx.expert_layer(x, idx, score, w1, None, w2, None, torch.nn.ReLU())

    with torch.no_grad():
        traced = torch.jit.trace(layer, _inputs(0), check_trace=False)
        for seed in (0, 1, 2):
            new = _inputs(seed)
            want = layer(*new)
            assert want.any() and torch.equal(traced(*new), want)
        assert not torch.equal(layer(*_inputs(1)), layer(*_inputs(2)))


@pytest.mark.parametrize("which", ["x", "score"])
def test_forward_mode_differentiation_is_refused(operators, which):
    from fastmoe_amd import mx

    w1, w2 = _weight(H, D, 1), _weight(D, H, 2)
    x, idx, score = _inputs(0)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x if which == "x" else score,
                                    torch.ones_like(x if which == "x" else score))
        x, score = (dual, score) if which == "x" else (x, dual)
        with pytest.raises((RuntimeError, NotImplementedError)):
            mx.expert_layer(x, idx, score, w1, None, w2, None, torch.nn.ReLU())


def _inputs_of(graph, kind):
    return [i.node().kind() for n in graph.nodes() if n.kind() == kind for i in n.inputs()]


@pytest.mark.parametrize("act", [torch.nn.ReLU(), torch.nn.SiLU()])
def test_traces_hand_no_uninitialised_memory_to_operators(operators, monkeypatch, act):
    """Real operators allocate their results with torch.empty and fill them behind tracing's back:
    a traced call may only ever see what a recorded function returned."""
    from fastmoe_amd import fmoe_cuda, mx

    def unseen(fn):
        def op(*args, **kwargs):
            def copy(t):
                out = torch.empty(t.shape, dtype=t.dtype)
                out.numpy()[...] = t.numpy()
                return out
            res = fn(*args, **kwargs)
            return tuple(map(copy, res)) if isinstance(res, tuple) else copy(res)
        return op

    for name in ("route", "mx_quantize_tokens", "mx_linear_act_fwd", "gather_combine_fwd"):
        monkeypatch.setattr(fmoe_cuda, name, unseen(getattr(fmoe_cuda, name)))
    monkeypatch.setattr(fmoe_cuda, "local_scatter", unseen(
        lambda x, pos, top_k, live: x.detach()[pos // top_k] + 0))

    class Linear(torch.autograd.Function):     # (MXLinear, which wants the GPU)
        @staticmethod
        def forward(ctx, x, seg, out_features):
            y = x.detach().mean(1, keepdim=True).repeat(1, out_features)
            y[int(seg[-1]):] = 0
            return y

        @staticmethod
        def backward(ctx, grad):
            return None, None, None

    def linear(x, counts, w, b):
        seg = counts if torch.is_tensor(counts) else counts.seg_off
        return Linear.apply(x, seg, int(w.codes.shape[-2]))

    monkeypatch.setattr(mx, "linear", linear)
    w1, w2 = _weight(H, D, 1), _weight(D, H, 2)

    def layer(x, idx, score):
        return mx.expert_layer(x, idx, score, w1, None, w2, None, act)

    with torch.no_grad():
        traced = torch.jit.trace(layer, _inputs(0), check_trace=False)
        for seed in (0, 1, 2):
            assert torch.equal(traced(*_inputs(seed)), layer(*_inputs(seed)))
        assert "aten::empty" not in _inputs_of(traced.graph, "prim::PythonOp")
        assert "prim::PythonOp" in [n.kind() for n in traced.graph.nodes()]


def test_a_segment_table_is_no_constant_of_a_trace():
    from fastmoe_amd import mx
    from fastmoe_amd.functions import SegmentTable

    w1, w2 = _weight(H, D, 1), _weight(D, H, 2)
    experts = mx.MXExpert(w1, None, w2, None, torch.nn.ReLU())
    segments = SegmentTable(torch.tensor([0, 2, 2, 5], dtype=torch.int32), torch.tensor([2, 0, 3]))
    for call in (lambda x: mx.linear(x, segments, w1), lambda x: experts(x, segments)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, torch.randn(5, D), check_trace=False)


# ------------------------------------------------------------------ quantising a layer
@pytest.fixture
def quantised(monkeypatch):
    """mx.quantize_experts on the CPU: codes and scales of the right shapes."""
    from fastmoe_amd import mx

    def quantize(x):
        k = x.shape[-1]
        return mx.MXTensor(*(torch.zeros(*x.shape[:-1], n, dtype=torch.uint8)
                             for n in (-(-k // 128) * 64, -(-k // 512) * 16)), k)

    monkeypatch.setattr(mx, "quantize", quantize)
    return mx.quantize_experts


def _layer(**kwargs):
    from fastmoe_amd import FMoETransformerMLP

    return FMoETransformerMLP(num_expert=E, d_model=D, d_hidden=H, **kwargs)


@pytest.mark.parametrize("comm", ["none", "dp"])
def test_quantised_experts_keep_tags_flags_and_gradients(quantised, comm):
    layer = _layer(expert_dp_comm=comm).eval()
    layer.experts.activation.train()
    layer.experts.h4toh.bias.requires_grad_(False)
    layer.experts.htoh4.bias.lr_scale = 3.0
    quantised(layer)
    ex = layer.experts
    assert not layer.training and not ex.training and ex.activation.training
    assert ex.b1.dp_comm == ex.b2.dp_comm == comm and ex.b1.lr_scale == 3.0
    assert ex.b1.requires_grad and not ex.b2.requires_grad
    assert quantised(_layer()).experts.training


def test_experts_without_biases_are_quantised(quantised):
    layer = _layer()
    layer.experts.htoh4.register_parameter("bias", None)
    quantised(layer)
    assert layer.experts.b1 is None and layer.experts.b2.dp_comm == "none"


def test_experts_that_compute_something_else_are_refused(quantised):
    from fastmoe_amd import FMoELinear
    from fastmoe_amd.transformer import _Expert

    class Doubled(_Expert):
        def forward(self, inp, fwd_expert_count):
            return 2 * super().forward(inp, fwd_expert_count)

    class Scaled(FMoELinear):
        def forward(self, inp, fwd_expert_count):
            return 2 * super().forward(inp, fwd_expert_count)

    def own_forward(layer):
        layer.experts.forward = lambda inp, counts: inp

    def own_linear(layer):
        layer.experts.htoh4 = Scaled(E, D, H)

    def own_linear_forward(layer):
        layer.experts.h4toh.forward = lambda inp, counts: inp

    def own_class(layer):
        layer.experts = Doubled(E, D, H, torch.nn.GELU())

    for change in (own_forward, own_linear, own_linear_forward, own_class):
        layer = _layer()
        change(layer)
        before = layer.experts
        with pytest.raises(TypeError):
            quantised(layer)
        assert layer.experts is before


# ------------------------------------------------------------------ the GELU between the products
def test_fitted_gelu_keeps_its_bounds():
    """mx_gelu of csrc/mx_gemm.hip in f32 arithmetic, its exponential and quotient correctly
    rounded: 2e-7 + 1e-7 |gelu| everywhere (the kernel's stated bound leaves 2e-7 |gelu| for the two
    approximate instructions) and 4e-6 of the value for |x| <= 6 (stated: 5e-6)."""
    from scipy.special import erfc

    with open(os.path.join(ROOT, "fastmoe_amd", "csrc", "mx_gemm.hip")) as f:
        body = re.search(r"float mx_gelu\(float x\) \{(.*?)\n\}", f.read(), re.S)[1]
    first, *rest = re.findall(r"p = (?:fmaf\(p, t, )?(-?[\d.e-]+)f\)?;", body)
    assert len(rest) == 12

    def exact(x):
        x = x.astype(np.float64)
        return 0.5 * x * erfc(-x / np.sqrt(2))

    def fitted(x):
        f32, wide = np.float32, np.float64

        def fma(a, b, c):                     # (a product of two f32 is exact in 64 bits)
            return (a.astype(wide) * b + wide(c)).astype(f32)
        t = np.minimum(fma(x * x, wide(f32(1 / 18)), -1.0), f32(1))
        p = np.full_like(x, f32(first))
        for c in rest:
            p = fma(p, t.astype(wide), f32(c))
        with np.errstate(over="ignore"):
            power = np.exp2((x * p).astype(wide)).astype(f32)
            quotient = (1 / (f32(1) + power).astype(wide)).astype(f32)
        return x * quotient

    everywhere = np.concatenate([np.linspace(-30, 30, 2_000_001), np.linspace(-2, 2, 1_000_001),
                                 -np.logspace(-20, 20, 100_001), np.logspace(-20, 20, 100_001)])
    x = everywhere.astype(np.float32)
    want = exact(x)
    assert (np.abs(fitted(x) - want) <= 2e-7 + 1e-7 * np.abs(want)).all()
    x = np.linspace(-6, 6, 2_000_000).astype(np.float32)
    want = exact(x)
    assert (np.abs(fitted(x) - want) <= 4e-6 * np.abs(want)).all()
