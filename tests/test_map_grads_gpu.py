"""Gradients of the moves along a map that nobody asked for are not made; the others stay the same."""
import pytest
import torch

from fastmoe_amd import _ctypes_ops, fmoe_cuda, functions
from helpers import randn

pytestmark = pytest.mark.gpu


def make(op, t, e, d, dtype, wtype):
    m = torch.rand(t, e, generator=torch.Generator().manual_seed(t)) < 0.4
    plan = functions.MapPlan(m.cuda(), int(m.sum()) + 7)
    n = plan.max_rows
    x = randn((t if op == "sort" else n, d), dtype, 1).cuda()
    w = randn((t, e), wtype, 2).cuda()
    g = randn((n if op == "sort" else t, d), dtype, 3).cuda()
    return (functions.sort_tokens if op == "sort" else functions.unsort_tokens), plan, x, w, g


@pytest.fixture(params=["extension", "ctypes"])
def binding(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(fmoe_cuda, "_compiled", None)
        for name in fmoe_cuda.OPERATORS:
            if name.startswith("map_"):
                monkeypatch.setattr(fmoe_cuda, name, getattr(_ctypes_ops, name))


@pytest.mark.parametrize("op", ["sort", "unsort"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,e,d", [(50, 5, 40), (30, 3, 777), (70, 130, 1024), (20, 4, 2048), (9, 6, 5000)])
def test_one_gradient_of_the_two(binding, op, t, e, d, dtype):
    f, plan, x, w, g = make(op, t, e, d, dtype, torch.float32)
    both = [v.clone().requires_grad_() for v in (x, w)]
    f(both[0], plan, both[1]).backward(g)
    only = w.clone().requires_grad_()
    f(x, plan, only).backward(g)
    assert torch.equal(only.grad, both[1].grad)
    only = x.clone().requires_grad_()
    f(only, plan, w).backward(g)
    assert torch.equal(only.grad, both[0].grad)
    # of a graph with both, one at a time
    a, b = (v.clone().requires_grad_() for v in (x, w))
    y = f(a, plan, b)
    assert torch.equal(torch.autograd.grad(y, b, g, retain_graph=True)[0], both[1].grad)
    assert torch.equal(torch.autograd.grad(y, a, g, retain_graph=True)[0], both[0].grad)
    for got, want in zip(torch.autograd.grad(y, (a, b), g), both):
        assert torch.equal(got, want.grad)


@pytest.mark.parametrize("op", ["sort", "unsort"])
def test_memory_of_a_gradient_of_weights_alone(binding, op):
    f, plan, x, w, g = make(op, 2000, 4, 2048, torch.float32, torch.float32)
    w.requires_grad_()
    y = f(x, plan, w)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y.backward(g)
    torch.cuda.synchronize()
    # (rows or tokens of 2048 features would take 16 MB at least)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


def test_calls_for_nothing_are_refused(binding):
    _, plan, x, w, g = make("sort", 10, 3, 16, torch.float32, torch.float32)
    tensors = plan._tensors()
    with pytest.raises(RuntimeError, match="nothing to do"):
        fmoe_cuda.map_expand(x, w, *tensors, None, False, False)
    with pytest.raises(RuntimeError, match="nothing to do"):
        fmoe_cuda.map_reduce(g, w, *tensors, None, False)
    # tokens of none
    none = functions.MapPlan(torch.zeros(0, 3, dtype=torch.bool, device="cuda"), 4)
    v = torch.zeros(0, 3, device="cuda", requires_grad=True)
    functions.sort_tokens(x[:0], none, v).sum().backward()
    assert v.grad.shape == (0, 3)
    v.grad = None
    functions.unsort_tokens(torch.zeros(4, 16, device="cuda"), none, v).sum().backward()
    assert v.grad.shape == (0, 3)
