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


@pytest.mark.parametrize("d", [8, 77, 1024])
def test_rows_behind_the_last_are_left_as_they_were(d):
    """On a buffer of the caller's own: without n_rows_dev nothing is written there, with it zeros."""
    from fastmoe_amd import _lib

    _, plan, x, w, _ = make("sort", 50, 6, d, torch.bfloat16, torch.float32)
    live = plan.n_rows_dev.item()
    assert live == plan.max_rows - 7
    seg, off, pairs = plan._tensors()
    want = functions.sort_tokens(x, plan, w)[:live]
    for end in (None, seg[-1:].data_ptr()):
        rows = torch.full((plan.max_rows, d), 5.0, dtype=torch.bfloat16, device="cuda")
        rc = _lib.load().fmoe_map_expand(x.data_ptr(), None, w.data_ptr(), off.data_ptr(),
                                         pairs.data_ptr(), end, rows.data_ptr(), None, 50, d, 6,
                                         plan.max_rows, 3, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(rows[:live], want) and (rows[live:] == (5 if end is None else 0)).all()


def test_gradients_beyond_32_bits():
    """2.2 M rows of 1024 features in bf16: byte offsets of rows past 2^32 in either direction."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough memory")
    g = torch.Generator("cuda").manual_seed(1)
    t, e, d = 1 << 20, 4, 1024
    m = torch.rand(t, e, device="cuda", generator=g) < 0.52
    plan = functions.MapPlan(m)
    n = plan.max_rows
    assert n * d * 2 > 1 << 32
    expert, token = m.t().nonzero(as_tuple=True)
    x = torch.randn(t, d, device="cuda", dtype=torch.bfloat16, generator=g)
    rows = torch.randn(n, d, device="cuda", dtype=torch.bfloat16, generator=g)
    w = torch.rand(t, e, device="cuda", generator=g)
    places = [slice(a, a + 3000) for a in (0, t // 2, t - 3000)]
    row_of = torch.full((t, e), -1, dtype=torch.long, device="cuda")
    row_of[token, expert] = torch.arange(n, device="cuda")

    def bound(want, size, dtype, terms):
        return torch.finfo(dtype).eps / 2 * want.abs() * (1 + 1e-6) + (terms + 1) * 2.0 ** -24 * size

    def check_weights(got):
        assert (got[~m] == 0).all()
        for p in places:
            a, b = x[p].double()[:, None], rows[row_of[p].clamp(min=0)].double()
            want, size = (a * b).sum(-1) * m[p], (a * b).abs().sum(-1)
            assert ((got[p] - want).abs() <= bound(want, size, torch.float32, d)).all()

    def check_tokens(got):
        for p in places:
            term = rows[row_of[p].clamp(min=0)].double() * (w[p] * m[p]).double()[..., None]
            want, size = term.sum(1), term.abs().sum(1)
            assert ((got[p] - want).abs() <= bound(want, size, torch.bfloat16, e)).all()

    def check_rows(got):
        for a in (0, n // 2, n - 3000):
            p = slice(a, a + 3000)
            want = x[token[p]].double() * w[token[p], expert[p]].double()[:, None]
            assert ((got[p] - want).abs() <= bound(want, want.abs(), torch.bfloat16, 1)).all()

    for f, have, grad, check in ((functions.sort_tokens, x, rows, check_tokens),
                                 (functions.unsort_tokens, rows, x, check_rows)):
        have, weight = have.detach().requires_grad_(), w.clone().requires_grad_()
        f(have, plan, weight).backward(grad)
        check(have.grad)
        check_weights(weight.grad)
        have.grad = None


def test_the_most_tokens():
    """2^23 tokens: a block each with the weights' gradient, 2^23 waves without."""
    t, e, d = 1 << 23, 2, 8
    m = torch.zeros(t, e, dtype=torch.bool, device="cuda")
    at = torch.tensor([0, 1, 4095, 1 << 22, t - 1], device="cuda")
    m[at, 1] = True
    plan = functions.MapPlan(m)
    x = torch.arange(t, device="cuda", dtype=torch.float32)[:, None].expand(t, d).contiguous()
    x.requires_grad_()
    w = torch.full((t, e), 2.0, device="cuda", requires_grad=True)
    rows = functions.sort_tokens(x, plan, w)
    assert torch.equal(rows[:, 0], 2.0 * at)
    y = functions.unsort_tokens(rows, plan)
    assert torch.equal(y[at, 3], 2.0 * at) and y.count_nonzero() == 4 * d
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad[at, 0], torch.full((5,), 2.0, device="cuda"))
    assert x.grad.count_nonzero() == 5 * d
    assert torch.equal(w.grad[at, 1], 8.0 * at) and w.grad.count_nonzero() == 4
