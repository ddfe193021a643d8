"""Tokens sorted by expert along a map of truth values, and back, against 64-bit arithmetic.

Tolerances are derived: a product and a sum of k terms in f32 are off by at most (k + 1) 2^-24 of
the sum of magnitudes, the rounding to type t by eps_t / 2 of the value."""
import pytest
import torch

from fastmoe_amd import FMoELinear, _ctypes_ops, fmoe_cuda, functions, i8
from helpers import randn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(want, dtype):
    info = torch.finfo(dtype)
    return torch.clamp(want.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def close(got, want, size, terms, dtype):
    tol = half_step(want, dtype) * (1 + 1e-6) + (terms + 1) * 2.0 ** -24 * size
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def make_map(t, e, share, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(t, e, generator=g) < share


def pairs_of(m, max_rows=None):
    """(expert, token) of every row, on the CPU."""
    expert, token = m.cpu().t().nonzero(as_tuple=True)
    return (expert, token) if max_rows is None else (expert[:max_rows], token[:max_rows])


MAPS = [(1, 1, 1.0), (1, 1, 0.0), (5, 3, 0.5), (64, 128, 0.06), (65, 8, 0.3), (1000, 300, 0.02),
        (129, 1024, 0.01), (300, 65, 1.0), (4096, 16, 0.1), (20000, 7, 0.4), (16384, 128, 0.06),
        (70001, 3, 0.5)]


@pytest.mark.parametrize("t,e,share", MAPS)
def test_plan(t, e, share):
    m = make_map(t, e, share, t + e)
    expert, token = pairs_of(m)
    n = len(token)
    for max_rows in {None, n + 5, n, n // 2, 0}:
        plan = functions.MapPlan(m.cuda(), max_rows)
        live = n if max_rows is None else min(n, max_rows)
        assert plan.max_rows == (n if max_rows is None else max_rows)
        counts = torch.bincount(expert[:live], minlength=e)
        assert torch.equal(plan.counts.cpu(), counts)
        seg = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0)))
        assert torch.equal(plan.segments.seg_off.cpu().long(), seg)
        assert plan.n_rows_dev.item() == live
        # token by token, experts ascending
        rows = torch.arange(live)
        order = (token[:live] * e + expert[:live]).argsort(stable=True)
        off = torch.zeros(t + 1, dtype=torch.long)
        off[1:] = torch.bincount(token[:live], minlength=t).cumsum(0)
        assert torch.equal(plan.token_off.cpu().long(), off)
        got = plan.pairs[:live].cpu().long()
        assert torch.equal(got[:, 0], rows[order]) and torch.equal(got[:, 1], expert[:live][order])


def test_plan_of_a_view_at_an_odd_address_and_of_no_tokens():
    m = make_map(200, 37, 0.2, 1).cuda()
    flat = torch.zeros(200 * 37 + 3, dtype=torch.bool, device="cuda")
    flat[3:] = m.view(-1)
    a, b = functions.MapPlan(m), functions.MapPlan(flat[3:].view(200, 37))
    assert torch.equal(a.pairs, b.pairs) and torch.equal(a.token_off, b.token_off)
    wide = torch.zeros(200, 74, dtype=torch.bool, device="cuda")
    wide[:, ::2] = m
    assert torch.equal(functions.MapPlan(wide[:, ::2]).pairs, a.pairs)
    none = functions.MapPlan(m[:0], 4)
    assert none.counts.tolist() == [0] * 37
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    rows = functions.sort_tokens(x, none)
    assert rows.shape == (4, 16)
    y = functions.unsort_tokens(rows.detach().requires_grad_(), none)
    assert y.shape == (0, 16)
    rows.sum().backward()
    assert x.grad.shape == (0, 16)


SIZES = [(1, 1, 1.0, 1), (5, 3, 0.5, 8), (64, 128, 0.06, 2048), (1000, 8, 0.25, 300),
         (65, 130, 0.5, 77), (2100, 16, 0.12, 1024), (2500, 5, 0.4, 2056), (300, 4, 0.5, 5000),
         (4000, 9, 0.2, 33)]


@pytest.mark.parametrize("wtype", ["none", "f32", "same"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,e,share,d", SIZES)
def test_rows_there_and_back(dtype, wtype, t, e, share, d):
    m = make_map(t, e, share, t + d)
    expert, token = pairs_of(m)
    n = len(token)
    w = None
    if wtype != "none":
        w = randn((t, e), torch.float32 if wtype == "f32" else dtype, 2).cuda().requires_grad_()
    w64 = torch.ones(t, e, dtype=torch.float64) if w is None else w.detach().cpu().double()
    we = w64[token, expert][:, None]
    plan = functions.MapPlan(m.cuda(), n + 3)
    most = int(m.sum(1).max())                     # rows of a token

    x, dy = randn((t, d), dtype, 3).cuda().requires_grad_(), randn((n + 3, d), dtype, 4).cuda()
    rows = functions.sort_tokens(x, plan, w)
    rows.backward(dy)
    x64, dy64 = x.detach().cpu().double(), dy.cpu().double()[:n]
    if w is None:
        assert torch.equal(rows[:n].cpu(), x.detach().cpu()[token])
    close(rows[:n].detach().cpu(), we * x64[token], (we * x64[token]).abs(), 1, dtype)
    term = we * dy64
    close(x.grad.cpu(), torch.zeros(t, d).double().index_add_(0, token, term),
          torch.zeros(t, d).double().index_add_(0, token, term.abs()), most, dtype)

    def weight_gradient(a, b):
        want, size = torch.zeros(t, e).double(), torch.zeros(t, e).double()
        want[token, expert], size[token, expert] = (a * b).sum(1), (a * b).abs().sum(1)
        close(w.grad.cpu(), want, size, d, w.dtype)
        assert (w.grad.cpu()[~m] == 0).all()

    if w is not None:
        weight_gradient(x64[token], dy64)
        w.grad = None

    r, dt = randn((n + 3, d), dtype, 5).cuda().requires_grad_(), randn((t, d), dtype, 6).cuda()
    y = functions.unsort_tokens(r, plan, w)
    y.backward(dt)
    r64, dt64 = r.detach().cpu().double()[:n], dt.cpu().double()
    term = we * r64
    close(y.detach().cpu(), torch.zeros(t, d).double().index_add_(0, token, term),
          torch.zeros(t, d).double().index_add_(0, token, term.abs()), most, dtype)
    close(r.grad[:n].cpu(), we * dt64[token], (we * dt64[token]).abs(), 1, dtype)
    assert (r.grad[n:] == 0).all()                 # rows behind the last
    assert (y.detach().cpu()[m.sum(1) == 0] == 0).all()
    if w is not None:
        weight_gradient(r64, dt64[token])


def test_rows_behind_the_last_and_rows_cut_off():
    m = make_map(50, 6, 0.5, 1)
    expert, token = pairs_of(m)
    n = len(token)
    x = randn((50, 64), torch.float32, 1).cuda()
    plan = functions.MapPlan(m.cuda(), n + 9)
    rows = torch.full((n + 9, 64), 5.0, device="cuda")
    tensors = plan._tensors()
    # (the operator writes into its own buffer: no row behind the last is looked at on the way back)
    rows[:n] = functions.sort_tokens(x, plan)[:n]
    rows[n:] = float("nan")
    want = functions.unsort_tokens(rows[:n].contiguous(), functions.MapPlan(m.cuda(), n))
    assert torch.equal(functions.unsort_tokens(rows, plan), want)
    cut = functions.MapPlan(m.cuda(), n // 2)
    got = functions.sort_tokens(x, cut)
    assert torch.equal(got.cpu(), x.cpu()[token[:n // 2]])
    back = torch.zeros(50, 64).double().index_add_(0, token[:n // 2], got.cpu().double())
    close(functions.unsort_tokens(got, cut).cpu(), back, back.abs(), 6, torch.float32)
    assert len(tensors) == 3


def test_no_rows_at_all():
    m = make_map(70, 5, 0.5, 1).cuda()
    for plan in (functions.MapPlan(m, 0), functions.MapPlan(torch.zeros_like(m), 4)):
        x = randn((70, 24), torch.bfloat16, 1).cuda().requires_grad_()
        w = torch.rand(70, 5, device="cuda", requires_grad=True)
        rows = functions.sort_tokens(x, plan, w)
        assert rows.shape == (plan.max_rows, 24) and plan.counts.tolist() == [0] * 5
        rows.backward(torch.ones_like(rows))
        assert not x.grad.any() and not w.grad.any()
        r = torch.ones(plan.max_rows, 24, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w.grad = None
        y = functions.unsort_tokens(r, plan, w)
        assert not y.any()
        y.backward(torch.ones_like(y))
        assert not r.grad.any() and not w.grad.any()


def test_plans_used_twice_and_traces():
    m = make_map(60, 7, 0.3, 2).cuda()
    plan = functions.MapPlan(m)
    x = randn((60, 40), torch.float32, 1).cuda().requires_grad_()
    a, b = functions.sort_tokens(x, plan), functions.sort_tokens(x, plan)
    (a.sum() + b.sum()).backward()
    want = 2.0 * m.sum(1, keepdim=True).expand(60, 40)
    assert torch.equal(x.grad, want)
    y = functions.sort_tokens(x, plan)
    plan.pairs.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda z: functions.sort_tokens(z, plan), x.detach())


def test_values_that_are_not_finite_stay_where_they_are():
    m = torch.tensor([[True, False], [True, True], [False, False]])
    plan = functions.MapPlan(m.cuda())
    w = torch.tensor([[1.0, float("nan")], [0.5, 2.0], [float("inf"), float("nan")]]).cuda()
    x = torch.ones(3, 16, device="cuda")
    x[2] = float("nan")
    rows = functions.sort_tokens(x, plan, w)
    assert torch.equal(rows[:, 0].cpu(), torch.tensor([1.0, 0.5, 2.0]))
    y = functions.unsort_tokens(rows, plan, w)
    assert torch.equal(y[:, 0].cpu(), torch.tensor([1.0, 4.25, 0.0]))


@pytest.mark.parametrize("op", ["sort", "unsort"])
def test_gradients_against_differences(op):
    """Both are linear in the rows and in the weights: differences are exact up to f32 sums."""
    m = make_map(12, 5, 0.4, 3)
    plan = functions.MapPlan(m.cuda())
    n = plan.max_rows
    f = functions.sort_tokens if op == "sort" else functions.unsort_tokens
    x = randn((12 if op == "sort" else n, 24), torch.float32, 1).cuda().requires_grad_()
    w = randn((12, 5), torch.float32, 2).cuda().requires_grad_()
    g = randn((n if op == "sort" else 12, 24), torch.float32, 3).cuda()
    f(x, plan, w).backward(g)
    for leaf in (x, w):
        for i, j in ((0, 0), (3, 1), (leaf.shape[0] - 1, leaf.shape[1] - 1)):
            step = torch.zeros_like(leaf)
            step[i, j] = 1.0
            with torch.no_grad():
                a, b = ((x + step, w), (x - step, w)) if leaf is x else ((x, w + step), (x, w - step))
                slope = ((f(a[0], plan, a[1]) - f(b[0], plan, b[1])).double() * g.double()).sum() / 2
            # values below 8, at most 24 * 5 of them, a few roundings each
            assert abs(slope - leaf.grad[i, j]) < 120 * 8 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
def test_there_and_back_is_a_weighted_copy(dtype):
    """Weights that add up to one: powers of two make it exact."""
    m = make_map(333, 12, 0.4, 3)
    m[:, 0] = True
    k = m.sum(1, keepdim=True)
    plan = functions.MapPlan(m.cuda())
    x = randn((333, 520), dtype, 1).cuda()
    w = (2.0 ** torch.floor(torch.log2(1.0 / k))).expand(333, 12).to(dtype).cuda()
    y = functions.unsort_tokens(functions.sort_tokens(x, plan), plan, w)
    want = x.double() * (w.double()[:, :1] * k.cuda())
    close(y, want, want.abs(), 12, dtype)


def test_with_the_expert_layers():
    """Experts that choose their tokens: sorted rows, 8-bit products, the weighted way back; then
    the same on a 16-bit FMoELinear, with gradients of everything."""
    t, e, d, h, cap = 96, 6, 128, 264, 20
    logits = randn((t, e), torch.float32, 1).cuda()
    taken = torch.zeros(t, e, dtype=torch.bool, device="cuda")
    taken.scatter_(0, logits.topk(cap, dim=0)[1], True)
    plan = functions.MapPlan(taken, e * cap)
    assert plan.counts.tolist() == [cap] * e
    x = randn((t, d), torch.bfloat16, 2).cuda().requires_grad_()
    weight = logits.sigmoid().requires_grad_()
    w1 = i8.quantize(randn((e, h, d), torch.float32, 3, 0.05).cuda())
    w2 = i8.quantize(randn((e, d, h), torch.float32, 4, 0.05).cuda())
    rows = functions.sort_tokens(x, plan)
    a = i8.linear(rows, plan.segments, w1)
    b = i8.linear(torch.relu(a), plan.segments, w2)
    y = functions.unsort_tokens(b, plan, weight)
    y.float().square().sum().backward()

    # in 64 bits from the same codes; the hidden rows come as they were rounded
    expert, token = (i.cuda() for i in pairs_of(taken))
    v1, v2 = (w.codes[..., :w.features].double() * w.scales.double()[..., None] for w in (w1, w2))

    def through(z, w):
        # (integer sums first, which f64 holds exactly, then the scales: a sum of scaled terms that
        # cancels would leave f64's own roundings where the result is zero)
        q = i8.quantize(z)
        return torch.cat([(q.codes[expert == i].double() @ w.codes[i].double().T)
                          * q.scales[expert == i].double()[:, None] * w.scales[i].double()
                          for i in range(e)])

    want = through(rows.detach(), w1)
    close(a.detach(), want, want.abs(), 8, torch.bfloat16)
    hidden = torch.relu(a).detach()
    want = through(hidden, w2)
    close(b.detach(), want, want.abs(), 8, torch.bfloat16)
    wt = weight.detach().double()[token, expert][:, None]
    term = wt * b.detach().double()
    close(y.detach(), torch.zeros(t, d, device="cuda").double().index_add_(0, token, term),
          torch.zeros(t, d, device="cuda").double().index_add_(0, token, term.abs()), e,
          torch.bfloat16)
    # gradients: from y's rounded gradient on, each stage's rounding eps / 2 of the largest value
    gy = (2 * y.detach().float()).to(torch.bfloat16).double()
    gb = wt * gy[token]
    ga = torch.cat([gb[expert == i] @ v2[i] for i in range(e)]) * (a.detach() > 0)
    gx = torch.cat([ga[expert == i] @ v1[i] for i in range(e)])
    gx = torch.zeros(t, d, device="cuda").double().index_add_(0, token, gx)
    # gb, the two products (weights and result) and the sum: 6 roundings of 2^-8, each of a value
    # that enters sums of random signs, so below 6 * 2^-8 of the norm
    assert (x.grad.double() - gx).norm() <= 6 * 2.0 ** -8 * gx.norm()
    dw = torch.zeros(t, e, device="cuda").double()
    dw[token, expert] = (b.detach().double() * gy[token]).sum(1)
    size = torch.zeros_like(dw)
    size[token, expert] = (b.detach().double() * gy[token]).abs().sum(1)
    close(weight.grad, dw, size, d, torch.float32)

    linear = FMoELinear(e, d, h).cuda().to(torch.bfloat16)
    out = functions.unsort_tokens(linear(functions.sort_tokens(x, plan), plan.segments), plan,
                                  weight.detach())
    out.sum().backward()
    assert linear.weight.grad.isfinite().all() and out.shape == (t, h)


def test_both_bindings_give_the_same_bits(monkeypatch):
    m = make_map(300, 20, 0.2, 1).cuda()
    x, w = randn((300, 136), torch.bfloat16, 1).cuda(), randn((300, 20), torch.float32, 2).cuda()
    n = int(m.sum())
    g, gy = randn((n + 2, 136), torch.bfloat16, 3).cuda(), randn((300, 136), torch.bfloat16, 4).cuda()

    def run():
        plan = functions.MapPlan(m, n + 2)
        z, v = x.clone().requires_grad_(), w.clone().requires_grad_()
        rows = functions.sort_tokens(z, plan, v)
        rows.backward(g)
        r, u = g.clone().requires_grad_(), w.clone().requires_grad_()
        y = functions.unsort_tokens(r, plan, u)
        y.backward(gy)
        return [plan.counts, plan.pairs[:n], plan.token_off, rows.detach()[:n], z.grad, v.grad,
                y.detach(), r.grad, u.grad]

    want = run()
    monkeypatch.setattr(fmoe_cuda, "_compiled", None)
    for name in fmoe_cuda.OPERATORS:
        if name.startswith("map_"):
            monkeypatch.setattr(fmoe_cuda, name, getattr(_ctypes_ops, name))
    for a, b in zip(want, run()):
        assert torch.equal(a, b)


def test_strides_another_stream_and_replays():
    m = make_map(3000, 16, 0.1, 1).cuda()
    x = randn((64, 3000), torch.bfloat16, 1).cuda().t()
    w = randn((16, 3000), torch.float32, 2).cuda().t()
    plan = functions.MapPlan(m, 6000)
    n = plan.n_rows_dev.item()
    want = functions.sort_tokens(x, plan, w)
    assert torch.equal(want[:n], functions.sort_tokens(x.contiguous(), plan, w.contiguous())[:n])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = functions.MapPlan(m, 6000)
        rows = functions.sort_tokens(x, other, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(rows[:n], want[:n]) and torch.equal(other.pairs[:n], plan.pairs[:n])
    # two graphs of plans and rows, replayed in turn with eager calls between
    graphs = []
    for seed in (1, 2):
        held, z = m.clone(), x.contiguous().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p = functions.MapPlan(held, 6000)
            r = functions.sort_tokens(z, p, w)
            y = functions.unsort_tokens(r, p)
        graphs.append((graph, held, z, p, r, y))
    for i in range(3):
        for j, (graph, held, z, p, r, y) in enumerate(graphs):
            held.copy_(make_map(3000, 16, 0.1, 10 * i + j))
            z.copy_(randn((3000, 64), torch.bfloat16, 20 * i + j))
            graph.replay()
            q = functions.MapPlan(held, 6000)
            s = functions.sort_tokens(z, q, w)
            k = q.n_rows_dev.item()
            assert torch.equal(p.counts, q.counts) and torch.equal(r[:k], s[:k])
            assert torch.equal(y, functions.unsort_tokens(s, q))


def test_rows_beyond_32_bits():
    """2^20 tokens, 2.2 M rows of 1024 features: byte offsets past 2^32."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough memory")
    g = torch.Generator("cuda").manual_seed(1)
    t, e, d = 1 << 20, 4, 1024
    m = torch.rand(t, e, device="cuda", generator=g) < 0.52
    x = torch.randn(t, d, device="cuda", dtype=torch.bfloat16, generator=g)
    plan = functions.MapPlan(m)
    assert plan.max_rows * d * 2 > 1 << 32
    rows = functions.sort_tokens(x, plan)
    expert, token = m.t().nonzero(as_tuple=True)
    for at in (0, plan.max_rows // 2, plan.max_rows - 5000):
        assert torch.equal(rows[at:at + 5000], x[token[at:at + 5000]])
    y = functions.unsort_tokens(rows, plan)
    k = m.sum(1, keepdim=True).double()
    for at in (0, t // 2, t - 5000):
        want = x[at:at + 5000].double() * k[at:at + 5000]
        close(y[at:at + 5000], want, want.abs(), 4, torch.bfloat16)


def test_refusals():
    m = make_map(10, 4, 0.5, 1).cuda()
    plan = functions.MapPlan(m, 30)
    x, w = torch.zeros(10, 8, device="cuda"), torch.zeros(10, 4, device="cuda")
    rows = torch.zeros(30, 8, device="cuda")
    for call in (lambda: functions.MapPlan(m.cpu()),
                 lambda: functions.MapPlan(m.int()),
                 lambda: functions.MapPlan(m[0]),
                 lambda: functions.MapPlan(m, -1),
                 lambda: functions.MapPlan(torch.ones(2, 1025, dtype=torch.bool, device="cuda")),
                 lambda: functions.sort_tokens(x[:9], plan),
                 lambda: functions.sort_tokens(x.double(), plan),
                 lambda: functions.sort_tokens(x.cpu(), plan),
                 lambda: functions.sort_tokens(x, plan, w[:, :3]),
                 lambda: functions.sort_tokens(x.half(), plan, w.bfloat16()),
                 lambda: functions.sort_tokens(x.long(), plan),
                 lambda: functions.unsort_tokens(rows[:29], plan),
                 lambda: functions.unsort_tokens(rows, plan, w.t()),
                 lambda: functions.unsort_tokens(rows[0], plan),
                 lambda: functions.unsort_tokens(rows, plan, w.cpu())):
        with pytest.raises(RuntimeError):
            call()
    y = functions.unsort_tokens(rows.requires_grad_(), plan, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), rows, create_graph=True)
