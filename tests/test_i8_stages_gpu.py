"""Whole layers of 8-bit experts stage by stage in 64 bits, each stage from what the library rounded in
front of it, so that no code of the hidden layer is off and a bound is the stage's own rounding."""
import pytest
import torch

from fastmoe_amd import i8
from fastmoe_amd.frozen import activate
from fastmoe_amd.functions import FusedGatherCombine, FusedScatter, RoutePlan
from helpers import make_gate, randn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = {"gelu": torch.nn.GELU(), "relu": torch.nn.ReLU()}
SIZES = [(1, 2, 1, 8, 8), (65, 4, 2, 100, 300), (500, 70, 4, 256, 384), (900, 3, 2, 130, 264)]


def half_step(want, dtype):
    info = torch.finfo(dtype)
    return torch.clamp(want.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def parts(t, e, k, d, h, dtype):
    gate = torch.from_numpy(make_gate(t, k, e, drop=0.1, seed=t, empty=(1,))).cuda()
    x = randn((t, d), dtype, 1).cuda()
    score = torch.rand(t, k, generator=torch.Generator().manual_seed(t)).to(dtype).cuda()
    w1 = i8.quantize(randn((e, h, d), torch.float32, 2, 0.05).cuda())
    w2 = i8.quantize(randn((e, d, h), torch.float32, 3, 0.05).cuda())
    b1, b2 = randn((e, h), dtype, 4).cuda(), randn((e, d), dtype, 5).cuda()
    return x, gate, score, w1, b1, w2, b2


def owners(plan):
    """The expert of every live row."""
    counts = plan.segments.counts
    return torch.repeat_interleave(torch.arange(len(counts), device=counts.device), counts)


def check_product(y, rows, owner, w, b):
    """y = rows' codes times w's plus b: 4 roundings of 2^-24 in f32 and one to y's type."""
    q, n = i8.quantize(rows), len(owner)
    want, size = (torch.zeros(n, y.shape[1], dtype=torch.float64, device="cuda") for _ in range(2))
    for e in owner.unique().tolist():
        r = owner == e
        p = (q.codes[:n][r].double() @ w.codes[e].double().T) * q.scales[:n][r].double()[:, None] \
            * w.scales[e].double()
        want[r], size[r] = p + b[e].double(), p.abs() + b[e].double().abs()
    tol = half_step(want, y.dtype) * (1 + 1e-6) + 4 * 2.0 ** -24 * size
    assert ((y[:n].double() - want).abs() <= tol).all()


def stages(x, gate, score, w1, b1, w2, b2, act):
    plan = RoutePlan(gate, w1.codes.shape[0])
    rows = FusedScatter.apply(x, plan)
    pre = i8.linear(rows, plan.segments, w1, b1)
    hidden = activate(act, pre, plan.n_rows_dev)
    out = i8.linear(hidden, plan.segments, w2, b2)
    return plan, rows, pre, hidden, out, FusedGatherCombine.apply(out, score, plan)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,e,k,d,h", SIZES)
def test_every_stage_of_a_layer(t, e, k, d, h, dtype, act):
    p = parts(t, e, k, d, h, dtype)
    x, gate, score, w1, b1, w2, b2 = p
    with torch.no_grad():
        whole = i8.expert_layer(*p, ACTS[act])
        plan, rows, pre, hidden, out, y = stages(*p, ACTS[act])
    assert torch.equal(whole, y)
    owner = owners(plan)
    n = len(owner)
    slot = plan.pos[:n].long()
    assert torch.equal(rows[:n], x[slot // k])
    check_product(pre, rows, owner, w1, b1)
    want = ACTS[act](pre[:n].double())
    # (f32's GELU: erff's error below 2^-21 of 1, a handful of f32 roundings beside it)
    slack = 2.0 ** -20 * pre[:n].double().abs() if dtype == torch.float32 and act == "gelu" else 0
    assert ((hidden[:n].double() - want).abs() <= half_step(want, dtype) * (1 + 1e-6) + slack).all()
    check_product(out, hidden, owner, w2, b2)
    term = out[:n].double() * score.reshape(-1)[slot].double()[:, None]
    want, size = (torch.zeros(t, d, dtype=torch.float64, device="cuda").index_add_(0, slot // k, v)
                  for v in (term, term.abs()))
    assert ((y.double() - want).abs() <= half_step(want, dtype) * (1 + 1e-6)
            + (k + 1) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,e,k,d,h", SIZES[1:])
def test_gradients_of_a_layer(t, e, k, d, h, dtype, act):
    """The layer's gradients from the pre-activations that the library rounded.  On the way to x: the
    combine's rows, the second product's gradient (1.03 roundings), the activation's, the first
    product's and the sum over a token's rows, each at most eps / 2 of a value; all enter sums of random
    signs, so that norms are off by less than 6 of them."""
    p = parts(t, e, k, d, h, dtype)
    with torch.no_grad():
        plan, _, pre, hidden, out, _ = stages(*p, ACTS[act])
    x, gate, score, w1, b1, w2, b2 = p
    leaves = [v.clone().requires_grad_() for v in (x, score, b1, b2)]
    dy = randn((t, d), dtype, 9).cuda()
    i8.expert_layer(leaves[0], gate, leaves[1], w1, leaves[2], w2, leaves[3], ACTS[act]).backward(dy)

    owner = owners(plan)
    n = len(owner)
    slot = plan.pos[:n].long()
    token = slot // k
    v1, v2 = (w.codes[..., :w.features].double() * w.scales.double()[..., None] for w in (w1, w2))
    given = dy.double()[token]
    z = pre[:n].double().requires_grad_()
    slope = torch.autograd.grad(ACTS[act](z).sum(), z)[0]
    g_out = given * score.reshape(-1)[slot].double()[:, None]
    g_hidden, g_rows = torch.empty(n, h, device="cuda").double(), torch.empty(n, d, device="cuda").double()
    for i in owner.unique().tolist():
        r = owner == i
        g_hidden[r] = g_out[r] @ v2[i]
        g_rows[r] = (g_hidden[r] * slope[r]) @ v1[i]
    g_pre = g_hidden * slope

    def per_expert(v):
        return torch.zeros(e, v.shape[1], dtype=torch.float64, device="cuda").index_add_(0, owner, v)

    step = torch.finfo(dtype).eps / 2
    wants = [torch.zeros(t, d, dtype=torch.float64, device="cuda").index_add_(0, token, g_rows), None,
             per_expert(g_pre), per_expert(g_out)]
    for leaf, want, roundings in zip(leaves, wants, (6, None, 5, 3)):
        if want is not None:
            # (f32: sums of up to max(d, h) products beside the roundings, 2^-24 each)
            err = (leaf.grad.double() - want).norm()
            assert err <= (roundings * step + (d + h) * 2.0 ** -24) * want.norm()
    dots = torch.zeros(t * k, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(dots)
    dots[slot] = (given * out[:n].double()).sum(1)
    size[slot] = (given * out[:n].double()).abs().sum(1)
    got = leaves[1].grad.reshape(-1).double()
    assert ((got - dots).abs() <= half_step(dots, dtype) * (1 + 1e-6) + (d + 1) * 2.0 ** -24 * size).all()
