"""Scored top-k routing on the GPU against its statement in 64 bits."""
import numpy as np
import pytest
import torch

import mx_reference as R
from helpers import DTYPES

pytestmark = pytest.mark.gpu

# f32: a score carries at most about 3 units in the last place (exponential, sum, division),
# a weight two more operations and the k-term sum; a decision may differ from the 64-bit one
# where it rests on less than the resulting 2^-22 or so.  f16/bf16 add one rounding.
UNIT = {"f32": 2.0 ** -23, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
MARGIN = 1e-6

CASES = [  # tokens, experts, top_k, score, bias, groups, kept, group_best, renormalize
    (1, 1, 1, "sigmoid", False, 1, 1, 2, True),
    (5, 2, 2, "softmax", True, 1, 1, 2, True),
    (33, 16, 2, "softmax", False, 1, 1, 2, False),
    (257, 128, 8, "sigmoid", True, 8, 3, 2, True),
    (100, 128, 8, "softmax", True, 16, 4, 1, True),
    (64, 100, 6, "sigmoid", True, 5, 2, 2, False),
    (17, 256, 16, "sigmoid", True, 1, 1, 2, True),
    (40, 512, 8, "softmax", False, 64, 8, 2, True),
    (31, 257, 3, "sigmoid", False, 1, 1, 2, True),
    (19, 48, 12, "softmax", True, 48, 12, 2, True),      # groups of one expert
    (3000, 60, 4, "sigmoid", True, 4, 2, 2, True),
    (9, 30, 16, "softmax", True, 2, 2, 2, False),        # all groups stay
]


def _inputs(t, e, dt, seed):
    rng = np.random.default_rng(seed)
    logits = torch.from_numpy(rng.standard_normal((t, e)) * 1.5).to(DTYPES[dt])
    bias = torch.from_numpy(rng.standard_normal(e) * 0.1).float()
    return logits, bias, rng


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,e,k,kind,with_bias,g,kept,best,renorm", CASES)
def test_forward_and_backward(dt, t, e, k, kind, with_bias, g, kept, best, renorm):
    from fastmoe_amd import functions

    logits, bias, rng = _inputs(t, e, dt, t * 7 + e)
    bias = bias if with_bias else None
    x = logits.cuda().requires_grad_(True)
    idx, weight = functions.score_topk(
        x, k, bias=None if bias is None else bias.cuda(), score=kind, n_group=g, top_group=kept,
        group_best=best, renormalize=renorm, scale=2.5)
    assert idx.shape == weight.shape == (t, k) and idx.dtype == torch.int64
    assert weight.dtype == DTYPES[dt]
    exact = logits.double().numpy()
    want_idx, want, margin = R.score_topk(exact, None if bias is None else bias.double().numpy(), k,
                                          kind, g, kept, best, renorm, 2.5)
    # equal logits without a bias are exact ties in both; with one, a tie has the margin 0
    sure = margin > MARGIN
    assert sure.mean() > (0.5 if dt == "bf16" else 0.9)
    assert (idx.cpu().numpy()[sure] == want_idx[sure]).all()
    got = weight.detach().double().cpu().numpy()
    tol = 2.5 * (16 * UNIT["f32"] + (UNIT[dt] if dt != "f32" else 0))
    assert np.abs(got - want)[sure].max() <= tol
    # gradient, at the kernel's own choice
    dweight = torch.from_numpy(rng.standard_normal((t, k))).to(DTYPES[dt])
    weight.backward(dweight.cuda())
    want_dl = R.score_topk_backward(dweight.double().numpy(), exact, idx.cpu().numpy(), kind,
                                    renorm, 2.5)
    dl = x.grad.double().cpu().numpy()
    # |dl| is bounded by scale / S * k * max |dw| * s; both sums have at most 16 terms
    size = np.abs(want_dl).max(initial=0) + 2.5 * np.abs(dweight.double().numpy()).max()
    assert np.abs(dl - want_dl).max() <= size * (64 * UNIT["f32"] + (UNIT[dt] if dt != "f32" else 0))


def test_bf16_ties_go_to_the_lower_index():
    from fastmoe_amd import functions

    logits = torch.tensor([[1.0, 3.0, 3.0, 0.5, 3.0, -0.0, 0.0, 3.0]]).cuda()
    for kind in ("sigmoid", "softmax"):
        assert functions.score_topk(logits, 3, score=kind)[0].tolist() == [[1, 2, 4]]
        assert functions.score_topk(logits[:, 5:7], 2, score=kind)[0].tolist() == [[0, 1]]
    equal = torch.zeros(3, 96).cuda()
    assert functions.score_topk(equal, 4)[0].tolist() == [[0, 1, 2, 3]] * 3
    # negative values of the choice: the larger, then the lower index
    bias = torch.full((8,), -2.0).cuda()
    bias[3] = -5.0
    idx, w = functions.score_topk(torch.zeros(1, 8).cuda(), 8, bias=bias)
    assert idx.tolist() == [[0, 1, 2, 4, 5, 6, 7, 3]]
    assert torch.equal(w, torch.full((1, 8), 0.125).cuda())
    # equal groups: the lower ones
    idx, _ = functions.score_topk(torch.zeros(1, 12).cuda(), 4, n_group=4, top_group=2)
    assert idx.tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_masked_experts_and_empty_rows(kind):
    from fastmoe_amd import functions

    ninf = float("-inf")
    x = torch.full((4, 8), ninf)
    x[0, 5], x[0, 2] = 1.0, 2.0             # two experts for three slots
    x[2] = torch.arange(8.0)                # nothing masked; rows 1 and 3 have nobody
    x = x.cuda().requires_grad_(True)
    idx, w = functions.score_topk(x, 3, score=kind)
    assert idx.tolist() == [[2, 5, -1], [-1] * 3, [7, 6, 5], [-1] * 3]
    want = R.score_topk(x.detach().double().cpu().numpy(), None, 3, kind)[1]
    assert np.abs(w.detach().double().cpu().numpy() - want).max() < 1e-6
    w.backward(torch.ones_like(w) + torch.arange(3.0).cuda())
    assert torch.isfinite(x.grad).all() and not x.grad[[1, 3]].any()
    assert not x.grad[0, [0, 1, 3, 4, 6, 7]].any() and x.grad[0, 2] != 0
    # a bias of -inf takes an expert out as well; a group with one live expert counts that one
    bias = torch.tensor([0.0, ninf, 0.0, 0.0, 0.0, 0.0, 0.0, ninf]).cuda()
    idx, _ = functions.score_topk(torch.arange(8.0).view(1, 8).cuda(), 2, bias=bias, score=kind,
                                  n_group=4, top_group=1)
    # (sigmoid: .99 + .98 of experts 4 and 5 against 1.0 of expert 6 alone; softmax: .085 + .031
    # against .23)
    assert idx.tolist() == ([[5, 4]] if kind == "sigmoid" else [[6, -1]])
    # the lowest finite value masks nothing by itself: those experts come last, with weight 0
    low = torch.full((1, 4), torch.finfo(torch.float32).min).cuda()
    low[0, 2] = 0.0
    idx, w = functions.score_topk(low, 3, score=kind)
    assert idx.tolist() == [[2, 0, 1]] and w.tolist() == [[1.0, 0.0, 0.0]]


def test_nan_ranks_first_and_infinity_counts():
    from fastmoe_amd import functions

    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[0.0, nan, 5.0, inf], [1.0, 2.0, 3.0, 4.0]]).cuda()
    idx, w = functions.score_topk(x, 2, score="sigmoid")
    assert idx.tolist() == [[1, 3], [3, 2]]
    assert torch.isnan(w[0]).all() and torch.isfinite(w[1]).all()
    idx, w = functions.score_topk(x, 2, score="softmax")     # the whole row is NaN
    assert idx.tolist() == [[0, 1], [3, 2]] and torch.isnan(w[0]).all()


def test_sizes_of_zero_strides_and_leading_dimensions():
    from fastmoe_amd import functions

    idx, w = functions.score_topk(torch.empty(0, 8).cuda(), 2)
    assert idx.shape == w.shape == (0, 2)
    x = torch.randn(6, 5, 16).cuda()
    a = functions.score_topk(x, 2)
    b = functions.score_topk(x.view(30, 16), 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    wide = torch.randn(30, 40).cuda()
    a = functions.score_topk(wide[:, 4:20], 2)
    b = functions.score_topk(wide[:, 4:20].contiguous(), 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals():
    from fastmoe_amd import functions

    x = torch.randn(4, 12).cuda()
    for bad in (dict(top_k=0), dict(top_k=13), dict(top_k=2, n_group=5),
                dict(top_k=2, n_group=4, top_group=5), dict(top_k=2, n_group=4, top_group=0),
                dict(top_k=4, n_group=4, top_group=1), dict(top_k=2, group_best=3)):
        with pytest.raises(RuntimeError):
            functions.score_topk(x, **bad)
    with pytest.raises(ValueError):
        functions.score_topk(x, 2, score="tanh")
    with pytest.raises(RuntimeError):
        functions.score_topk(x.double(), 2)
    with pytest.raises(RuntimeError):
        functions.score_topk(torch.randn(4, 513).cuda(), 2)
    with pytest.raises(RuntimeError):
        functions.score_topk(torch.randn(4, 32).cuda(), 17)
    with pytest.raises(RuntimeError):
        functions.score_topk(x, 2, bias=torch.zeros(11).cuda())
    with pytest.raises(RuntimeError):
        functions.score_topk(x.cpu(), 2)
    y = x.clone().requires_grad_(True)
    idx, w = functions.score_topk(y, 2)
    with pytest.raises(RuntimeError):                  # no gradient of a gradient
        g, = torch.autograd.grad(w.sum(), y, create_graph=True)
        g.sum().backward()


def test_both_bindings_agree():
    from fastmoe_amd import _ext, fmoe_cuda

    py, cx = fmoe_cuda.ctypes_ops, _ext.load()
    x, bias = torch.randn(50, 24).cuda(), torch.randn(24).cuda()
    for score in (0, 1):
        a = py.score_topk_fwd(x, bias, 3, 4, 2, 1, score, False, 1.5)
        b = cx.score_topk_fwd(x, bias, 3, 4, 2, 1, score, False, 1.5)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        dw = torch.randn(50, 3).cuda()
        assert torch.equal(py.score_topk_bwd(dw, x, a[0], score, True, 1.5),
                           cx.score_topk_bwd(dw, x, b[0], score, True, 1.5))


def test_gate_module_balances_its_load():
    from fastmoe_amd import FMoETransformerMLP, ScoreGate

    torch.manual_seed(0)
    layer = FMoETransformerMLP(num_expert=16, d_model=64, d_hidden=96, top_k=2,
                               gate=ScoreGate.configured(n_group=4, top_group=2, scale=1.5))
    layer = layer.to(torch.bfloat16).cuda()
    gate = layer.gate
    assert gate.balance_bias.dtype == torch.float32 and gate.balance_bias.is_cuda
    assert gate.options["scale"] == 1.5 and "gate.balance_bias" in layer.state_dict()
    x = torch.randn(512, 64, dtype=torch.bfloat16).cuda()

    def spread():
        gate.load.zero_()
        y = layer(x)
        assert int(gate.load.sum()) == 1024
        return gate.load.float().std().item(), y

    before, y = spread()
    y.float().square().sum().backward()
    assert gate.gate.weight.grad.abs().sum() > 0 and gate.get_loss().item() == 0.0
    for _ in range(60):
        layer(x)
        gate.update_bias(0.01)
        assert not gate.load.any()
    assert spread()[0] < 0.5 * before
    layer.eval()
    gate.load.zero_()
    layer(x)
    assert not gate.load.any()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("e,n_group,top_group", [(17, 1, 1), (48, 4, 2), (64, 1, 1), (65, 5, 3),
                                                 (128, 8, 3), (200, 25, 4), (256, 1, 1),
                                                 (257, 1, 1), (320, 64, 9), (512, 8, 4)])
def test_many_tokens_route_as_few(e, n_group, top_group, dt):
    """However many lanes share a token, its slots, weights and gradients have the same bits."""
    from fastmoe_amd.functions import score_topk

    g = torch.Generator().manual_seed(e)
    logits = torch.randn(4611, e, generator=g).to(DTYPES[dt]).cuda()
    logits[5, : e // 2] = float("-inf")
    logits[4500] = float("-inf")
    bias = (torch.randn(e, generator=g) * 0.1).cuda()
    k = min(8, e // n_group * top_group)
    dw = torch.randn(4611, k, generator=g).to(DTYPES[dt]).cuda()
    for score in ("sigmoid", "softmax"):
        def run(rows):
            x = logits[rows].clone().requires_grad_(True)
            idx, w = score_topk(x, k, bias=bias, score=score, n_group=n_group, top_group=top_group)
            w.backward(dw[rows])
            return idx, w.detach(), x.grad

        many = run(slice(None))
        for rows in (slice(0, 1), slice(1, 700), slice(700, 2748), slice(2748, 4611)):
            for whole, part in zip(many, run(rows)):
                assert torch.equal(whole[rows], part)
