"""Whole layers of 8-bit experts against 64-bit arithmetic, and the two ways they run."""
import copy

import pytest
import torch

from fastmoe_amd import FMoETransformerMLP, ScoreGate, fmoe_cuda, graphed, i8
from helpers import make_gate, randn

pytestmark = pytest.mark.gpu

ACTS = {"gelu": torch.nn.GELU(), "relu": torch.nn.ReLU(), "silu": torch.nn.SiLU()}


def parts(t, e, k, d, h, dtype, drop=0.0, seed=0):
    gate = torch.from_numpy(make_gate(t, k, e, drop=drop, seed=seed, empty=(1,))).cuda()
    x = randn((t, d), dtype, seed + 1).cuda()
    score = torch.rand(t, k, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    w1 = i8.quantize(randn((e, h, d), torch.float32, seed + 2, 0.05).cuda())
    w2 = i8.quantize(randn((e, d, h), torch.float32, seed + 3, 0.05).cuda())
    b1, b2 = randn((e, h), dtype, seed + 4).cuda(), randn((e, d), dtype, seed + 5).cuda()
    return x, gate, score, w1, b1, w2, b2


def exact(x, gate, score, w1, b1, w2, b2, act):
    """In 64 bits, but for the hidden layer's codes: these come from its values rounded to x's
    dtype, of which the layer's own are one rounding away at borders, so that a code may be one off."""
    y = torch.zeros(x.shape[0], b2.shape[1], dtype=torch.float64, device=x.device)

    def values(q):
        return q.codes[..., :q.features].double() * q.scales.double()[..., None]

    for e in range(b1.shape[0]):
        t, j = torch.nonzero(gate == e, as_tuple=True)
        if not len(t):
            continue
        h = values(i8.quantize(x[t])) @ values(w1)[e].T + b1[e].double()
        h = act(h.to(x.dtype).double()).to(x.dtype)
        out = values(i8.quantize(h)) @ values(w2)[e].T + b2[e].double()
        y.index_add_(0, t, out * score[t, j].double()[:, None])
    return y


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,e,k,d,h,drop", [(1, 2, 1, 8, 8, 0.0), (65, 4, 2, 100, 300, 0.2),
                                            (500, 70, 4, 256, 384, 0.1), (300, 4, 2, 130, 77, 0.0)])
def test_layer(t, e, k, d, h, drop, dtype, act):
    p = parts(t, e, k, d, h, dtype, drop)
    with torch.no_grad():
        y = i8.expert_layer(*p, ACTS[act])
    assert y.dtype == dtype and y.shape == (t, d)
    want = exact(*p, ACTS[act])
    # A code of the hidden layer that is one off moves a row's result by scale * weight, at most
    # max|h| / 127 of random sign for the few that are next to a border: below 1 % of a row's norm
    # with sqrt(h) of h codes off.  Beyond it: the expert row's rounding and the combine's, the
    # latter of top_k terms, each half a step of the largest value.
    step = torch.finfo(dtype).eps / 2
    err = (y.double() - want).norm(dim=1)
    assert (err <= (0.01 + 4 * step) * want.norm(dim=1) + 1e-6).all()
    # and over all rows the roundings alone, were it not for such codes
    if dtype == torch.float32:
        assert (y.double() - want).norm() <= 1e-3 * want.norm()


@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_one_call_gives_the_bits_of_the_chain(dtype, act, monkeypatch):
    p = parts(130, 6, 2, 136, 264, dtype, 0.15)
    with torch.no_grad():
        whole = i8.expert_layer(*p, ACTS[act])
    chain = i8.expert_layer(p[0].clone().requires_grad_(), *p[1:], ACTS[act])
    assert chain.requires_grad and torch.equal(whole, chain.detach())
    monkeypatch.setattr(fmoe_cuda, "_compiled", None)
    with torch.no_grad():
        assert torch.equal(i8.expert_layer(*p, ACTS[act]), whole)


def test_gradients_through_the_layer():
    """ReLU in f32: the layer is linear in between, so that its gradients are those of the weights'
    values, the signs of the hidden layer given."""
    x, gate, score, w1, b1, w2, b2 = parts(40, 4, 2, 48, 64, torch.float32, 0.1)
    leaves = [t.clone().requires_grad_() for t in (x, score, b1, b2)]
    dy = randn((40, 48), torch.float32, 9).cuda()
    i8.expert_layer(leaves[0], gate, leaves[1], w1, leaves[2], w2, leaves[3],
                    torch.nn.ReLU()).backward(dy)
    v1, v2 = (w.codes[..., :w.features].double() * w.scales.double()[..., None] for w in (w1, w2))
    zs = [t.double().clone().requires_grad_() for t in (x, score, b1, b2)]
    y = torch.zeros(40, 48, dtype=torch.float64, device="cuda")

    def straight(z):
        """The values of z's codes, with z's gradient."""
        q = i8.quantize(z.detach().float())
        return z + (q.codes[:, :z.shape[1]].double() * q.scales.double()[:, None] - z).detach()

    for e in range(4):
        t, j = torch.nonzero(gate == e, as_tuple=True)
        if not len(t):
            continue
        h = torch.relu(straight(zs[0][t]) @ v1[e].T + zs[2][e])
        out = straight(h) @ v2[e].T + zs[3][e]
        y = y.index_add(0, t, out * zs[1][t, j][:, None])
    y.backward(dy.double())
    for got, want in zip(leaves, zs):
        # (a hidden code next to a border may be one off: it enters the scores' gradient alone)
        tol = 2e-3 if got is leaves[1] else 2e-5
        assert (got.grad.double() - want.grad).norm() <= tol * want.grad.norm()
    assert (leaves[2].grad[1] == 0).all()           # an expert nobody chose


def test_layers_of_the_framework():
    gate = ScoreGate.configured(score="sigmoid", n_group=2, top_group=1)
    layer = FMoETransformerMLP(num_expert=8, d_model=128, d_hidden=256, top_k=2,
                               activation=torch.nn.GELU(), gate=gate).cuda().bfloat16()
    plain = copy.deepcopy(layer)
    assert i8.quantize_experts(layer) is layer
    x = randn((3, 40, 128), torch.bfloat16, 1).cuda()
    with torch.no_grad():
        y, z = layer(x), plain(x)
    assert y.shape == x.shape
    # two roundings to 8 bits each way, half a step of max|row| / 127 (rms 0.29 steps; max about 3
    # times the rms): 0.7 % of a product's norm each, four of them
    assert (y - z).float().norm() <= 0.03 * z.float().norm()
    # something trained in front: the gradient reaches it, the gate and the biases
    x.requires_grad_()
    layer(x).float().sum().backward()
    assert x.grad.isfinite().all() and layer.experts.b1.grad is not None
    assert layer.gate.gate.weight.grad is not None
    # the state dict carries codes and scales
    other = i8.quantize_experts(copy.deepcopy(plain))
    other.experts.w1_codes.zero_()
    other.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x.detach()), y)
        assert torch.equal(layer.experts[0](x[0].detach(), torch.tensor([40])),
                           other.experts[0](x[0].detach(), torch.tensor([40])))


def test_hooks_see_the_activation():
    layer = FMoETransformerMLP(num_expert=4, d_model=64, d_hidden=64, top_k=2,
                               activation=torch.nn.ReLU()).cuda()
    i8.quantize_experts(layer)
    x, seen = randn((20, 64), torch.float32, 1).cuda(), []
    with torch.no_grad():
        want = layer(x)
        handle = layer.experts.activation.register_forward_hook(lambda m, a, o: seen.append(o))
        assert torch.equal(layer(x), want) and len(seen) == 1
        handle.remove()


def test_replays_of_a_layer():
    layer = FMoETransformerMLP(num_expert=4, d_model=128, d_hidden=256, top_k=2,
                               activation=torch.nn.GELU()).cuda().half()
    i8.quantize_experts(layer)
    x = randn((50, 128), torch.float16, 1).cuda()
    with torch.no_grad():
        fmoe_cuda.init()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)
        torch.cuda.current_stream().wait_stream(side)
        graph, held = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph):
            y = layer(held)
        for seed in (2, 3, 4):
            held.copy_(randn((50, 128), torch.float16, seed))
            graph.replay()
            assert torch.equal(y, layer(held))
            torch.cuda.synchronize()


def test_a_trained_layer_with_its_passes_captured():
    layer = FMoETransformerMLP(num_expert=4, d_model=64, d_hidden=128, top_k=2,
                               activation=torch.nn.ReLU()).cuda()
    i8.quantize_experts(layer)
    eager = copy.deepcopy(layer)
    run = graphed(layer, randn((30, 64), torch.float32, 1).cuda().requires_grad_())
    for seed in (2, 3):
        x = randn((30, 64), torch.float32, seed).cuda().requires_grad_()
        z = x.detach().clone().requires_grad_()
        dy = randn((30, 64), torch.float32, seed + 10).cuda()
        y, w = run(x), eager(z)
        y.backward(dy)
        w.backward(dy)
        assert torch.equal(y, w) and torch.equal(x.grad, z.grad)


def test_refusals():
    x, gate, score, w1, b1, w2, b2 = parts(10, 3, 2, 16, 24, torch.float32)
    relu = torch.nn.ReLU()
    for args in ((x[:, :8], gate, score, w1, b1, w2, b2), (x, gate, score, w2, b1, w1, b2),
                 (x, gate[:5], score, w1, b1, w2, b2), (x, gate, score[:5], w1, b1, w2, b2),
                 (x.double(), gate, score.double(), w1, b1, w2, b2)):
        with pytest.raises(RuntimeError), torch.no_grad():
            i8.expert_layer(*args, relu)


def test_traces_follow_their_inputs_and_forward_mode_is_refused():
    x, gate, score, w1, b1, w2, b2 = parts(30, 4, 2, 64, 96, torch.float32)
    relu = torch.nn.ReLU()
    counts = torch.tensor([10, 0, 12, 8], device="cuda")
    with torch.no_grad():
        one = torch.jit.trace(lambda z, c: i8.linear(z, c, w1, b1), (x, counts))
        whole = torch.jit.trace(lambda z, g, s: i8.expert_layer(z, g, s, w1, b1, w2, b2, relu),
                                (x, gate, score))
        z, other = randn((30, 64), torch.float32, 7).cuda(), torch.tensor([0, 30, 0, 0], device="cuda")
        assert torch.equal(one(z, other), i8.linear(z, other, w1, b1))
        flipped = gate.flip(0)
        assert torch.equal(whole(z, flipped, score.flip(0)),
                           i8.expert_layer(z, flipped, score.flip(0), w1, b1, w2, b2, relu))
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        i8.linear(dual, counts, w1, b1)
