"""4-bit experts on the GPU as user programs call them: traced, under forward-mode
differentiation, with counts, dtypes and modules that differ from the plain ones."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from helpers import DTYPES, make_gate

pytestmark = pytest.mark.gpu


def _layer(n_expert=8, d_model=96, d_hidden=160, dtype=torch.bfloat16, **kwargs):
    import fastmoe_amd as fm
    from fastmoe_amd import mx

    torch.manual_seed(3)
    layer = fm.FMoETransformerMLP(num_expert=n_expert, d_model=d_model, d_hidden=d_hidden,
                                  gate=fm.ScoreGate, **kwargs).to(dtype).cuda()
    with torch.no_grad():
        for p in (layer.experts.htoh4.bias, layer.experts.h4toh.bias):
            p.normal_(0, 0.1)
    return mx.quantize_experts(layer)


# ------------------------------------------------------------------ tracing, forward mode
@pytest.mark.parametrize("act", [torch.nn.GELU(), torch.nn.ReLU(), torch.nn.SiLU()])
def test_traced_layer_follows_its_input(act):
    layer = _layer(activation=act).eval()
    rows = [torch.randn(n, 96, device="cuda").bfloat16() for n in (40, 40, 40)]
    with torch.no_grad():
        traced = torch.jit.trace(layer, rows[0], check_trace=False)
        for x in rows:
            assert torch.equal(traced(x), layer(x))
        assert not torch.equal(layer(rows[1]), layer(rows[2]))
    # and its gradients, traced with them
    traced = torch.jit.trace(layer, rows[0].clone().requires_grad_(True), check_trace=False)
    for x in rows:
        grads = []
        for run in (traced, layer):
            a = x.clone().requires_grad_(True)
            y = run(a)
            y.float().square().sum().backward()
            grads.append((y.detach(), a.grad))
        assert all(torch.equal(a, b) for a, b in zip(*grads))
        assert grads[0][1].any()


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_traced_linear_and_quantisation_follow_their_inputs(where):
    from fastmoe_amd import mx

    w = mx.quantize(torch.randn(3, 48, 96, device="cuda"))
    b = torch.randn(3, 48, device="cuda")
    run = lambda x, counts: mx.linear(x, counts, w, b)
    there_and_back = lambda x: mx.quantize(x).dequantize(torch.float32)
    counts = [torch.tensor(c, device=where) for c in ([10, 0, 20], [0, 30, 0], [7, 11, 12])]
    rows = [torch.randn(30, 96, device="cuda") for _ in counts]
    with torch.no_grad():
        traced = torch.jit.trace(run, (rows[0], counts[0]), check_trace=False)
        back = torch.jit.trace(there_and_back, rows[0], check_trace=False)
        for x, c in zip(rows, counts):
            assert torch.equal(traced(x, c), run(x, c))
            assert torch.equal(back(x), there_and_back(x))


def test_forward_mode_differentiation_is_refused():
    from fastmoe_amd import mx

    layer = _layer().eval()
    for p in layer.parameters():
        p.requires_grad_(False)
    ex = layer.experts
    x = torch.randn(20, 96, device="cuda").bfloat16()
    idx, score = layer.gate(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for act in (torch.nn.GELU(), torch.nn.SiLU()):
            with pytest.raises((RuntimeError, NotImplementedError)):
                mx.expert_layer(dual, idx, score, ex.w1, ex.b1, ex.w2, ex.b2, act)
        with pytest.raises((RuntimeError, NotImplementedError)):
            mx.expert_layer(x, idx, forward_ad.make_dual(score, torch.ones_like(score)), ex.w1,
                            ex.b1, ex.w2, ex.b2, torch.nn.GELU())
        with pytest.raises((RuntimeError, NotImplementedError)):
            mx.linear(dual, torch.tensor([20] + [0] * 7), ex.w1, ex.b1)
        # codes carry no tangent, and nothing else is lost
        q = mx.quantize(dual)
        assert torch.equal(q.codes, mx.quantize(x).codes)
        y = mx.expert_layer(x, idx, score, ex.w1, ex.b1, ex.w2, ex.b2, torch.nn.GELU())
    with torch.no_grad():
        assert torch.equal(y, layer(x))


@pytest.mark.parametrize("act", [torch.nn.GELU(), torch.nn.ReLU(), torch.nn.SiLU()])
def test_operator_by_operator_gives_the_same_bits(act):
    """While somebody watches the single operators, the layer runs them one by one."""
    from fastmoe_amd import fmoe_cuda

    layer = _layer(activation=act).eval()
    x = torch.randn(50, 96, device="cuda").bfloat16()

    def both(fn):
        a = fn()
        names = []
        fmoe_cuda.profile_hook = lambda name, *events: names.append(name)
        try:
            b = fn()
        finally:
            fmoe_cuda.profile_hook = None
        assert "route" in names
        return zip(a, b)

    def train():
        layer.zero_grad()
        a = x.clone().requires_grad_(True)
        y = layer(a)
        y.float().square().sum().backward()
        return [y.detach(), a.grad, layer.experts.b1.grad.clone(), layer.experts.b2.grad.clone()]

    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in both(lambda: [layer(x)]))
    assert all(torch.equal(a, b) for a, b in both(train))


# ------------------------------------------------------------------ hooks
@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("act", [torch.nn.GELU, torch.nn.ReLU, torch.nn.SiLU])
def test_hooks_on_the_activation_run(act, grads):
    from fastmoe_amd import mx

    layer = _layer(activation=act()).eval()
    ex, x = layer.experts, torch.randn(30, 96, device="cuda").bfloat16().requires_grad_(grads)
    idx, score = (t.detach() for t in layer.gate(x))
    live = int((idx >= 0).sum())
    counts = torch.tensor([5, 0, 10, 15, 0, 0, 0, 0])
    calls = {"layer": lambda: layer(x), "experts": lambda: ex(x, counts),
             "function": lambda: mx.expert_layer(x, idx, score, ex.w1, ex.b1, ex.w2, ex.b2,
                                                 ex.activation)}
    with torch.set_grad_enabled(grads):
        for name, call in calls.items():
            seen = []
            plain = call()
            rows = 30 if name == "experts" else live
            hooks = [ex.activation.register_forward_hook(lambda m, i, o: seen.append(o.shape)),
                     ex.activation.register_forward_pre_hook(lambda m, i: seen.append("before"))]
            if grads:
                hooks.append(ex.activation.register_full_backward_hook(
                    lambda m, i, o: seen.append("back")))
            watched = call()
            if grads:
                watched.float().sum().backward()
            for h in hooks:
                h.remove()
            assert seen[0] == "before" and seen[1] == (rows, 160), name
            assert seen[2:] == (["back"] if grads else []), name
            # the chain of single operators: the fused form but for the hidden layer's rounding
            err = (watched - plain).float().norm() / plain.float().norm()
            assert err < 0.05, name
            # and what a hook returns counts
            h = ex.activation.register_forward_hook(lambda m, i, o: o * 0)
            none = call()
            h.remove()
            b2 = ex.b2.detach()
            if name == "experts":
                want = b2.repeat_interleave(counts.cuda(), 0)
                assert torch.equal(none, want)
            else:
                want = (b2[idx].float() * score[..., None].float()).sum(1)
                assert (none.float() - want).abs().max() <= 2 ** -7 * want.abs().max()
        ex.activation.forward = lambda t: t * 0
        assert torch.equal(ex(x, counts), b2.repeat_interleave(counts.cuda(), 0))
        assert torch.equal(layer(x), none)


@pytest.mark.parametrize("act", [torch.nn.GELU, torch.nn.ReLU])
def test_hooks_on_all_modules_see_what_they_saw_before(act):
    import fastmoe_amd as fm
    from fastmoe_amd import mx

    full = fm.FMoETransformerMLP(num_expert=4, d_model=64, d_hidden=96, activation=act()).cuda()
    x = torch.randn(20, 64, device="cuda")

    def seen(layer):
        names = []
        hook = torch.nn.modules.module.register_module_forward_hook(
            lambda m, *_: names.append(type(m).__name__))
        try:
            with torch.no_grad():
                layer(x)
        finally:
            hook.remove()
        return [n.replace("MXExpert", "_Expert") for n in names]

    before = seen(full)
    assert seen(mx.quantize_experts(full)) == before


# ------------------------------------------------------------------ counts that leave rows over
def _nan_memory(*shape, dtype):
    """Leaves NaN behind in the memory that the next tensor of this size gets."""
    held = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts", [[0, 0, 0], [7, 0, 60], [100, 30, 0], [0, 0, 131]])
@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_rows_that_no_expert_owns_have_no_gradient(dt, counts, where):
    from fastmoe_amd import mx

    rows, k, n, dtype = 131, 72, 40, DTYPES[dt]
    w = mx.quantize(torch.randn(3, n, k, device="cuda"))
    counts = torch.tensor(counts)
    live = int(counts.sum())
    dy = torch.randn(rows, n, device="cuda").to(dtype)
    x = torch.randn(rows, k, device="cuda").to(dtype).requires_grad_(True)
    y = mx.linear(x, counts.to(where), w)
    _nan_memory(rows, k, dtype=dtype)
    y.backward(dy)
    assert not x.grad[live:].any()
    # the covered rows as if the others were not there
    z = x.detach()[:live].clone().requires_grad_(True)
    mx.linear(z, counts, w).backward(dy[:live])
    assert torch.equal(x.grad[:live], z.grad)


def test_both_bindings_clear_what_no_expert_owns():
    from fastmoe_amd import _ext, fmoe_cuda, mx

    w = mx.quantize(torch.randn(2, 40, 300, device="cuda"))
    dy = torch.randn(3000, 40, device="cuda").bfloat16()
    for bounds in ([0, 0, 0], [0, 1000, 1777], [0, 5, 3000]):
        seg = torch.tensor(bounds, dtype=torch.int32).cuda()
        got = []
        for ops in (fmoe_cuda.ctypes_ops, _ext.load()):
            _nan_memory(3000, 300, dtype=torch.bfloat16)
            got.append(ops.mx_linear_bwd(dy, seg, w.codes, w.scales, 300)[0])
        assert torch.equal(*got) and not got[0][bounds[-1]:].any()


# ------------------------------------------------------------------ dtypes
def test_layer_takes_rows_of_another_dtype_as_before():
    """`_Expert` casts its rows to its parameters' dtype; so do the experts in its place."""
    import fastmoe_amd as fm
    from fastmoe_amd import mx

    torch.manual_seed(0)
    layer = fm.FMoETransformerMLP(num_expert=4, d_model=64, d_hidden=96).cuda().eval()
    x, counts = torch.randn(30, 64, device="cuda"), torch.tensor([5, 0, 10, 15])
    half = x.bfloat16()

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return layer(half)

    full = run()
    mx.quantize_experts(layer)
    ex = layer.experts
    for rows in (half, x.half(), x.double()):
        assert torch.equal(ex(rows, counts), ex(rows.float(), counts))
    for grads in (False, True):
        with torch.set_grad_enabled(grads):
            y = run()
            assert y.dtype == full.dtype == torch.float32
            assert 0.01 < (y - full).norm() / full.norm() < 0.5
            if grads:
                y.sum().backward()
                assert ex.b1.grad.dtype == torch.float32 and ex.b1.grad.any()
    # a first layer of another dtype than the second
    ex.b1.data = ex.b1.data.half()
    ex.b1.grad = None
    y = ex(half, counts)
    assert y.dtype == torch.float32 and torch.equal(y, ex(half.half(), counts))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert layer(half).dtype == torch.float32


@pytest.mark.parametrize("act", [torch.nn.GELU(), torch.nn.SiLU()])
def test_expert_layer_takes_biases_of_another_dtype(act):
    from fastmoe_amd import mx

    ex = _layer(dtype=torch.float32).experts
    x = torch.randn(40, 96, device="cuda").bfloat16()
    idx = torch.from_numpy(make_gate(40, 2, 8, drop=0.1)).cuda()
    score = torch.rand(40, 2, device="cuda")
    run = lambda b1, b2: mx.expert_layer(x, idx, score, ex.w1, b1, ex.w2, b2, act)
    b1, b2 = ex.b1.detach(), ex.b2.detach()
    with torch.no_grad():
        want = run(b1.bfloat16(), b2.bfloat16())
        assert torch.equal(run(b1.bfloat16(), b2), want) and want.dtype == torch.bfloat16
        got = run(b1, b2)
        assert (got - want).float().norm() <= 0.02 * want.float().norm()
    leaf1, leaf2 = ex.b1, ex.b2
    y = run(leaf1, leaf2)
    y.float().square().sum().backward()
    same1, same2 = (b.bfloat16().requires_grad_(True) for b in (b1, b2))
    z = run(same1, same2)
    z.float().square().sum().backward()
    assert torch.equal(y, z)
    assert torch.equal(leaf1.grad, same1.grad.float()) and torch.equal(leaf2.grad, same2.grad.float())


@pytest.mark.parametrize("k", [1, 32, 300, 513])
def test_a_single_row_without_leading_dimensions(k):
    from fastmoe_amd import fmoe_cuda, mx

    x = torch.randn(k, device="cuda")
    q, rows = mx.quantize(x), mx.quantize(x[None])
    assert q.shape == (k,) and torch.equal(q.codes, rows.codes[0])
    back = q.dequantize(torch.float32)
    assert back.shape == (k,) and torch.equal(back, rows.dequantize(torch.float32)[0])
    fmoe_cuda.profile_hook = lambda *event: None          # (the operators one by one)
    try:
        assert torch.equal(mx.quantize(x).dequantize(torch.float32), back)
    finally:
        fmoe_cuda.profile_hook = None
    with pytest.raises(RuntimeError):
        mx.linear(x, torch.tensor([1]), mx.quantize(torch.randn(1, 8, k, device="cuda")))
    with pytest.raises(RuntimeError):                      # a weight is [E, out, in]
        mx.linear(x[None], torch.tensor([1]), q)


# ------------------------------------------------------------------ GELU between the products
@pytest.mark.parametrize("k,n,counts", [
    (200, 6020, [3001, 0, 700, 2500]), (4100, 13000, [9000, 0, 4001, 7000]),
    (1030, 260, [60, 0, 200, 1] * 20), (520, 1500, [1, 30, 0, 65, 17] * 30),
    (512, 1499, [60, 0, 200, 1] * 32)])
def test_gelu_moves_only_codes_on_a_boundary(k, n, counts):
    """The kernel's GELU is within 2e-7 + 3e-7 |gelu| of gelu, the 64-bit one behind it is rounded
    to f32 here (6e-8): a code may be another only where a rounding boundary is as near as that,
    and a block's scale only where its largest value is as near to a power of two."""
    from fastmoe_amd import fmoe_cuda, mx

    g = torch.Generator(device="cuda").manual_seed(k)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    xq, wq = mx.quantize(draw(sum(counts), k)), mx.quantize(draw(len(counts), n, k) * 0.1)
    b = draw(len(counts), n)
    seg = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(counts).cumsum(0)]).int().cuda()
    y = fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k, b, seg,
                                torch.empty(sum(counts), n, device="cuda"))
    codes, scales = fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k, b,
                                                seg, 1)
    got = mx.MXTensor(codes, scales, n).dequantize(torch.float32).double()
    assert torch.isfinite(got).all()
    y = y.double()
    h = 0.5 * y * torch.special.erfc(-y / 2 ** 0.5)
    want = mx.quantize(h.float())
    row, col = torch.nonzero(got != want.dequantize(torch.float32).double(), as_tuple=True)
    assert len(row) <= 1e-4 * got.numel()
    near = lambda v: 2e-7 + 4e-7 * v.abs()
    got, other, true = got[row, col], want.dequantize(torch.float32)[row, col].double(), h[row, col]
    on_boundary = (true - (got + other) / 2).abs() <= near(true)
    block = col // 32
    mine, theirs = scales[row, block], want.scales[row, block]
    pad = torch.nn.functional.pad(h, (0, -n % 32)).view(len(h), -1, 32)
    top = pad[row, block].abs().amax(-1)
    power = torch.exp2(torch.round(torch.log2(top)))
    assert ((mine == theirs) | ((top - power).abs() <= near(top))).all()
    assert (on_boundary | (mine != theirs)).all()


def test_rows_of_dropped_slots_are_not_quantised(monkeypatch):
    from fastmoe_amd import fmoe_cuda, mx
    from fastmoe_amd.functions import RoutePlan

    w = mx.quantize(torch.randn(9, 40, 96, device="cuda"))
    plan = RoutePlan(torch.from_numpy(make_gate(200, 2, 9, drop=0.4)).cuda(), 9)
    live = int(plan.n_rows_dev)
    x = torch.randn(400, 96, device="cuda")
    y = mx.linear(x, plan.segments, w)
    assert 0 < live < 300 and torch.equal(y[:live], mx.linear(x, plan.segments.counts, w)[:live])
    told = []
    quantize = fmoe_cuda.mx_quantize
    monkeypatch.setattr(fmoe_cuda, "mx_quantize",
                        lambda x, n=None: told.append(n) or quantize(x, n))
    monkeypatch.setattr(fmoe_cuda, "profile_hook", lambda *event: None)
    assert torch.equal(mx.linear(x, plan.segments, w)[:live], y[:live])
    assert [int(n) for n in told] == [live]
    assert torch.equal(mx.linear(x, plan.segments.cpu(), w)[:live], y[:live]) and told[1] is None
    with pytest.raises(RuntimeError):                      # no segment table
        mx.linear(x, torch.empty(0, dtype=torch.int32, device="cuda"), w)


# ------------------------------------------------------------------ single experts
def test_single_experts_are_views_of_the_module():
    ex = _layer(dtype=torch.float32).experts
    x, counts = torch.randn(40, 96, device="cuda"), [5, 0, 10, 15, 0, 3, 0, 7]
    whole = ex(x, torch.tensor(counts))
    dy = torch.randn_like(whole)
    whole.backward(dy)
    grads = [b.grad.clone() for b in (ex.b1, ex.b2)]
    ex.zero_grad()
    at = 0
    assert len(list(ex)) == len(ex) == 8
    for i, (one, c) in enumerate(zip(ex, counts)):
        y = one(x[at:at + c], torch.tensor([c]))
        assert torch.equal(y, ex[i - 8](x[at:at + c], torch.tensor([c])))
        # (fewer rows may take a kernel that adds in another order: 1e-6, and a hidden value in
        # 10^5 on the other side of a rounding boundary)
        assert (y - whole[at:at + c]).norm() <= 2e-3 * whole.norm()
        assert len(list(one.parameters())) == 2
        y.backward(dy[at:at + c])
        at += c
    for b, g in zip((ex.b1, ex.b2), grads):
        assert (b.grad - g).norm() <= 2e-3 * g.norm()
    for i in (8, -9):
        with pytest.raises(IndexError):
            ex[i]


# ------------------------------------------------------------------ values of whole layers
# The hidden values are taken from the kernels, in 4 bits (other tests hold what these may be), so
# that no code on the other side of a rounding boundary blurs the rest.
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # bounds of one rounding


def _problem(dt, n_expert=6, tokens=150, top_k=3, d=160, h=288):
    from fastmoe_amd import mx

    g = torch.Generator(device="cuda").manual_seed(len(dt) + d)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    idx = torch.from_numpy(make_gate(tokens, top_k, n_expert, drop=0.15, seed=4)).cuda()
    idx[7] = -1
    w1, w2 = mx.quantize(draw(n_expert, h, d) * 0.1), mx.quantize(draw(n_expert, d, h) * 0.1)
    put = lambda a: a.to(DTYPES[dt])
    return (idx, w1, w2, put(draw(tokens, d)), put(draw(tokens, top_k).abs()),
            put(draw(n_expert, h) * 0.2), put(draw(n_expert, d) * 0.2), put(draw(tokens, d)))


def _rows(idx, n_expert):
    """(token, slot, expert) of the live rows in expert order."""
    flat = idx.reshape(-1)
    order = flat.sort(stable=True)[1][int((flat < 0).sum()):]
    return order // idx.shape[1], order % idx.shape[1], flat[order]


def _values64(w):
    return w.dequantize(torch.float32).double()


def _per_row(rows, w, expert):
    """rows @ w[expert of the row].T"""
    out = rows.new_zeros(len(rows), w.shape[1])
    for e in range(w.shape[0]):
        out[expert == e] = rows[expert == e] @ w[e].T
    return out


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", [1, 2])
def test_expert_layer_value_by_value(dt, act):
    from fastmoe_amd import fmoe_cuda, mx

    idx, w1, w2, x, score, b1, b2, _ = _problem(dt)
    module = (torch.nn.GELU(), torch.nn.ReLU())[act - 1]
    got = mx.expert_layer(x, idx, score, w1, b1, w2, b2, module)
    tok, slot, expert = _rows(idx, 6)
    seg = torch.bincount(expert, minlength=6).cumsum(0)
    seg = torch.cat([seg.new_zeros(1), seg]).int()
    q = mx.quantize(x[tok])
    hidden = mx.MXTensor(*fmoe_cuda.mx_linear_act_fwd(q.codes, q.scales, w1.codes, w1.scales,
                                                      160, b1, seg, act), 288)
    hidden, v2 = _values64(hidden), _values64(w2)
    y = _per_row(hidden, v2, expert) + b2.double()[expert]
    mag = _per_row(hidden.abs(), v2.abs(), expert) + b2.double().abs()[expert]
    s = score.double()[tok, slot, None]
    zero = torch.zeros(len(x), 160, dtype=torch.float64, device="cuda")
    want = zero.index_add(0, tok, s * y)
    # a row's sum in f32, its rounding to the type, the weighted sum, its rounding to the type
    tol = UNIT[dt] * (zero.index_add(0, tok, s * y.abs()) + want.abs()) + \
        2.0 ** -22 * (288 / 128 + 8) * zero.index_add(0, tok, s * mag)
    assert ((got.double() - want).abs() <= tol).all()
    assert not got[7].any()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", [torch.nn.GELU(), torch.nn.ReLU(), torch.nn.SiLU()])
def test_expert_layer_trains_in_every_type(dt, act):
    from fastmoe_amd import functions, mx

    idx, w1, w2, *tensors = _problem(dt)
    x, score, b1, b2 = (t.clone().requires_grad_(True) for t in tensors[:4])
    dy = tensors[4]
    got = mx.expert_layer(x, idx, score, w1, b1, w2, b2, act)
    got.backward(dy)
    got = [got.detach(), x.grad, score.grad, b1.grad, b2.grad]
    assert all(g.dtype == DTYPES[dt] for g in got)
    x, score, b1, b2 = tensors[:4]
    tok, slot, expert = _rows(idx, 6)
    counts = torch.bincount(expert, minlength=6)
    pre = mx.linear(x[tok], counts, w1, b1)
    hidden = _values64(mx.quantize(functions.apply_activation(act, pre)))
    v1, v2, s, g = _values64(w1), _values64(w2), score.double()[tok, slot, None], dy.double()[tok]
    y = _per_row(hidden, v2, expert) + b2.double()[expert]
    # the rounding of the hidden layer passes its gradient straight through
    leaf = pre.double().requires_grad_(True)
    act(leaf).backward(_per_row(s * g, v2.transpose(1, 2), expert))
    zero = torch.zeros(len(x), 160, dtype=torch.float64, device="cuda")
    by_expert = lambda a: a.new_zeros(6, a.shape[1]).index_add(0, expert, a)
    dscore = torch.zeros(idx.shape, dtype=torch.float64, device="cuda")
    dscore[tok, slot] = (g * y).sum(1)
    want = [zero.index_add(0, tok, s * y),
            zero.index_add(0, tok, _per_row(leaf.grad, v1.transpose(1, 2), expert)), dscore,
            by_expert(leaf.grad), by_expert(s * g)]
    # at most eight roundings to the type in a row (dx: the row of dy, of dh, of the activation's
    # gradient, of dx, their sum), in the norm; in f32 also sums of up to 450 terms
    tol = 8 * UNIT[dt] + 450 * 2.0 ** -24
    for a, b, name in zip(got, want, ("y", "dx", "dscore", "db1", "db2")):
        assert (a.double() - b).norm() <= tol * b.norm(), name
    assert not got[1][7].any() and not got[2][idx < 0].any()
