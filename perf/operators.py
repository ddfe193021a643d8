r"""The operators of 4-bit expert layers with scored routing, as a training step or a serving
call of a user's program makes them, beside their plain forms.

  route    `functions.score_topk`: sigmoid or softmax scores of the gate's logits, a bias that
           takes part in the choice only, groups of experts, top-k, renormalised weights; with
           `train`, the gradient of the logits too
  quant    `mx.quantize` and back: blocks of 32 values, E2M1 codes, one power of two per block
  linear   `mx.linear`: rows in expert order, quantised in the call, times 4-bit weights of
           their expert, plus a bias; with `train`, the gradient of the rows too
  experts  `mx.expert_layer`: dispatch, both linear layers with the activation between them,
           weighted combine

Fields of a case: `op`; `dtype` of the floating inputs and outputs; `tokens`; `experts`; `top_k`;
route: `score`, `bias`, `groups`, `keep`; quant: `features`; linear and experts: `d_model`,
`d_hidden`, `dead` (experts that nobody chooses), `drop` (share of the slots that a capacity
limit took away), `act`; `train`.

Inputs are N(0, 1), weights N(0, 0.02) held in 4 bits, as they are kept between calls: codes two
to a byte (the even feature in the low half) in rows padded to 128 features, a scale byte
(exponent + 127) per 32 features in rows padded to 16 bytes.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
MX_BYTES = 0.5 + 1 / 32                       # of one value: its code and its share of a scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SCALE = 2.5                                   # of the routing weights
EPS = 1e-20


def _route(name, dtype, tokens, experts, top_k, score, bias, groups, keep, train):
    return dict(name=name, op="route", dtype=dtype, tokens=tokens, experts=experts, top_k=top_k,
                score=score, bias=bias, groups=groups, keep=keep, train=train)


def _quant(name, dtype, tokens, features):
    return dict(name=name, op="quant", dtype=dtype, tokens=tokens, features=features)


def _linear(name, dtype, tokens, d_model, d_hidden, experts, top_k, dead, train):
    return dict(name=name, op="linear", dtype=dtype, tokens=tokens, d_model=d_model,
                d_hidden=d_hidden, experts=experts, top_k=top_k, dead=dead, train=train)


def _experts(name, dtype, tokens, d_model, d_hidden, experts, top_k, dead, drop, act):
    return dict(name=name, op="experts", dtype=dtype, tokens=tokens, d_model=d_model,
                d_hidden=d_hidden, experts=experts, top_k=top_k, dead=dead, drop=drop, act=act)


def listed():
    return [
        # one decode step of a batch of sequences: all launch latency
        _route("route_decode", "f32", 64, 128, 8, "sigmoid", True, 8, 3, False),
        # a training step of an ordinary layer's router, softmax as in the plain gate
        _route("route_softmax", "bf16", 8192, 16, 2, "softmax", False, 1, 1, True),
        # many experts in groups, the largest training batch of one GPU
        _route("route_groups", "f32", 16384, 128, 8, "sigmoid", True, 8, 3, True),
        # activations of an odd batch in full precision, rows that end inside a block
        _quant("quant_rows", "f32", 1000, 300),
        # a checkpoint's expert weights (8 experts, 4096 -> 14336) on their way into 4 bits
        _quant("quant_weights", "bf16", 8 * 14336, 4096),
        # one decode step through an ordinary layer's first product
        _linear("linear_decode", "bf16", 32, 1024, 4096, 16, 2, 0, False),
        # word-vector sized embeddings, full precision in and out
        _linear("linear_odd", "f32", 1000, 300, 1200, 8, 2, 0, False),
        # adapters or prompts trained in front of frozen 4-bit experts
        _linear("linear_train", "bf16", 8192, 1024, 4096, 16, 2, 0, True),
        # the largest prompt through the widest experts: the product is everything
        _linear("linear_prefill", "bf16", 16384, 4096, 14336, 8, 2, 0, False),
        # one decode step through the widest experts: every weight for a few rows each
        _experts("experts_decode", "bf16", 64, 4096, 14336, 8, 2, 0, 0.0, "gelu"),
        # a ragged prompt through many narrow experts, some never chosen, some slots dropped
        _experts("experts_fine", "bf16", 2047, 2048, 1408, 128, 8, 13, 0.05, "gelu"),
        # a large batch in half precision through an ordinary layer
        _experts("experts_batch", "f16", 8192, 1024, 4096, 16, 2, 0, 0.0, "relu"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("route", "quant", "linear", "linear", "experts", "experts"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * rng.randint(4, 512 // groups if groups > 1 else 256)
        keep = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, experts // groups * keep))
        case = _route("", dtype, _spread(rng, 1, 16384), experts, top_k,
                      rng.choice(("sigmoid", "softmax")), rng.random() < 0.6, groups, keep,
                      rng.random() < 0.5)
    elif op == "quant":
        tokens, features = _spread(rng, 16, 65536), _spread(rng, 32, 14336)
        case = _quant("", dtype, min(tokens, 2 ** 28 // features), features)
    else:
        while True:
            d_model = _spread(rng, 128, 4096)
            d_hidden = int(d_model * rng.choice((0.6875, 2, 3.5, 4)))
            step = rng.choice((64, 64, 32, 1))
            d_model, d_hidden = (max(step, v // step * step) for v in (d_model, d_hidden))
            experts = 2 ** rng.randint(2, 7)
            top_k = rng.choice((1, 2, 2, 4, 8))
            tokens = _spread(rng, 1, 16384)
            dead = experts // 10 if rng.random() < 0.25 else 0
            train = op == "linear" and rng.random() < 0.4
            products = 1 if op == "linear" and not train else 2
            if (top_k <= experts - dead and experts * d_model * d_hidden <= 2 ** 29
                    and products * tokens * top_k * d_model * d_hidden < 1.9e12):
                break
        if op == "linear":
            case = _linear("", dtype, tokens, d_model, d_hidden, experts, top_k, dead, train)
        else:
            case = _experts("", rng.choice(("bf16", "f16")), tokens, d_model, d_hidden, experts,
                            top_k, dead, rng.choice((0.0, 0.0, 0.1)),
                            rng.choice(("gelu", "relu")))
    del case["name"]
    return case


# ------------------------------------------------------------------ plain 4-bit arithmetic
def _blocks(x):
    """[..., K] f32 as [..., blocks, 32], zeros behind the last feature."""
    pad = -x.shape[-1] % 32
    x = torch.nn.functional.pad(x, (0, pad)) if pad else x
    return x.reshape(*x.shape[:-1], -1, 32)


def _exponent(b):
    """Scale bytes [..., blocks, 1] int32 of f32 blocks: floor(log2(max |x|)) - 2 + 127."""
    e = (b.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 2
    return e.clamp(min=0)


def _power(byte):
    """2^(byte - 127) as f32; byte 0 is the subnormal 2^-127."""
    return torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)


def _codes(q):
    """E2M1 codes 0..7 of |q|: nearest, ties to the even code, saturated."""
    return ((q > 0.25).int() + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5)
            + (q > 5.0))


def _round_trip(x):
    """f32 [..., K] as the values that its 4-bit form stands for."""
    b = _blocks(x)
    scale = _power(_exponent(b))
    value = torch.tensor(E2M1, device=x.device)[_codes(b.abs() / scale)]
    value = torch.copysign(value, b) * scale
    bad = ~torch.isfinite(b.abs().amax(-1, keepdim=True))
    value = torch.where(bad, float("nan"), value)
    return value.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _packed(x):
    """Codes and scales of f32 [N, K] as they are kept: rows of 64 ceil(K / 128) and of
    16 ceil(K / 512) bytes."""
    n, k = x.shape
    b = _blocks(x)
    byte = _exponent(b)
    code = _codes(b.abs() / _power(byte)) + 8 * torch.signbit(b).int()
    code = code.reshape(n, -1)
    code = torch.nn.functional.pad(code, (0, -k // 128 * -128 - code.shape[1]))
    byte = byte.reshape(n, -1)
    byte = torch.nn.functional.pad(byte, (0, -k // 512 * -16 - byte.shape[1]))
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def _values(codes, scales, k):
    """The values that codes [..., bytes] and scales stand for, f32 [..., K]."""
    one = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    at = torch.arange(256, device=codes.device)
    pairs = torch.stack((one[at & 15], one[at >> 4]), -1)
    v = pairs[codes.int()].reshape(*codes.shape[:-1], -1)[..., :k]
    scale = _power(scales[..., :-(-k // 32)].int())
    return (_blocks(v) * scale[..., None]).reshape(*v.shape[:-1], -1)[..., :k]


# ------------------------------------------------------------------ inputs
def _choices(case, gen):
    """Distinct experts per token, uniform over the live ones, [T, k]; -1 where dropped."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    p = torch.rand(t, e, device="cuda", generator=gen)
    for i in range(case["dead"]):
        p[:, i * e // case["dead"]] = -1.0
    idx = p.sort(dim=-1, descending=True, stable=True)[1][:, :k].contiguous()
    if case.get("drop"):
        idx[torch.rand(t, k, device="cuda", generator=gen) < case["drop"]] = -1
    return idx


def _weights(n_expert, out, inp, gen):
    parts = [_packed(torch.randn(out, inp, device="cuda", generator=gen) * 0.02)
             for _ in range(n_expert)]
    return torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])


def _padded(counts):
    """Expert-ordered rows as [experts, most rows]: the row of every place (the row count where
    it is empty) and the place of every row."""
    n, most = int(counts.sum()), max(1, int(counts.max()))
    start = torch.cumsum(counts, 0) - counts
    col = torch.arange(most, device=counts.device)
    row = torch.where(col < counts[:, None], start[:, None] + col, n)
    expert = torch.repeat_interleave(torch.arange(len(counts), device=counts.device), counts)
    place = expert * most + torch.arange(n, device=counts.device) - start[expert]
    return row, place


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    state = {"case": case}
    t = case["tokens"]
    if case["op"] == "route":
        e = case["experts"]
        # biases as a balancing rule leaves them: small against the scores' spread
        bias = torch.randn(e, device="cuda", generator=gen) * 0.05 if case["bias"] else None
        state |= {"logits": randn(t, e).requires_grad_(case["train"]), "bias": bias,
                  "dweight": randn(t, case["top_k"])}
        return state
    if case["op"] == "quant":
        return state | {"x": randn(t, case["features"])}
    d, h, e = case["d_model"], case["d_hidden"], case["experts"]
    idx = _choices(case, gen)
    counts = torch.bincount(idx[idx >= 0], minlength=e)
    state["counts"] = counts
    state["row"], state["place"] = _padded(counts)
    state["w1"], state["b1"] = _weights(e, h, d, gen), randn(e, h, scale=0.02)
    if case["op"] == "linear":
        state |= {"x": randn(t * case["top_k"], d).requires_grad_(case["train"]),
                  "dy": randn(t * case["top_k"], h)}
        return state
    score = torch.rand(t, case["top_k"], device="cuda", generator=gen) + 0.1
    state |= {"x": randn(t, d), "idx": idx, "score": (score / score.sum(-1, True)).to(dtype),
              "w2": _weights(e, d, h, gen), "b2": randn(e, d, scale=0.02)}
    return state


# ------------------------------------------------------------------ plain forms
def _plain_route(case, logits, bias, dweight):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    l = logits.detach().float()
    if case["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        s = torch.exp(l - l.amax(-1, keepdim=True))
        s = s / s.double().sum(-1, keepdim=True).float()
    v = s if bias is None else s + bias
    if case["groups"] > 1:
        by = v.view(t, case["groups"], -1)
        best = by.sort(dim=-1, descending=True)[0][..., :2]
        best = best.sum(-1).sort(dim=-1, descending=True, stable=True)[1][:, :case["keep"]]
        kept = torch.zeros(t, case["groups"], dtype=torch.bool, device=l.device)
        kept.scatter_(1, best, True)
        v = torch.where(kept[..., None], by, float("-inf")).view(t, e)
    idx = v.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    chosen = s.gather(1, idx)
    total = chosen.sum(-1, keepdim=True) + EPS
    weight = (chosen / total * SCALE).to(logits.dtype)
    if not case["train"]:
        return [idx, weight]
    dw = dweight.float()
    ds = (dw - (dw * chosen).sum(-1, keepdim=True) / total) * (SCALE / total)
    ds = torch.zeros_like(s).scatter_(1, idx, ds)
    if case["score"] == "sigmoid":
        dl = ds * s * (1 - s)
    else:
        dl = s * (ds - (ds * s).sum(-1, keepdim=True))
    return [idx, weight, dl.to(logits.dtype)]


def _by_expert(rows, row):
    """Expert-ordered f32 rows [n, K] as [experts, most rows, K], zeros in empty places."""
    return torch.cat((rows, rows.new_zeros(1, rows.shape[1])))[row]


def _plain_product(rows, state, name, k):
    """Padded f32 rows [E, most, K] times their expert's weight, plus its bias."""
    w = _values(*state["w" + name], k)
    return torch.bmm(rows, w.transpose(1, 2).contiguous()) + state["b" + name].float()[:, None]


def _plain_linear(case, state):
    x, d, h = state["x"].detach(), case["d_model"], case["d_hidden"]
    n = len(state["place"])
    y = _plain_product(_by_expert(_round_trip(x.float()), state["row"]), state, "1", d)
    y = y.reshape(-1, h)[state["place"]].to(x.dtype)
    if not case["train"]:
        return [y]
    dy = _by_expert(state["dy"].float()[:n], state["row"])
    dx = torch.bmm(dy, _values(*state["w1"], d)).reshape(-1, d)[state["place"]]
    return [y, dx.to(x.dtype)]


def _activation(case, x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5))) if case["act"] == "gelu" else x.relu()


def _plain_experts(case, state):
    x, idx, k = state["x"], state["idx"].reshape(-1), case["top_k"]
    n, d, h = len(state["place"]), case["d_model"], case["d_hidden"]
    # live slots in expert order; dropped ones (-1) sort to the front
    order = idx.sort(stable=True)[1][idx.numel() - n:]
    rows = _by_expert(_round_trip(x.float())[order // k], state["row"])
    hidden = _round_trip(_activation(case, _plain_product(rows, state, "1", d)))
    y = _plain_product(hidden, state, "2", h).reshape(-1, d)[state["place"]]
    slots = y.new_zeros(idx.numel(), d)
    slots[order] = y
    score = state["score"].float()[..., None]
    return [(slots.view(-1, k, d) * score).sum(1).to(x.dtype)]


# ------------------------------------------------------------------ the framework's calls
def _own(case, state):
    from fastmoe_amd import functions, mx

    if case["op"] == "route":
        logits = state["logits"]
        idx, weight = functions.score_topk(
            logits, case["top_k"], bias=state["bias"], score=case["score"],
            n_group=case["groups"], top_group=case["keep"], renormalize=True, scale=SCALE)
        if not case["train"]:
            return [idx, weight]
        logits.grad = None
        weight.backward(state["dweight"])
        return [idx, weight.detach(), logits.grad]
    if case["op"] == "quant":
        return [mx.quantize(state["x"]).dequantize(state["x"].dtype)]
    w1 = mx.MXTensor(*state["w1"], case["d_model"])
    if case["op"] == "linear":
        x = state["x"]
        y = mx.linear(x, state["counts"], w1, state["b1"])
        if not case["train"]:
            return [y]
        x.grad = None
        y.backward(state["dy"])
        return [y.detach(), x.grad]
    w2 = mx.MXTensor(*state["w2"], case["d_hidden"])
    act = torch.nn.GELU() if case["act"] == "gelu" else torch.nn.ReLU()
    return [mx.expert_layer(state["x"], state["idx"], state["score"], w1, state["b1"], w2,
                            state["b2"], act)]


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["op"] == "route":
        return _plain_route(case, state["logits"], state["bias"], state["dweight"])
    if case["op"] == "quant":
        return [_round_trip(state["x"].float()).to(state["x"].dtype)]
    return _plain_linear(case, state) if case["op"] == "linear" else _plain_experts(case, state)


# ------------------------------------------------------------------ what a pass cannot avoid
def _live(case):
    """Expected number of experts with rows."""
    e = case["experts"] - case["dead"]
    return e * (1 - (1 - 1 / e) ** (case["tokens"] * case["top_k"]))


def work(case):
    t, s = case["tokens"], SIZE[case["dtype"]]
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        b = t * e * s + t * k * (8 + s) + (4 * e if case["bias"] else 0)
        if case["train"]:
            b += t * k * s + t * e * s
        return {"bytes": b, "flops": 10.0 * t * e}
    if case["op"] == "quant":
        return {"bytes": 2.0 * t * case["features"] * s, "flops": 0}
    d, h, e = case["d_model"], case["d_hidden"], case["experts"]
    rows = t * case["top_k"] * (1 - case.get("drop", 0.0))
    weight = _live(case) * (d * h * MX_BYTES)
    if case["op"] == "linear":
        b = weight + _live(case) * h * s + rows * (d + h) * s
        if case["train"]:
            b += rows * (d + h) * s
        return {"bytes": b, "flops": (4.0 if case["train"] else 2.0) * rows * d * h}
    b = 2 * weight + _live(case) * (d + h) * s + 2.0 * t * d * s + t * case["top_k"] * (8 + s)
    return {"bytes": b, "flops": 4.0 * rows * d * h}


# ------------------------------------------------------------------ in 64 bits
def _exact_quantised(x):
    """What MXFP4 makes of f64 [n, K]: per block of 32 the power of two two below the largest
    magnitude's own, each value at the nearest of the sixteen, halfway ones at the even code."""
    n, k = x.shape
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    out = x.new_zeros(n, -(-k // 32) * 32)
    out[:, :k] = x
    v = out.view(n, -1, 32)
    _, e = torch.frexp(v.abs().max(dim=-1, keepdim=True).values)     # m in [1/2, 1): floor + 1
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device),
                     (e.double() - 3).clamp(min=-127))
    r = (v.abs() / unit).clamp(max=6)
    # spacing of the grid at r: 1/2 below 2, 1 below 4, 2 above; round() takes ties to even
    step = 0.5 * (1 + (r >= 2).double() + 2 * (r >= 4).double())
    r = torch.round(r / step) * step
    assert torch.isin(r.flatten()[:4096], grid).all()
    return (torch.sign(v) * r * unit).view(n, -1)[:, :k]


def _exact_weight(codes, scales, k):
    """f64 [N, K] of one expert."""
    low, high = codes & 15, codes >> 4
    c = torch.stack((low, high), -1).reshape(codes.shape[0], -1)[:, :k]
    mag = (c & 7).double()
    expo, man = torch.floor(mag / 2), mag % 2
    value = torch.where(expo == 0, man / 2, torch.exp2(expo - 1) * (1 + man / 2))
    value = torch.where(c >= 8, -value, value)
    power = torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)[:, :k]
    return value * power


def _exact_route(case, state):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    l = state["logits"].detach().double()
    s = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, -1)
    v = s if state["bias"] is None else s + state["bias"].double()
    if case["groups"] > 1:
        size = e // case["groups"]
        score = torch.stack([v[:, g * size:(g + 1) * size].topk(2, dim=-1)[0].sum(-1)
                             for g in range(case["groups"])], -1)
        for g in range(case["groups"]):
            better = (score > score[:, g:g + 1]).sum(-1) + (score[:, :g] == score[:, g:g + 1]).sum(-1)
            v[:, g * size:(g + 1) * size][better >= case["keep"]] = -1e9
    idx = torch.argsort(v, dim=-1, descending=True, stable=True)[:, :k]
    leaf = s.clone().requires_grad_(True)
    c = torch.gather(leaf, 1, idx)
    w = SCALE * c / c.sum(-1, keepdim=True)
    if not case["train"]:
        return [None, w.detach()]
    (ds,) = torch.autograd.grad(w, leaf, state["dweight"].double())
    dl = ds * s * (1 - s) if case["score"] == "sigmoid" else s * (ds - (ds * s).sum(-1, True))
    return [None, w.detach(), dl]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    x = state["x"].detach().double()
    if case["op"] == "quant":
        return [torch.cat([_exact_quantised(p) for p in x.split(8192)])]
    d, h, e = case["d_model"], case["d_hidden"], case["experts"]
    counts = state["counts"].tolist()
    if case["op"] == "linear":
        ys, dxs, at = [], [], 0
        for i in range(e):
            w = _exact_weight(state["w1"][0][i], state["w1"][1][i], d)
            rows = slice(at, at + counts[i])
            ys.append(_exact_quantised(x[rows]) @ w.T + state["b1"][i].double())
            if case["train"]:
                dxs.append(state["dy"][rows].double() @ w)
            at += counts[i]
        return [torch.cat(ys)] + ([torch.cat(dxs)] if case["train"] else [])
    y = torch.zeros_like(x)
    for i in range(e):
        tok, slot = torch.nonzero(state["idx"] == i, as_tuple=True)
        if not len(tok):
            continue
        w1 = _exact_weight(state["w1"][0][i], state["w1"][1][i], d)
        w2 = _exact_weight(state["w2"][0][i], state["w2"][1][i], h)
        a = _exact_quantised(x[tok]) @ w1.T + state["b1"][i].double()
        a = 0.5 * a * torch.erfc(-a * math.sqrt(0.5)) if case["act"] == "gelu" else a.clamp(min=0)
        out = _exact_quantised(a) @ w2.T + state["b2"][i].double()
        y.index_add_(0, tok, out * state["score"][tok, slot].double()[:, None])
    return [y]
