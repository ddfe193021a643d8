r"""The operators of expert layers in 8-bit integers and of tokens sorted by a routing map, as a
training step or a serving call of a user's program makes them, beside their plain forms.

  sort     `functions.MapPlan` and `functions.sort_tokens`: the tokens that each expert takes, by a
           truth value per token and expert, as rows in expert order, weighted or not; with
           `train`, the gradients of the tokens and of the weights too
  unsort   `functions.MapPlan` and `functions.unsort_tokens`: each token's rows, weighted, summed
           up; with `train`, the gradients of the rows and of the weights too
  quant    `i8.quantize` and back: one scale per row, the row's largest magnitude at 127
  linear   `i8.linear`: rows in expert order, quantised in the call, times 8-bit weights of their
           expert with a scale per output channel, plus a bias; with `train`, the gradient of the
           rows too

Fields of a case: `op`; `dtype` of the floating inputs and outputs; `tokens`; `train`; sort and
unsort: `features`, `experts`, `mean` (experts that take a token, on average), `choice` (every
expert takes equally many tokens, those with its highest logits; otherwise the highest logits of
the whole batch take part), `weight` (their dtype, or "none"); quant: `features`; linear: `d_model`,
`d_hidden`, `experts` (0: one weight for all rows), `top_k`, `dead` (experts without rows).

Inputs are N(0, 1), weights of the linear maps N(0, 0.02) held in 8 bits, as they are kept between
calls: codes in rows padded with zeros to 128 features, a scale in f32 per row.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "none": 0}


def _moved(name, op, dtype, tokens, features, experts, mean, choice, weight, train):
    return dict(name=name, op=op, dtype=dtype, tokens=tokens, features=features, experts=experts,
                mean=mean, choice=choice, weight=weight, train=train)


def _quant(name, dtype, tokens, features):
    return dict(name=name, op="quant", dtype=dtype, tokens=tokens, features=features, train=False)


def _linear(name, dtype, tokens, d_model, d_hidden, experts, top_k, dead, train):
    return dict(name=name, op="linear", dtype=dtype, tokens=tokens, d_model=d_model,
                d_hidden=d_hidden, experts=experts, top_k=top_k, dead=dead, train=train)


def listed():
    return [
        # one decode step of a batch of sequences through many experts: all launch latency
        _moved("sort_decode", "sort", "bf16", 64, 2048, 128, 8, False, "none", False),
        # a training step of an ordinary layer, the batch's highest logits
        _moved("sort_train", "sort", "bf16", 8192, 1024, 16, 2, False, "none", True),
        # word-vector sized embeddings, weights applied in front of the experts
        _moved("sort_odd", "sort", "f32", 1000, 300, 8, 2, False, "f32", True),
        # the way back of a decode step
        _moved("unsort_decode", "unsort", "bf16", 64, 2048, 128, 8, False, "f32", False),
        # experts that choose their tokens, the largest training batch of one GPU
        _moved("unsort_choice", "unsort", "bf16", 16384, 2048, 128, 8, True, "f32", True),
        # activations of an odd batch in full precision
        _quant("quant_rows", "f32", 1000, 300),
        # a checkpoint's expert weights (8 experts, 4096 -> 14336) on their way into 8 bits
        _quant("quant_weights", "bf16", 8 * 14336, 4096),
        # one decode step through an ordinary layer's first product
        _linear("linear_decode", "bf16", 32, 1024, 4096, 16, 2, 0, False),
        # one weight for all rows, as in a shared expert, a ragged batch in half precision
        _linear("linear_shared", "f16", 2047, 2048, 5632, 0, 1, 0, False),
        # many narrow experts, some never chosen
        _linear("linear_fine", "bf16", 2047, 2048, 1408, 128, 8, 13, False),
        # adapters or prompts trained in front of frozen 8-bit experts
        _linear("linear_train", "bf16", 8192, 1024, 4096, 16, 2, 0, True),
        # the largest prompt through the widest experts: the product is everything
        _linear("linear_prefill", "bf16", 16384, 4096, 14336, 8, 2, 0, False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sort", "unsort", "quant", "linear", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op in ("sort", "unsort"):
        while True:
            tokens, features = _spread(rng, 16, 16384), _spread(rng, 128, 4096)
            step = rng.choice((64, 64, 8, 1))
            features = max(step, features // step * step)
            experts, mean = _spread(rng, 4, 256), rng.choice((1, 2, 4, 8))
            if mean <= experts // 2 and tokens * mean * features <= 2 ** 27:
                break
        case = _moved("", op, dtype, tokens, features, experts, mean, rng.random() < 0.5,
                      rng.choice(("none", "f32", dtype)), rng.random() < 0.5)
    elif op == "quant":
        tokens, features = _spread(rng, 16, 65536), _spread(rng, 32, 14336)
        case = _quant("", dtype, min(tokens, 2 ** 28 // features), features)
    else:
        while True:
            d_model = _spread(rng, 128, 4096)
            d_hidden = int(d_model * rng.choice((0.6875, 2, 2.75, 3.5, 4)))
            step = rng.choice((64, 64, 32, 1))
            d_model, d_hidden = (max(step, v // step * step) for v in (d_model, d_hidden))
            experts = 2 ** rng.randint(2, 7) if rng.random() < 0.75 else 0
            top_k = rng.choice((1, 2, 2, 4, 8)) if experts else 1
            tokens = _spread(rng, 1, 16384)
            dead = experts // 10 if rng.random() < 0.25 else 0
            train = rng.random() < 0.4
            products = 2 if train else 1
            if (top_k <= max(experts - dead, 1) and experts * d_model * d_hidden <= 2 ** 29
                    and products * tokens * top_k * d_model * d_hidden < 1.9e12):
                break
        case = _linear("", dtype, tokens, d_model, d_hidden, experts, top_k, dead, train)
    del case["name"]
    return case


# ------------------------------------------------------------------ plain 8-bit arithmetic
def _codes(x):
    """Codes (as f32) and scales [..., 1] of x [..., K]: the integers nearest to 127 x / max |x|,
    ties to even, in 64 bits because a value next to a border lands on the wrong side in 32.  Rows
    of zeros have scale zero; rows with an infinity or a NaN have scale NaN and codes zero."""
    top = x.float().abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top)
    q = torch.round(127.0 * x.double() / torch.where(top > 0, top, 1.0).double())
    q = torch.where(ok, q, 0.0).float()
    return q, torch.where(ok, top / 127.0, float("nan"))


def _packed(x):
    """Codes int8 [N, 128 ceil(K / 128)] and scales [N] of f32 [N, K], as they are kept."""
    q, scale = _codes(x)
    q = torch.nn.functional.pad(q, (0, -x.shape[1] % 128))
    return q.to(torch.int8), scale[:, 0]


# ------------------------------------------------------------------ inputs
def _choices(case, gen):
    """Distinct experts per token, uniform over the live ones, [T, k]."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    p = torch.rand(t, e, device="cuda", generator=gen)
    for i in range(case["dead"]):
        p[:, i * e // case["dead"]] = -1.0
    return p.sort(dim=-1, descending=True, stable=True)[1][:, :k]


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


def _routing(case, gen):
    """(truth values [T, E], logits [T, E]): some experts better liked than others; the number of
    pairs taken is always the same."""
    t, e, mean = case["tokens"], case["experts"], case["mean"]
    logits = (torch.randn(t, e, device="cuda", generator=gen) * 0.9
              + torch.randn(e, device="cuda", generator=gen) * math.sqrt(0.19))
    taken = torch.zeros(t, e, dtype=torch.bool, device="cuda")
    if case["choice"]:
        best = logits.sort(dim=0, descending=True, stable=True)[1][:_take(case)]
        return taken.scatter_(0, best, True), logits
    best = logits.view(-1).sort(descending=True, stable=True)[1][:t * mean]
    taken.view(-1)[best] = True
    return taken, logits


def _take(case):
    """Tokens of every expert that chooses."""
    return max(1, round(case["tokens"] * case["mean"] / case["experts"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    state = {"case": case}
    t, train = case["tokens"], case["train"]
    if case["op"] in ("sort", "unsort"):
        f = case["features"]
        taken, logits = _routing(case, gen)
        state |= {"taken": taken, "rows": int(taken.sum()), "weight": None}
        if case["weight"] != "none":
            state["weight"] = (torch.sigmoid(logits).to(DTYPES[case["weight"]])
                               .requires_grad_(train))
        shapes = ((t, f), (state["rows"], f))
        have, grad = shapes if case["op"] == "sort" else shapes[::-1]
        return state | {"x": randn(*have).requires_grad_(train), "dy": randn(*grad)}
    if case["op"] == "quant":
        return state | {"x": randn(t, case["features"])}
    d, h, e = case["d_model"], case["d_hidden"], case["experts"]
    counts = (torch.bincount(_choices(case, gen).reshape(-1), minlength=e) if e
              else torch.full((1,), t, device="cuda"))
    state["counts"] = counts
    state["row"], state["place"] = _padded(counts)
    state["w"], state["b"] = _weights(max(e, 1), h, d, gen), randn(max(e, 1), h, scale=0.02)
    state |= {"x": randn(t * case["top_k"], d).requires_grad_(train), "dy": randn(t * case["top_k"], h)}
    return state


# ------------------------------------------------------------------ plain forms
def _plain_moved(case, state):
    x, dy = state["x"].detach().float(), state["dy"].float()
    dtype, taken = state["x"].dtype, state["taken"]
    expert, token = taken.t().nonzero(as_tuple=True)       # in expert order, tokens ascending
    w = None if state["weight"] is None else state["weight"].detach().float()

    def weighted(rows):
        return rows if w is None else rows * w[token, expert][:, None]

    def summed(rows):
        return torch.zeros(len(taken), rows.shape[1], device=x.device).index_add_(
            0, token, weighted(rows))

    if case["op"] == "sort":
        out = [taken.sum(0), weighted(x[token]).to(dtype)]
        there, back = x[token], dy
        grad = summed
    else:
        out = [summed(x).to(dtype)]
        there, back = x, dy[token]
        grad = lambda g: weighted(g[token])
    if case["train"]:
        out.append(grad(dy).to(dtype))
        if w is not None:
            dw = torch.zeros_like(w)
            dw[token, expert] = (there * back).sum(-1)
            out.append(dw.to(state["weight"].dtype))
    return out


def _by_expert(rows, row):
    """Expert-ordered f32 rows [n, K] as [experts, most rows, K], zeros in empty places."""
    return torch.cat((rows, rows.new_zeros(1, rows.shape[1])))[row]


def _plain_linear(case, state):
    x, d, h = state["x"].detach(), case["d_model"], case["d_hidden"]
    q, scale = _codes(x)
    codes, channel = state["w"][0][..., :d].float(), state["w"][1]
    y = torch.bmm(_by_expert(q, state["row"]), codes.transpose(1, 2).contiguous())
    y = y * _by_expert(scale, state["row"]) * channel[:, None] + state["b"].float()[:, None]
    y = y.reshape(-1, h)[state["place"]].to(x.dtype)
    if not case["train"]:
        return [y]
    dy = _by_expert(state["dy"].float(), state["row"])
    dx = torch.bmm(dy, codes * channel[..., None]).reshape(-1, d)[state["place"]]
    return [y, dx.to(x.dtype)]


# ------------------------------------------------------------------ the framework's calls
def _own(case, state):
    from fastmoe_amd import functions, i8

    x = state["x"]
    if case["op"] == "quant":
        return [i8.quantize(x).dequantize(x.dtype)]
    if case["op"] == "linear":
        codes, scales = state["w"]
        if case["experts"]:
            counts, w, b = state["counts"], i8.I8Tensor(codes, scales, case["d_model"]), state["b"]
        else:
            counts, w, b = None, i8.I8Tensor(codes[0], scales[0], case["d_model"]), state["b"][0]
        y = i8.linear(x, counts, w, b)
        if not case["train"]:
            return [y]
        x.grad = None
        y.backward(state["dy"])
        return [y.detach(), x.grad]
    weight = state["weight"]
    plan = functions.MapPlan(state["taken"], state["rows"])
    move = functions.sort_tokens if case["op"] == "sort" else functions.unsort_tokens
    y = move(x, plan, weight)
    out = [plan.counts, y.detach()] if case["op"] == "sort" else [y.detach()]
    if case["train"]:
        x.grad = None
        if weight is not None:
            weight.grad = None
        y.backward(state["dy"])
        out += [x.grad] if weight is None else [x.grad, weight.grad]
    return out


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["op"] == "quant":
        q, scale = _codes(state["x"])
        return [(q * scale).to(state["x"].dtype)]
    return _plain_linear(case, state) if case["op"] == "linear" else _plain_moved(case, state)


# ------------------------------------------------------------------ what a pass cannot avoid
def work(case):
    t, s = case["tokens"], SIZE[case["dtype"]]
    if case["op"] in ("sort", "unsort"):
        f, e = case["features"], case["experts"]
        ws = SIZE[case["weight"]]
        rows = e * _take(case) if case["choice"] else t * case["mean"]
        # the truth values, weights of the rows there are, one side in and the other out
        b = t * e + rows * ws + (t + rows) * f * s
        flops = 2.0 * rows * f
        if case["train"]:
            # the gradient in and out; for the weights' also the forward's input, and all of theirs
            b += (t + rows) * f * s
            if ws:
                b += t * e * ws + (t if case["op"] == "sort" else rows) * f * s
                flops *= 2
            flops *= 2
        return {"bytes": b, "flops": flops}
    if case["op"] == "quant":
        return {"bytes": 2.0 * t * case["features"] * s, "flops": 0}
    d, h, e = case["d_model"], case["d_hidden"], case["experts"]
    rows, live = t * case["top_k"], 1.0
    if e:
        live = (e - case["dead"]) * (1 - (1 - 1 / (e - case["dead"])) ** rows)
    b = live * (d * h + h * (4 + s)) + rows * (d + h) * s
    if case["train"]:
        b += rows * (d + h) * s
    return {"bytes": b, "flops": (4.0 if case["train"] else 2.0) * rows * d * h}


# ------------------------------------------------------------------ in 64 bits
def _exact_codes(x):
    """For f64 [n, K]: the code of x is the number of borders (k - 1/2) max / 127, k = 1 .. 127,
    that |x| passes, one on a border counting where k is even; whole rows of zeros are zeros."""
    top = x.abs().max(dim=-1, keepdim=True).values
    unit = top.clamp(min=1e-300)
    k = torch.floor(x.abs() / unit * 127)             # one of this, one less and one more
    best = torch.zeros_like(k)
    for c in (k - 1, k, k + 1):
        side = 254 * x.abs() - (2 * c - 1) * top      # whole in units of the last place
        passed = (side > 0) | ((side == 0) & (c % 2 == 0))
        best = torch.where(passed & (c >= 1) & (c <= 127), c, best)
    return torch.copysign(best, x), top / 127


def _exact_moved(case, state):
    x, dy = state["x"].detach().double(), state["dy"].double()
    taken = state["taken"]
    w = (taken if state["weight"] is None else state["weight"].detach()).double()
    tokens, rows = len(taken), state["rows"]
    sort = case["op"] == "sort"
    out = x.new_zeros(rows if sort else tokens, x.shape[1])
    dx = torch.zeros_like(x) if case["train"] else None
    dw = torch.zeros_like(w)
    at = 0
    for e in range(case["experts"]):
        t = torch.nonzero(taken[:, e]).reshape(-1)
        mine = slice(at, at + len(t))
        at += len(t)
        we = w[t, e].unsqueeze(1)
        if sort:
            out[mine] = we * x[t]
        else:
            out[t] += we * x[mine]                   # (a token once per expert)
        if not case["train"]:
            continue
        if sort:
            dx[t] += we * dy[mine]
            dw[t, e] = torch.linalg.vecdot(x[t], dy[mine])
        else:
            dx[mine] = we * dy[t]
            dw[t, e] = torch.linalg.vecdot(x[mine], dy[t])
    result = ([None] if sort else []) + [out]
    if case["train"]:
        result += [dx] if state["weight"] is None else [dx, dw]
    return result


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("sort", "unsort"):
        return _exact_moved(case, state)
    x = state["x"].detach().double()
    if case["op"] == "quant":
        parts = [_exact_codes(p) for p in x.split(8192)]
        return [torch.cat([q * unit for q, unit in parts])]
    d = case["d_model"]
    ys, dxs, at = [], [], 0
    for i, n in enumerate(state["counts"].tolist()):
        rows = slice(at, at + n)
        at += n
        if not n:
            continue
        w = state["w"][0][i, :, :d].double() * state["w"][1][i].double().unsqueeze(1)
        q, unit = _exact_codes(x[rows])
        ys.append((q * unit) @ w.T + state["b"][i].double())
        if case["train"]:
            dxs.append(state["dy"][rows].double() @ w)
    return [torch.cat(ys)] + ([torch.cat(dxs)] if case["train"] else [])
