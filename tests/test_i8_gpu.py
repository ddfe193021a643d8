"""Rows and products in 8-bit integers against 64-bit arithmetic.

Tolerances are derived: a rounding to type t is off by eps_t / 2 of the value, and below the normal
numbers by half the smallest step; the product rounds its exact integer sum to f32, multiplies twice
and adds the bias in f32 (4 roundings of 2^-24), then rounds to t."""
import math

import numpy as np
import pytest
import torch

from fastmoe_amd import _ctypes_ops, fmoe_cuda, i8
from fastmoe_amd.functions import SegmentTable
from helpers import randn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(want, dtype):
    """Most that rounding to dtype moves `want` (f64)."""
    info = torch.finfo(dtype)
    return torch.clamp(want.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def oracle(x):
    """Codes (f64) and scales (f32) of rows x [n, k] on the CPU.  127 x / a in f64 is an exact tie
    where the quotient is one: its nearest neighbours are further away than f64's steps."""
    x = x.detach().cpu()
    top = x.float().abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top)
    safe = torch.where(ok & (top > 0), top, torch.ones_like(top)).double()
    codes = torch.where(ok, torch.round(127.0 * x.double() / safe), torch.zeros(()).double())
    scales = torch.from_numpy(top.numpy() / np.float32(127.0))
    return codes, torch.where(ok, scales, torch.tensor(float("nan")))[..., 0]


def check_rows(q, x):
    k = x.shape[-1]
    codes, scales = oracle(x)
    assert q.codes.dtype == torch.int8 and q.codes.shape[-1] == -(-k // 128) * 128
    assert torch.equal(q.codes[..., :k].cpu().double(), codes)
    assert not q.codes[..., k:].any()
    torch.testing.assert_close(q.scales.cpu(), scales, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 5), (64, 127), (7, 128), (9, 129), (1000, 300),
                                    (5, 512), (4100, 513), (4100, 1024), (3, 4096), (4097, 4096),
                                    (2, 4100), (33, 16384), (2, 16385), (1, 131072)])
def test_codes_and_scales(dtype, rows, k):
    x = randn((rows, k), dtype, rows + k).cuda()
    check_rows(i8.quantize(x), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_on_borders_go_to_the_even_code(dtype):
    """x = (j + 1/2) a / 127 for every j, with a = 127 * 2^e: exact ties in every type; beside them
    the next values on either side."""
    ties = (torch.arange(127, dtype=torch.float64) + 0.5)
    for e in (0, -9, 5):
        a = 127.0 * 2.0 ** e
        t = (ties * 2.0 ** e).to(dtype)
        row = torch.cat((torch.tensor([a], dtype=dtype), t, -t))
        near = torch.cat((torch.tensor([a], dtype=dtype), torch.nextafter(t, t * 2),
                          torch.nextafter(t, t * 0))) if dtype == torch.float32 else row
        x = torch.stack((row, near)).cuda()
        q = i8.quantize(x)
        check_rows(q, x)
        assert q.codes[0, 1:128].remainder(2).eq(0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_half_of_the_largest(dtype):
    """x = a / 2 is a tie at 63.5 for every a; it goes to 64."""
    a = randn((256, 1), dtype, 3).abs() + 0.5
    x = torch.cat((a, (a / 2).to(dtype), -(a / 2).to(dtype)), 1).cuda()
    q = i8.quantize(x)
    check_rows(q, x)
    assert (q.codes[:, 1] == 64).all() and (q.codes[:, 2] == -64).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_rows(dtype):
    info = torch.finfo(dtype)
    x = randn((9, 200), torch.float32, 5)
    x = x / x.abs().amax(-1, keepdim=True)
    x[0] = 0
    x[1] *= info.max / 2
    x[2] *= info.smallest_normal * 4
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    x[5, 0] = -float("inf")
    x[6] = 0
    x[6, 199] = info.smallest_normal * info.eps       # the smallest number there is
    x[7, :100] = -0.0
    x[8] = info.max
    x = x.to(dtype).cuda()
    q = i8.quantize(x)
    check_rows(q, x)
    got = q.dequantize(torch.float32)
    assert got[3].isnan().all() and got[4].isnan().all() and got[5].isnan().all()
    assert (got[0] == 0).all() and (got[8] == got[8, 0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 5), (1000, 300), (9000, 520), (17, 4096), (5, 777)])
def test_values(dtype, rows, k):
    q = i8.quantize(randn((rows, k), dtype, k).cuda())
    want = (q.codes[:, :k].cpu().float() * q.scales.cpu()[:, None])      # one f32 rounding
    for out in TYPES:
        assert torch.equal(q.dequantize(out).cpu(), want.to(out))


def test_leading_dimensions_strides_and_checkpoints():
    x = randn((3, 4, 300), torch.bfloat16, 1).cuda()
    q = i8.quantize(x)
    assert q.shape == x.shape and q.scales.shape == (3, 4)
    check_rows(i8.I8Tensor(q.codes.view(12, -1), q.scales.view(12), 300), x.view(12, 300))
    t = i8.quantize(x.transpose(0, 1))
    assert torch.equal(t.codes, q.codes.transpose(0, 1))
    one = i8.quantize(x[0, 0])
    assert torch.equal(one.codes, q.codes[0, 0]) and one.dequantize().shape == (300,)
    assert torch.equal(one.dequantize(), q.dequantize()[0, 0])
    # a view whose rows start at odd addresses
    odd = randn((50, 301), torch.float16, 2).cuda().reshape(-1)[1:1 + 50 * 300].view(50, 300)
    check_rows(i8.quantize(odd), odd)
    c = i8.I8Tensor.from_codes(q.codes[..., :300], q.scales[..., None])
    assert torch.equal(c.codes, q.codes) and torch.equal(c.scales, q.scales)
    empty = i8.quantize(x[:0])
    assert empty.codes.shape == (0, 4, 384) and empty.dequantize().shape == (0, 4, 300)


# ------------------------------------------------------------------ products
def product(x, counts, w, bias):
    """(y, sum of magnitudes) in f64 from the codes, on x's device; rows behind the last: zeros."""
    q = i8.quantize(x)
    k = x.shape[1]
    y = torch.zeros(x.shape[0], w.codes.shape[1], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    at = 0
    for e, n in enumerate(counts):
        r = slice(at, at + n)
        at += n
        qx, qw = q.codes[r, :k].double(), w.codes[e, :, :k].double()
        p = (qx @ qw.T) * q.scales[r].double()[:, None] * w.scales[e].double()
        b = 0 if bias is None else bias[e].double()
        y[r] = p + b
        size[r] = p.abs() + (0 if bias is None else b.abs())
    return y, size


def weights(e, out, k, seed, bias_dtype=None):
    w = i8.quantize(randn((e, out, k), torch.float32, seed, 0.02).cuda())
    b = None if bias_dtype is None else randn((e, out), bias_dtype, seed + 1).cuda()
    return w, b


def check_product(y, x, counts, w, bias):
    want, size = product(x, counts, w, bias)
    n = sum(counts)
    err = (y[:n].double() - want[:n]).abs()
    tol = half_step(want[:n], y.dtype) * (1 + 1e-6) + 4 * 2.0 ** -24 * size[:n]
    assert (err <= tol).all(), (err / tol).max().item()


CASES = [  # counts, in, out: the kernel of few rows, ...
    ([1], 1, 1), ([1, 0, 3], 5, 7), ([0, 0, 2, 0], 128, 32), ([16, 1, 17], 300, 40),
    ([3] * 70, 129, 65), ([2] * 5, 4096, 64), ([1], 1408, 2048), ([5, 0, 9], 131072, 24),
    # ... 128 x 64 tiles, with one group of stages and several, odd ones among them
    ([20, 0, 33, 40], 128, 136), ([30] * 40, 256, 520), ([50, 1, 0, 64, 20], 300, 1200),
    ([17] * 80, 640, 264), ([31, 8], 1408, 8200), ([40] * 3, 1000, 999),
    # ... 128 x 128 tiles
    ([128, 0, 300, 1], 128, 128), ([500, 129], 384, 600), ([100] * 130, 256, 264),
    ([1000, 24], 1024, 4096), ([700], 777, 333), ([257, 3], 2048, 1000),
    # ... 256 x 256 tiles
    ([6400, 0, 6300], 2048, 4096), ([12900], 2176, 4104), ([6300, 6600], 1100, 4103),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,k,n", CASES, ids=lambda c: str(c)[:24])
def test_linear(dtype, counts, k, n):
    rows = sum(counts)
    x = randn((rows, k), dtype, rows + k).cuda()
    for with_bias in (True, False):
        w, b = weights(len(counts), n, k, n, dtype if with_bias else None)
        y = i8.linear(x, torch.tensor(counts, device="cuda"), w, b)
        assert y.dtype == dtype
        check_product(y, x, counts, w, b)


def test_one_weight_for_all_rows():
    x = randn((77, 300), torch.bfloat16, 1).cuda()
    w, b = weights(1, 500, 300, 2, torch.bfloat16)
    one = i8.I8Tensor(w.codes[0], w.scales[0], 300)
    y = i8.linear(x, None, one, b[0])
    check_product(y, x, [77], w, b)
    assert torch.equal(y, i8.linear(x, torch.tensor([77]), w, b))
    assert torch.equal(i8.linear(x, None, w, b), y)
    assert i8.linear(x[:0], None, one, b[0]).shape == (0, 500)
    single = i8.linear(x[5:6], None, one)
    check_product(single, x[5:6], [1], w, None)


def test_counts_of_every_kind_and_rows_behind_the_last():
    counts = [3, 0, 40, 7]
    x = randn((64, 256), torch.float16, 1).cuda()
    w, b = weights(4, 136, 256, 2, torch.float16)
    c = torch.tensor(counts)
    seg = torch.tensor([0, 3, 3, 43, 50], dtype=torch.int32, device="cuda")
    ys = [i8.linear(x, c, w, b), i8.linear(x, c.cuda(), w, b),
          i8.linear(x, SegmentTable(seg, c.cuda()), w, b)]
    for y in ys:
        check_product(y, x, counts, w, b)
        assert torch.equal(y[:50], ys[0][:50])
    # the product itself leaves them as they were
    q = i8.quantize(x)
    out = torch.full((64, 136), 7.0, dtype=torch.float16, device="cuda")
    fmoe_cuda.i8_linear_fwd(q.codes, q.scales, w.codes, w.scales, 256, b, seg, out)
    assert torch.equal(out[:50], ys[0][:50]) and (out[50:] == 7).all()
    # device counts that claim too much or too little
    wild = torch.tensor([3, -5, 1000, 7], device="cuda")
    y = i8.linear(x, wild, w, b)
    check_product(y, x, [3, 0, 61, 0], w, b)


@pytest.mark.parametrize("counts", [[5, 2], [40, 60], [400, 200]])
def test_rows_that_are_not_finite(counts):
    x = randn((sum(counts), 512), torch.bfloat16, 1)
    x[1, 3], x[4, 500] = float("inf"), float("nan")
    w, b = weights(2, 256, 512, 2, torch.bfloat16)
    y = i8.linear(x.cuda(), torch.tensor(counts), w, b)
    bad = torch.zeros(sum(counts), dtype=torch.bool)
    bad[1] = bad[4] = True
    assert torch.equal(y.isnan().all(1).cpu(), bad) and torch.equal(y.isnan().any(1).cpu(), bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,k,n", [([3, 0, 5], 40, 24), ([70, 1, 0, 100], 300, 136), ([1], 1, 1),
                                        ([9], 129, 77), ([300, 200], 512, 1024), ([700], 300, 130),
                                        ([20], 520, 4096), ([33, 0, 17], 1000, 2048),
                                        ([2] * 70 + [40], 129, 65), ([16, 17, 32, 1], 1408, 999),
                                        ([70], 300, 600), ([64, 0, 80, 33], 4096, 1000)],
                         ids=lambda c: str(c)[:24])
def test_gradients(dtype, counts, k, n):
    """dx = dy times the weights' values.  Few rows: the result's rounding, f32 sums of f32 products
    and, for 16-bit types, 2^-17 of a term that two bf16 numbers leave.  Many: the values' rounding
    to dtype as well."""
    rows = sum(counts) + 6                       # some that nobody owns
    x = randn((rows, k), dtype, 1).cuda().requires_grad_()
    w, b = weights(len(counts), n, k, 2, dtype)
    b.requires_grad_()
    dy = randn((rows, n), dtype, 3).cuda()
    i8.linear(x, torch.tensor(counts, device="cuda"), w, b).backward(dy)
    half = torch.finfo(dtype).eps / 2
    few = dtype == torch.float32 or rows <= len(counts) * 96
    term = half if not few else 0 if dtype == torch.float32 else 2.0 ** -17
    at = 0
    for e, c in enumerate(counts):
        r = slice(at, at + c)
        at += c
        v = w.codes[e, :, :k].double() * w.scales[e].double()[:, None]
        g = dy[r].double()
        want, size = g @ v, g.abs() @ v.abs()
        # (f32's weights are rounded once, too)
        tol = half_step(want, dtype) + (term + (n + 20) * 2.0 ** -24) * size
        assert ((x.grad[r].double() - want).abs() <= tol).all()
        db, size = g.sum(0), g.abs().sum(0)
        assert ((b.grad[e].double() - db).abs() <= half_step(db, dtype) + c * 2.0 ** -24 * size).all()
    assert (x.grad[at:] == 0).all()


def test_gradients_repeat_themselves_and_keep_infinities():
    x = randn((40, 520), torch.bfloat16, 1).cuda().requires_grad_()
    w, _ = weights(1, 2048, 520, 2)
    dy = randn((40, 2048), torch.bfloat16, 3).cuda()
    dy[3, 7], dy[20, 9], dy[30, 11] = float("inf"), float("nan"), 3e38
    grads = []
    for _ in range(3):
        x.grad = None
        i8.linear(x, None, w).backward(dy)
        grads.append(x.grad)
    for g in grads[1:]:
        torch.testing.assert_close(g, grads[0], rtol=0, atol=0, equal_nan=True)
    bad = ~grads[0].isfinite().all(1)
    assert bad[3] and bad[20] and bad.sum() == 2          # 3e38 times a weight is a number
    sign = w.codes[0, 7, :520].sign()
    assert (grads[0][3][sign > 0] == float("inf")).all() and (grads[0][3][sign < 0] == -float("inf")).all()
    assert grads[0][3][sign == 0].isnan().all() and grads[0][20].isnan().all()


def test_gradient_against_differences():
    """The rows' gradient passes straight through their rounding: differences of the product with
    the weights' values, which is linear."""
    x = randn((6, 64), torch.float32, 1).cuda().requires_grad_()
    w, _ = weights(2, 32, 64, 2)
    dy = randn((6, 32), torch.float32, 3).cuda()
    i8.linear(x, torch.tensor([4, 2]), w).backward(dy)
    v = w.dequantize(torch.float32).double()

    def loss(z):
        return ((z[:4] @ v[0].T) * dy[:4]).sum() + ((z[4:] @ v[1].T) * dy[4:]).sum()

    z = x.detach().double()
    for r, c in ((0, 0), (3, 63), (5, 17)):
        step = torch.zeros_like(z)
        step[r, c] = 0.5
        slope = loss(z + step) - loss(z - step)
        # weights' values: one f32 rounding; 32 products summed in f32
        size = (dy[r].double().abs() * v[0 if r < 4 else 1][:, c].abs()).sum()
        assert abs(slope - x.grad[r, c]) <= 36 * 2.0 ** -24 * size
    bias = randn((2, 32), torch.float32, 5).cuda().requires_grad_()
    i8.linear(x.detach(), torch.tensor([4, 2]), w, bias).backward(dy)
    torch.testing.assert_close(bias.grad[1], dy[4:].sum(0), rtol=2 ** -22, atol=2 ** -22)


def test_frozen_inputs_and_second_derivatives():
    x = randn((8, 64), torch.bfloat16, 1).cuda()
    w, b = weights(1, 32, 64, 2, torch.bfloat16)
    b.requires_grad_()
    y = i8.linear(x, None, w, b)
    y.sum().backward()
    assert torch.equal(b.grad, torch.full_like(b, 8.0))
    with torch.no_grad():
        assert not i8.linear(x, None, w, b).requires_grad
    x.requires_grad_()
    y = i8.linear(x, None, w, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_outputs_and_rows_beyond_32_bits():
    """Rows of output past 2^32 bytes, codes past 2^31: first and last rows are right."""
    rows, k, n = 150000, 256, 16384                  # 4.9 GB of output in bf16
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough memory")
    x = torch.randn(rows, k, device="cuda", dtype=torch.bfloat16,
                    generator=torch.Generator("cuda").manual_seed(1))
    w, b = weights(1, n, k, 2, torch.bfloat16)
    y = i8.linear(x, None, w, b)
    for r in (slice(0, 70), slice(65500, 65600), slice(131060, 131100), slice(rows - 70, rows)):
        check_product(y[r], x[r], [y[r].shape[0]], w, b)
    del y
    x = torch.zeros(140000, 16384, device="cuda", dtype=torch.bfloat16)      # 2.3 GB of codes
    x[-3:] = randn((3, 16384), torch.bfloat16, 5).cuda()
    w, b = weights(1, 8, 16384, 3, torch.bfloat16)
    y = i8.linear(x, None, w, b)
    check_product(y[-3:], x[-3:], [3], w, b)
    assert torch.equal(y[:100], b.expand(100, 8))
    q = i8.quantize(x)
    assert torch.equal(q.codes[-3:], i8.quantize(x[-3:]).codes)
    assert torch.equal(q.dequantize()[-3:], i8.quantize(x[-3:]).dequantize())


@pytest.mark.parametrize("rows", [3, 60, 200])
def test_the_largest_sums_fit(rows):
    """131072 products of 127 * 127 are just below 2^31."""
    x = torch.ones(rows, 131072, device="cuda")
    x[1] = -1
    w = i8.quantize(torch.ones(1, 8, 131072, device="cuda"))
    y = i8.linear(x, None, w)
    # two scales of 1 / 127, the sum, two products: 5 roundings of 2^-24
    assert ((y - 131072 * x[:, :8]).abs() <= 5 * 2.0 ** -24 * 131072).all()


def test_no_rows_and_experts_without_any():
    w, b = weights(3, 16, 40, 2, torch.bfloat16)
    b.requires_grad_()
    for rows in (0, 4):
        x = torch.ones(rows, 40, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        for counts in (torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64).cuda()):
            b.grad = x.grad = None
            y = i8.linear(x, counts, w, b)
            assert y.shape == (rows, 16)
            y.backward(torch.ones_like(y))
            assert not x.grad.any() and not b.grad.any()


def test_weights_changed_before_the_backward_pass_are_noticed():
    x = randn((8, 64), torch.float32, 1).cuda().requires_grad_()
    w, _ = weights(1, 32, 64, 2)
    y = i8.linear(x, None, w)
    w.scales.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_both_bindings_give_the_same_bits(monkeypatch):
    x = randn((60, 300), torch.float16, 1).cuda()
    w, b = weights(3, 136, 300, 2, torch.float16)
    counts = torch.tensor([20, 0, 37], device="cuda")
    dy = randn((60, 136), torch.float16, 3).cuda()

    def run():
        z, c = x.clone().requires_grad_(), b.clone().requires_grad_()
        y = i8.linear(z, counts, w, c)
        y.backward(dy)
        return [y.detach()[:57], z.grad, c.grad, i8.quantize(x).dequantize(torch.float32),
                i8.linear(x, None, i8.I8Tensor(w.codes[0], w.scales[0], 300), b[0])]

    want = run()
    monkeypatch.setattr(fmoe_cuda, "_compiled", None)
    for name in fmoe_cuda.OPERATORS:
        if name.startswith("i8_"):
            monkeypatch.setattr(fmoe_cuda, name, getattr(_ctypes_ops, name))
    for a, c in zip(want, run()):
        assert torch.equal(a, c)


def test_another_stream_and_graph_replays():
    w, b = weights(4, 264, 512, 2, torch.bfloat16)
    x = randn((200, 512), torch.bfloat16, 1).cuda()
    counts = torch.tensor([50, 0, 100, 50], device="cuda")
    want = i8.linear(x, counts, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = i8.linear(x, counts, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    static, held = x.clone(), counts.clone()
    with torch.cuda.graph(graph):
        out = i8.linear(static, held, w, b)
    for i, c in enumerate(([50, 0, 100, 50], [200, 0, 0, 0], [1, 2, 3, 194])):
        static.copy_(randn((200, 512), torch.bfloat16, 10 + i).cuda())
        held.copy_(torch.tensor(c))
        graph.replay()
        assert torch.equal(out, i8.linear(static, held, w, b))
        torch.cuda.synchronize()


def test_refusals():
    x = randn((8, 64), torch.bfloat16, 1).cuda()
    w, b = weights(2, 32, 64, 2, torch.bfloat16)
    c = torch.tensor([4, 4])
    for call in (lambda: i8.linear(x, None, w, b),                        # two experts, no counts
                 lambda: i8.linear(x, c, i8.I8Tensor(w.codes[0], w.scales[0], 64)),
                 lambda: i8.linear(x, torch.tensor([4, 4, 0]), w, b),
                 lambda: i8.linear(x, torch.tensor([4, 5]), w, b),
                 lambda: i8.linear(x, torch.tensor([-1, 5]), w, b),
                 lambda: i8.linear(x[:, :32], c, w, b),
                 lambda: i8.linear(x, c, w, b.float()),
                 lambda: i8.linear(x.double(), c, w),
                 lambda: i8.linear(x, c, w, b[:1]),
                 lambda: i8.linear(x.cpu(), c, w, b),
                 lambda: i8.linear(x, c, i8.I8Tensor(w.codes, w.scales, 200), b),
                 lambda: i8.linear(x, c, i8.I8Tensor(w.codes, w.scales[:, :8], 64), b),
                 lambda: i8.linear(x, c, i8.I8Tensor(w.codes.short(), w.scales, 64), b),
                 lambda: i8.quantize(x.double()),
                 lambda: i8.quantize(torch.zeros(2, 131073, device="cuda")),
                 lambda: i8.quantize(x).dequantize(torch.float64)):
        with pytest.raises(RuntimeError):
            call()
