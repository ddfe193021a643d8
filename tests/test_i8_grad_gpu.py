"""The gradient of 8-bit products' rows is as exact for many rows as for few.

Terms v = dy s of a sum over n of v q, with size = sum |v q| and l1 = sum |v|.  Few rows: 2^-17 of a
term, f32 sums.  Many rows: v, scaled, is an f16 number (bf16 rows: eps / 2 = 2^-11 of a term) or two
of them (f16: 2^-22), or off by f16's smallest half step of 2^-25 where l1 is at least 2^14 and the
code a 128th part.  The product is rounded to f16, 2^-11 of it, and then to dx's type; f16 numbers that
are not subnormal there stay what they are."""
import pytest
import torch

from fastmoe_amd import FMoETransformerMLP, _ctypes_ops, fmoe_cuda, graphed, i8
from helpers import randn

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
# rows per expert up to which the gradient comes straight from the codes
FEW = {torch.float16: 512, torch.bfloat16: 96}


def rows_of(counts, dtype):
    """As many rows of f16 as pass its border where so many of bf16 pass theirs."""
    return [c * 6 if dtype == torch.float16 else c for c in counts]


def test_the_border_between_few_and_many_rows():
    from fastmoe_amd import _lib
    for dtype, code in ((torch.float16, 2), (torch.bfloat16, 3)):
        assert [_lib.load().fmoe_i8_few_rows(3 * FEW[dtype] + i, 3, code) for i in (0, 1)] == [1, 0]


def half_step(want, dtype):
    info = torch.finfo(dtype)
    return torch.clamp(want.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def weights(e, n, k, seed):
    return i8.quantize(randn((e, n, k), torch.float32, seed, 0.02).cuda())


def gradient(dy, counts, w, x_dtype=None):
    x = torch.zeros(dy.shape[0], w.features, dtype=dy.dtype, device="cuda", requires_grad=True)
    i8.linear(x, torch.tensor(counts, device="cuda"), w).backward(dy)
    return x.grad


def formula(dy, counts, w):
    """(dx, size, l1) in f64 of the rows that experts own."""
    parts, at = [], 0
    for e, c in enumerate(counts):
        v = dy[at:at + c].double() * w.scales[e].double()
        q = w.codes[e, :, :w.features].double()
        at += c
        parts.append((v @ q, v.abs() @ q.abs(), v.abs().sum(1, keepdim=True)))
    return [torch.cat(p) for p in zip(*parts)]


def check(got, dy, counts, w):
    want, size, l1 = formula(dy, counts, w)
    n = dy.shape[1]
    rows, dtype = sum(counts), dy.dtype
    bf16 = dtype == torch.bfloat16
    term = 2.0 ** -11 if bf16 else 2.0 ** -17
    twice = 1.0 if bf16 else (want.abs() < torch.finfo(dtype).smallest_normal).double()
    tol = (half_step(want, dtype) * (1 + 2.0 ** -10) + twice * 2.0 ** -11 * want.abs()
           + (term + (n + 20) * 2.0 ** -24) * size + (n + 1) * 2.0 ** -32 * l1)
    err = (got[:rows].double() - want).abs()
    big = torch.finfo(dtype).max
    fits = want.abs() + tol < big
    assert (err <= tol)[fits].all(), (err / tol)[fits].max().item()
    over = want.abs() - tol > big * (1 + torch.finfo(dtype).eps / 4)
    assert (got[:rows].double()[over] == want[over].sign() * float("inf")).all()
    assert (got[rows:] == 0).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("counts,k,n", [("few", 520, 1024), ("many", 520, 1024),
                                        ([400, 0, 500, 300], 512, 1408), ([1000], 1024, 2048)])
def test_the_error_is_that_of_the_results_rounding(dtype, counts, k, n):
    """In mean squares, with bf16's step as the unit and f16's an eighth of it: 1 / 12 for the result's
    rounding.  Of many bf16 rows, 1 / 64 of that for the terms' rounding to f16 and as much for the
    product's; and what is rounded to bf16 is then a multiple j / 8, whose errors j / 8, j = -4 .. 4, have
    the mean square (28 + 16) / 64 / 8 = (1 + 2 / 64) / 12.  Together (1 + 4 / 64) / 12: 1.031 times the
    rounding alone; all else is less.  10^5 elements leave the ratio of two norms within 0.01."""
    few = FEW[dtype]
    if isinstance(counts, str):
        counts = [few, few + (counts == "many")]
    else:
        counts = rows_of(counts, dtype)
    w = weights(len(counts), n, k, 1)
    dy = randn((sum(counts), n), dtype, 2).cuda()
    want, _, _ = formula(dy, counts, w)
    rounding = (want.to(dtype).double() - want).norm()
    assert (gradient(dy, counts, w).double() - want).norm() <= 1.041 * rounding


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("counts,k,n", [([300], 77, 333), ([100, 0, 200, 1, 300], 128, 136),
                                        ([200, 150], 300, 2049), ([120] * 70, 64, 72),
                                        ([130], 24, 9001), ([97], 1, 1), ([250], 1000, 8),
                                        ([110], 40, 131072)], ids=lambda c: str(c)[:24])
def test_many_rows(dtype, counts, k, n):
    counts = rows_of(counts, dtype)
    w = weights(len(counts), n, k, 1)
    dy = randn((sum(counts) + 5, n), dtype, 2).cuda()
    # (behind the last row anything may lie)
    dy[sum(counts):] = float("nan")
    check(gradient(dy, counts, w), dy, counts, w)


@pytest.mark.parametrize("more", [0, 1, 200])
@pytest.mark.parametrize("dtype", HALF)
def test_channels_beyond_the_range_of_16_bits(dtype, more):
    """Weights that f16 holds with few bits, not at all, or as infinities, alone and beside others."""
    rows = FEW[dtype] + more
    k, n = 136, 256
    unit = randn((1, n, k), torch.float32, 1, 0.25)
    exponents = torch.arange(n)
    for seed, (factor, grad) in enumerate(((torch.full((n,), 2.0 ** -20), 2.0 ** 9),
                                           (torch.full((n,), 2.0 ** -34), 2.0 ** 13),
                                           (torch.full((n,), 2.0 ** 20), 2.0 ** -14),
                                           (2.0 ** (exponents % 40 - 30).double(), 2.0 ** -6),
                                           (torch.where(exponents % 2 == 0, 2.0 ** -24, 1.0), 1.0))):
        w = i8.quantize((unit * factor.float()[None, :, None]).cuda())
        dy = randn((rows, n), torch.float32, seed, grad).to(dtype)
        if seed == 4:
            dy[:, 1::2] = 0           # only the channels of small weights count
            dy[:, ::2] *= 2.0 ** 10
        dy = dy.cuda()
        got = gradient(dy, [rows], w)
        assert got.isfinite().all() and got.any()
        check(got, dy, [rows], w)


@pytest.mark.parametrize("dtype", HALF)
def test_rows_with_one_value_far_above_the_others(dtype):
    """What the largest one's code of zero leaves of a column is as exact as the rest."""
    k, n, rows = 264, 4096, FEW[dtype] + 104
    w = weights(1, n, k, 1)
    dy = randn((rows, n), torch.float32, 2, 2.0 ** -10)
    dy[:, 17] = 2.0 ** 6
    dy = dy.to(dtype).cuda()
    got = gradient(dy, [rows], w)
    check(got, dy, [rows], w)
    zero = w.codes[0, 17, :k] == 0
    assert zero.any()
    want = formula(dy, [rows], w)[0][:, zero]
    # (1.031 as above; some hundred elements leave the ratio of norms within a few hundredths)
    assert (got.double()[:, zero] - want).norm() <= 1.15 * (want.to(dtype).double() - want).norm()


def test_infinities_and_the_largest_numbers():
    k, n = 520, 2048
    w = weights(1, n, k, 1)
    for dtype in HALF:
        rows = FEW[dtype] + 104
        dy = randn((rows, n), dtype, 3).cuda()
        dy[3, 7], dy[20, 9], dy[150, 0] = float("inf"), float("nan"), -float("inf")
        dy[30, 11] = torch.finfo(dtype).max
        got = gradient(dy, [rows], w)
        bad = ~got.isfinite().all(1)
        assert bad[[3, 20, 150]].all() and bad.sum() == 3
        sign = w.codes[0, 7, :k].sign()
        assert (got[3][sign > 0] == float("inf")).all() and (got[3][sign < 0] == -float("inf")).all()
        assert got[3][sign == 0].isnan().all() and got[20].isnan().all()
        keep = [i for i in range(rows) if i not in (3, 20, 150)]
        check(got[keep], dy[keep], [rows - 3], w)
    # rows whose magnitudes add up to more than f32 has, and rows of the smallest numbers
    w = i8.quantize(randn((1, n, k), torch.float32, 5, 2.0 ** -9).cuda())
    rows = 200
    dy = torch.full((rows, n), 3e38, dtype=torch.bfloat16, device="cuda")
    dy *= randn((rows, n), torch.bfloat16, 6).cuda().sign()
    dy[100:] = dy[100:].sign() * 1e-36
    dy[150:] = 0
    got = gradient(dy, [rows], w)
    check(got[:150], dy[:150], [150], w)
    assert (got[150:] == 0).all()
    # a weight that is not finite
    w.scales[0, 5] = float("nan")
    assert gradient(randn((600, n), torch.float16, 7).cuda(), [600], w).isnan().all()


def test_many_rows_repeat_themselves_in_both_bindings(monkeypatch):
    w = weights(3, 1000, 264, 1)
    for dtype in HALF:
        counts = rows_of([300, 0, 250], dtype)
        dy = randn((sum(counts) + 10, 1000), dtype, 2).cuda()
        want = gradient(dy, counts, w)
        for _ in range(3):
            assert torch.equal(gradient(dy, counts, w), want)
        with monkeypatch.context() as m:
            m.setattr(fmoe_cuda, "_compiled", None)
            for name in fmoe_cuda.OPERATORS:
                if name.startswith("i8_"):
                    m.setattr(fmoe_cuda, name, getattr(_ctypes_ops, name))
            assert torch.equal(gradient(dy, counts, w), want)


@pytest.mark.parametrize("dtype", HALF)
def test_many_rows_captured_and_on_another_stream(dtype):
    layer = FMoETransformerMLP(num_expert=2, d_model=64, d_hidden=136, top_k=2,
                               activation=torch.nn.ReLU()).cuda().to(dtype)
    i8.quantize_experts(layer)
    eager = FMoETransformerMLP(num_expert=2, d_model=64, d_hidden=136, top_k=2,
                               activation=torch.nn.ReLU()).cuda().to(dtype)
    i8.quantize_experts(eager)
    eager.load_state_dict(layer.state_dict())
    t = FEW[dtype] + 100
    run = graphed(layer, randn((t, 64), dtype, 1).cuda().requires_grad_())
    for seed in (2, 3, 4):
        x = randn((t, 64), dtype, seed).cuda().requires_grad_()
        z = x.detach().clone().requires_grad_()
        dy = randn((t, 64), dtype, seed + 10).cuda()
        y, v = run(x), eager(z)
        y.backward(dy)
        v.backward(dy)
        assert torch.equal(y, v) and torch.equal(x.grad, z.grad)
        torch.cuda.synchronize()
    w = weights(1, 136, 64, 5)
    dy = randn((t, 136), dtype, 6).cuda()
    want = gradient(dy, [t], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [gradient(dy, [t], w) for _ in range(2)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("dtype", HALF)
def test_many_rows_beyond_32_bits(dtype):
    """dy of 5.2 GB, its parts of as much or twice that; weights of 4.3 GB in f16."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    g = torch.Generator("cuda").manual_seed(1)
    for rows, e, n, k in ((40000, 1, 65536, 64), (8 * 600, 8, 16384, 16384)):
        # (random codes in place of quantised weights: less memory)
        codes = torch.randint(-127, 128, (e, n, -(-k // 128) * 128), dtype=torch.int8, device="cuda",
                              generator=g)
        codes[..., k:] = 0
        w = i8.I8Tensor(codes, torch.rand(e, n, device="cuda", generator=g) * 1e-3, k)
        dy = torch.randn(rows, n, device="cuda", generator=g, dtype=dtype)
        each = rows // e
        got = gradient(dy, [each] * e, w)
        for i in {0, e - 1}:
            one = i8.I8Tensor(codes[i:i + 1], w.scales[i:i + 1], k)
            for r in {i * each, (i + 1) * each - 40}:
                check(got[r:r + 40], dy[r:r + 40], [40], one)
        del codes, w, dy, got
