"""Rows in MXFP4, their grouped products and the experts built on them, against plain
statements in 64 bits."""
import numpy as np
import pytest
import torch

import mx_reference as R
from helpers import DTYPES, make_gate

pytestmark = pytest.mark.gpu

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # of one rounding
SIZES = [1, 31, 32, 33, 100, 128, 300, 512, 513, 1408, 2049, 4096]


def _rows(rows, k, dt, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-6, 7, size=(rows, 1)))
    return torch.from_numpy(x).to(DTYPES[dt])


def _unpack(q):
    codes = q.codes.reshape(-1, q.codes.shape[-1]).cpu().numpy()
    scales = q.scales.reshape(-1, q.scales.shape[-1]).cpu().numpy()
    return R.unpack(codes, scales, q.features)


# ------------------------------------------------------------------ the format
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", SIZES)
def test_codes_and_scales_are_exact(dt, k):
    from fastmoe_amd import mx

    for rows in (1, 7, 300):
        x = _rows(rows, k, dt, k + rows)
        q = mx.quantize(x.cuda())
        assert q.shape == (rows, k) and q.features == k
        assert q.codes.shape[-1] == -(-k // 128) * 64 and q.scales.shape[-1] == -(-k // 512) * 16
        codes, byte = _unpack(q)
        want_codes, want_byte = R.quantize(x.double().numpy())
        assert (byte == want_byte).all() and (codes == want_codes).all()
        # nothing behind the last feature
        tail = q.codes.cpu().numpy()[:, -(-k // 2):]
        assert not tail.any()
        assert not q.scales.cpu().numpy()[:, -(-k // 32):].any()
        back = q.dequantize(DTYPES[dt])
        assert back.dtype == DTYPES[dt]
        want = torch.from_numpy(R.values(want_codes, want_byte, k)).to(DTYPES[dt])
        assert torch.equal(back.cpu(), want)


def test_ties_saturation_zeros_and_tiny_values():
    from fastmoe_amd import mx

    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 4.0])
    around = torch.cat([mids, mids * (1 + 2.0 ** -20), mids * (1 - 2.0 ** -20)])
    x = torch.zeros(12, 64)
    x[0, :33] = around.clamp(max=7.99)
    x[1] = -x[0]
    x[2, 5] = -0.0
    x[3, 40] = 2.0 ** -149                       # the smallest number there is
    x[4, 1], x[4, 2] = 2.0 ** -126, -2.0 ** -127
    x[5, 0], x[5, 1] = torch.finfo(torch.float32).max, 2.0 ** 120
    x[6, 0], x[6, 33] = float("inf"), 1.0
    x[7, 10], x[7, 50] = float("nan"), -3.0
    x[8, 0], x[8, 63] = float("-inf"), float("nan")
    x[9], x[10], x[11] = 2.0 ** -125, 3 * 2.0 ** -127, 1.0
    q = mx.quantize(x.cuda())
    codes, byte = _unpack(q)
    want_codes, want_byte = R.quantize(x.double().numpy())
    assert (byte == want_byte).all() and (codes == want_codes).all()
    back = q.dequantize(torch.float32).double().cpu().numpy()
    want = R.values(want_codes, want_byte, 64)
    assert (np.isnan(back) == np.isnan(want)).all()
    assert np.array_equal(back[~np.isnan(back)], want[~np.isnan(want)])
    assert np.isnan(back[6, :32]).all() and back[6, 33] == 1.0


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_every_code_under_extreme_scales(dt):
    from fastmoe_amd import mx

    codes = torch.arange(256, dtype=torch.uint8).view(4, 64)
    scales = torch.zeros(4, 16, dtype=torch.uint8)
    for row, group in enumerate([(0, 1, 2, 254), (120, 127, 130, 255), (103, 110, 140, 142),
                                 (255, 0, 141, 253)]):
        scales[row, :4] = torch.tensor(group, dtype=torch.uint8)
    q = mx.MXTensor(codes.cuda(), scales.cuda(), 128)
    want = R.values(*R.unpack(codes.numpy(), scales.numpy(), 128), 128)
    got = q.dequantize(DTYPES[dt]).cpu()
    want = torch.from_numpy(want).to(torch.float32).to(DTYPES[dt])
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    live = ~torch.isnan(want)
    assert torch.equal(got[live], want[live])


def test_strides_leading_dimensions_and_empty_tensors():
    from fastmoe_amd import mx

    x = torch.randn(5, 6, 200).cuda()
    q = mx.quantize(x)
    assert q.shape == (5, 6, 200) and q.dequantize().shape == (5, 6, 200)
    wide = torch.randn(30, 401).bfloat16().cuda()
    a, b = mx.quantize(wide[:, 1:301]), mx.quantize(wide[:, 1:301].clone())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    # an address that is no multiple of 16 bytes
    flat = torch.randn(8 * 64 + 1).cuda()
    a, b = mx.quantize(flat[1:].view(8, 64)), mx.quantize(flat[1:].clone().view(8, 64))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    empty = mx.quantize(torch.empty(0, 96).cuda())
    assert empty.shape == (0, 96) and empty.dequantize().shape == (0, 96)


def test_from_blocks_takes_the_tight_layout():
    from fastmoe_amd import mx

    rng = np.random.default_rng(1)
    codes = torch.from_numpy(rng.integers(0, 256, (2, 3, 80)).astype(np.uint8))
    scales = torch.from_numpy(rng.integers(100, 140, (2, 3, 5)).astype(np.uint8))
    q = mx.MXTensor.from_blocks(codes.cuda(), scales.cuda())
    assert q.shape == (2, 3, 160)
    got = q.dequantize(torch.float32).double().cpu().numpy().reshape(6, 160)
    c = codes.numpy().reshape(6, 80)
    c = np.stack([c & 15, c >> 4], -1).reshape(6, 160)
    assert np.array_equal(got, R.values(c, scales.numpy().reshape(6, 5).astype(np.int64), 160))
    with pytest.raises(ValueError):
        mx.MXTensor.from_blocks(codes, scales[..., :4])


def test_live_rows_and_the_token_form():
    from fastmoe_amd import fmoe_cuda

    x = torch.randn(40, 300).half().cuda()
    n = torch.tensor([25], dtype=torch.int32).cuda()
    whole, part = fmoe_cuda.mx_quantize(x), fmoe_cuda.mx_quantize(x, n)
    assert all(torch.equal(a[:25], b[:25]) for a, b in zip(whole, part))
    for top_k in (1, 2, 8):
        gate = torch.from_numpy(make_gate(40, top_k, 9, drop=0.2, seed=top_k)).cuda()
        pos, _, seg, inv = fmoe_cuda.route(gate, 9)
        live = int(seg[-1])
        got = fmoe_cuda.mx_quantize_tokens(x, inv, top_k)
        want = fmoe_cuda.mx_quantize(x[pos[:live] // top_k].contiguous())
        assert all(torch.equal(a[:live], b) for a, b in zip(got, want))


# ------------------------------------------------------------------ the product
def _problem(counts, k, n, dt, seed, bias=True):
    rng = np.random.default_rng(seed)
    rows, e = sum(counts), len(counts)
    x = torch.from_numpy(rng.standard_normal((rows, k))).to(DTYPES[dt])
    w = torch.from_numpy(rng.standard_normal((e * n, k)) * 0.05).float()
    b = torch.from_numpy(rng.standard_normal((e, n))).to(DTYPES[dt]) if bias else None
    return x, w, b


def _exact(x, w, b, counts, n):
    """(y, what its sums' magnitudes are) in 64 bits."""
    xq, wq = R.round_trip(x.double().numpy()), R.round_trip(w.double().numpy())
    ys, mags, at = [], [], 0
    for e, c in enumerate(counts):
        rows, we = xq[at:at + c], wq[e * n:(e + 1) * n]
        y, mag = rows @ we.T, np.abs(rows) @ np.abs(we).T
        if b is not None:
            y, mag = y + b[e].double().numpy(), mag + np.abs(b[e].double().numpy())
        ys.append(y)
        mags.append(mag)
        at += c
    return np.concatenate(ys), np.concatenate(mags)


COUNTS = [[1], [0, 3, 0, 1], [16, 17, 0, 5], [64, 1, 63, 65, 0], [300, 0, 129, 1],
          [2] * 70 + [0] * 5 + [40], [513, 260]]
SHAPES = [(32, 32), (128, 64), (300, 130), (512, 256), (640, 33), (1408, 96), (1, 1), (2080, 520)]


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "rows%d" % sum(c))
def test_product_against_64_bits(dt, counts):
    from fastmoe_amd import mx

    for k, n in SHAPES:
        x, w, b = _problem(counts, k, n, dt, k * 3 + n, bias=n != 64)
        wq = mx.quantize(w.view(len(counts), n, k).cuda())
        y = mx.linear(x.cuda(), torch.tensor(counts), wq, None if b is None else b.cuda())
        assert y.dtype == DTYPES[dt] and y.shape == (sum(counts), n)
        want, mag = _exact(x, w, b, counts, n)
        # products are exact; each matrix instruction's sum and the bias round once, in f32
        tol = UNIT[dt] * np.abs(want) + 2.0 ** -23 * (k / 128 + 4) * mag + 1e-30
        assert (np.abs(y.double().cpu().numpy() - want) <= tol).all(), (k, n)
        # device counts give the same bits
        again = mx.linear(x.cuda(), torch.tensor(counts).cuda(), wq,
                          None if b is None else b.cuda())
        assert torch.equal(y, again)


@pytest.mark.parametrize("dt,n", [("bf16", 6016), ("f32", 6016), ("f16", 6011)])
def test_many_tiles(dt, n):
    """More tiles than there are compute units, so that a workgroup runs several."""
    from fastmoe_amd import mx

    counts, k = [3001, 0, 700, 2500], 200
    x, w, b = _problem(counts, k, n, dt, 12)
    wq, xd, bd = mx.quantize(w.view(4, n, k).cuda()), x.cuda(), b.cuda()
    y = mx.linear(xd, torch.tensor(counts), wq, bd)
    again = mx.linear(xd, torch.tensor(counts), wq, bd)
    assert torch.equal(y, again)
    xv, wv = mx.quantize(xd).dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    at = 0
    for e, c in enumerate(counts):
        rows = xv[at:at + c]
        want = rows @ wv[e].T + bd[e].double()
        mag = rows.abs() @ wv[e].abs().T + bd[e].double().abs()
        tol = UNIT[dt] * want.abs() + 2.0 ** -23 * (k / 128 + 4) * mag
        assert ((y[at:at + c].double() - want).abs() <= tol).all(), e
        at += c


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("counts", [[5, 0, 1], [70, 33], [300, 129, 0]], ids=lambda c: str(sum(c)))
def test_product_with_activation_comes_out_quantised(act, counts):
    from fastmoe_amd import fmoe_cuda, mx
    from scipy.special import erfc

    for k, n in [(128, 64), (300, 130), (512, 513), (96, 32), (640, 1)]:
        x, w, b = _problem(counts, k, n, "bf16", k + n + act)
        wq = mx.quantize(w.view(len(counts), n, k).cuda())
        xq = mx.quantize(x.cuda())
        seg = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
        codes, scales = fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k,
                                                    b.cuda(), seg, act)
        got = mx.MXTensor(codes, scales, n).dequantize(torch.float32).double().cpu().numpy()
        y, _ = _exact(x, w, b, counts, n)
        y = {0: y, 1: 0.5 * y * erfc(-y * np.sqrt(0.5)), 2: np.maximum(y, 0)}[act]
        # the f32 value differs from the 64-bit one by far less than 1e-4 of its block's
        # largest: a code may differ only where a rounding boundary is as near as that
        sure = R.boundary_distance(y) > 1e-3
        assert sure.mean() > 0.9 or n == 1
        assert np.array_equal(got[sure], R.round_trip(y)[sure]), (k, n)
        # codes behind the last feature are zero: the next product runs over whole steps
        assert not codes.cpu().numpy()[:, -(-n // 2):].any()
        pad = scales.cpu().numpy()[:, :-(-n // 128) * 4]
        assert (pad != 255).all()


def test_many_tiles_come_out_quantised():
    from fastmoe_amd import fmoe_cuda, mx

    counts, k, n = [3001, 0, 700, 2500], 200, 6020
    x, w, b = _problem(counts, k, n, "bf16", 13)
    wq, xq, bd = mx.quantize(w.view(4, n, k).cuda()), mx.quantize(x.cuda()), b.cuda()
    seg = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
    y = fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k, bd.float(), seg,
                                torch.empty(sum(counts), n).cuda())
    for act in (0, 1, 2):
        codes, scales = fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k,
                                                    bd, seg, act)
        got = mx.MXTensor(codes, scales, n).dequantize(torch.float32)
        h = [y, torch.nn.functional.gelu(y.double()).float(), y.relu()][act]
        want = mx.quantize(h).dequantize(torch.float32)
        if act != 1:
            assert torch.equal(got, want)
        else:                    # the two GELUs differ by up to 1e-6
            assert (got != want).float().mean() < 1e-4


# by the rule on rows, features and tiles: tiles of 256 x 256 with fewer and with more experts
# than lanes, tiles of 128 x 128 with more experts than lanes, many small ones, the split sums
BY_RULE = {"256": ([3001, 0, 700, 2500], 2100, 8200),
           "256 odd": ([3001, 0, 700, 2500], 2100, 8203),
           "256 many": ([300, 210, 0, 393, 255, 0, 257] * 14, 2049, 3000),
           "128 many": ([60, 0, 200, 1] * 20, 513, 300),
           "64 many": ([1, 30, 0, 65, 17] * 30, 1100, 260),
           "split": ([1, 0, 2, 17, 0, 0, 3, 16], 4100, 330)}


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("case", BY_RULE)
def test_every_tile_shape(case, dt):
    from fastmoe_amd import mx

    counts, k, n = BY_RULE[case]
    g = torch.Generator(device="cuda").manual_seed(len(counts))
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    x = draw(sum(counts), k).to(DTYPES[dt])
    b = draw(len(counts), n).to(DTYPES[dt])
    wq = mx.quantize(draw(len(counts), n, k) * 0.05)
    y = mx.linear(x, torch.tensor(counts), wq, b)
    assert torch.equal(y, mx.linear(x, torch.tensor(counts).cuda(), wq, b))
    xv, at = mx.quantize(x).dequantize(torch.float32).double(), 0
    for e, c in enumerate(counts):
        rows = xv[at:at + c]
        we = mx.MXTensor(wq.codes[e], wq.scales[e], k).dequantize(torch.float32).double()
        want = rows @ we.T + b[e].double()
        mag = rows.abs() @ we.abs().T + b[e].double().abs()
        # as above: the instructions' sums and the bias in f32, then the output's rounding
        tol = UNIT[dt] * want.abs() + 2.0 ** -23 * (k / 128 + 4) * mag
        assert ((y[at:at + c].double() - want).abs() <= tol).all(), e
        at += c


@pytest.mark.parametrize("k,n,counts", [
    (4100, 13000, [9000, 0, 4001, 7000]), (1030, 4000, [900, 0, 401, 700]),
    (1030, 260, [60, 0, 200, 1] * 20), (520, 1500, [1, 30, 0, 65, 17] * 30)])
def test_every_tile_shape_comes_out_quantised(k, n, counts):
    from fastmoe_amd import fmoe_cuda, mx

    g = torch.Generator(device="cuda").manual_seed(n)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    xq, wq = mx.quantize(draw(sum(counts), k)), mx.quantize(draw(len(counts), n, k) * 0.05)
    b = draw(len(counts), n)
    seg = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
    y = fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k, b, seg,
                                torch.empty(sum(counts), n).cuda())
    for act in (0, 1, 2):
        codes, scales = fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k,
                                                    b, seg, act)
        got = mx.MXTensor(codes, scales, n).dequantize(torch.float32)
        h = [lambda: y, lambda: torch.nn.functional.gelu(y.double()).float(), lambda: y.relu()][act]()
        want = mx.quantize(h).dequantize(torch.float32)
        # sums in the same order in every tile shape; the two GELUs differ by up to 1e-6
        assert torch.equal(got, want) if act != 1 else (got != want).float().mean() < 1e-4
        tail = codes[:, -(-n // 2):]
        assert not tail.any()


# More experts than lanes, where the owner of a row tile is looked up through LDS, K of one group
# of scales, and several tiles per workgroup: the next tile is looked up while the last one's
# results pass through the same LDS.
@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("counts", [[60, 0, 200, 1] * 32, [30, 0, 65, 17] * 32],
                         ids=["tiles of 128 rows", "tiles of 64 rows"])
@pytest.mark.parametrize("k,n", [(96, 1504), (512, 1504), (512, 1499), (300, 3001)])
def test_short_rows_of_many_experts(dt, counts, k, n):
    from fastmoe_amd import fmoe_cuda, mx

    g = torch.Generator(device="cuda").manual_seed(k + n)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    x, b = draw(sum(counts), k).to(DTYPES[dt]), draw(len(counts), n).to(DTYPES[dt])
    wq, xq = mx.quantize(draw(len(counts), n, k) * 0.05), mx.quantize(x)
    y = mx.linear(x, torch.tensor(counts), wq, b)
    xv, at = xq.dequantize(torch.float32).double(), 0
    for e, c in enumerate(counts):
        rows = xv[at:at + c]
        we = mx.MXTensor(wq.codes[e], wq.scales[e], k).dequantize(torch.float32).double()
        want = rows @ we.T + b[e].double()
        mag = rows.abs() @ we.abs().T + b[e].double().abs()
        # as above: the instructions' sums and the bias in f32, then the output's rounding
        tol = UNIT[dt] * want.abs() + 2.0 ** -23 * (k / 128 + 4) * mag
        assert ((y[at:at + c].double() - want).abs() <= tol).all(), e
        at += c
    for _ in range(5):
        assert torch.equal(mx.linear(x, torch.tensor(counts), wq, b), y)
    seg = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
    y32 = fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k, b.float(), seg,
                                  torch.empty(sum(counts), n, device="cuda"))
    for act, h in ((0, y32), (2, y32.relu())):
        codes, scales = fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k,
                                                    b, seg, act)
        assert torch.equal(mx.MXTensor(codes, scales, n).dequantize(torch.float32),
                           mx.quantize(h).dequantize(torch.float32))


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("case", BY_RULE)
def test_no_bias_is_a_bias_of_zeros(case, dt):
    from fastmoe_amd import fmoe_cuda, mx

    counts, k, n = BY_RULE[case]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(sum(counts), k, device="cuda", generator=g).to(DTYPES[dt])
    wq = mx.quantize(torch.randn(len(counts), n, k, device="cuda", generator=g))
    zeros = torch.zeros(len(counts), n, device="cuda", dtype=DTYPES[dt])
    # (one value further on: rows of the bias that start inside a word)
    inside = torch.zeros(len(counts) * n + 1, device="cuda", dtype=DTYPES[dt])[1:].view(zeros.shape)
    y = mx.linear(x, torch.tensor(counts), wq)
    assert torch.equal(y, mx.linear(x, torch.tensor(counts), wq, zeros))
    assert torch.equal(y, mx.linear(x, torch.tensor(counts), wq, inside))
    xq = mx.quantize(x)
    seg = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
    for act in (0, 1, 2):
        run = lambda b: fmoe_cuda.mx_linear_act_fwd(xq.codes, xq.scales, wq.codes, wq.scales, k,
                                                    b, seg, act)
        blocks = -(-n // 128) * 4                     # (scales further on are not written)
        (c0, s0), (c1, s1), (c2, s2) = run(None), run(zeros), run(inside)
        assert torch.equal(c0, c1) and torch.equal(c0, c2)
        assert torch.equal(s0[:, :blocks], s1[:, :blocks])
        assert torch.equal(s0[:, :blocks], s2[:, :blocks])


def test_counts_that_do_not_fit_are_cut_off():
    """On the device nobody looks at them: negative counts are none, rows there are not are left."""
    from fastmoe_amd import mx

    x = torch.randn(20, 96).cuda()
    w = mx.quantize(torch.randn(3, 40, 96).cuda())
    fit = mx.linear(x, torch.tensor([5, 0, 15]), w)
    for counts in ([5, -3, 15], [5, -3, 10 ** 12], [5, -2 ** 62, 2 ** 62]):
        assert torch.equal(mx.linear(x, torch.tensor(counts).cuda(), w), fit), counts
    all_first = mx.linear(x, torch.tensor([20, 0, 0]), w)
    assert torch.equal(mx.linear(x, torch.tensor([2 ** 62, 2 ** 62, 2 ** 62]).cuda(), w), all_first)
    assert mx.linear(x, torch.tensor([-1, -1, -1]).cuda(), w).shape == (20, 40)


def test_both_bindings_count_alike():
    from fastmoe_amd import _ext, fmoe_cuda

    py, cx = fmoe_cuda.ctypes_ops, _ext.load()
    x = torch.randn(130, 72).cuda()
    counts = torch.tensor([0, 1, 60, 0, 64] + [0] * 70 + [5]).cuda()
    p, c = py.mx_quantize_counted(x, counts), cx.mx_quantize_counted(x, counts)
    assert all(torch.equal(a, b) for a, b in zip(p, c))
    want = torch.cumsum(counts, 0).cpu()
    assert torch.equal(p[2].cpu(), torch.cat([torch.zeros(1).long(), want]).int())
    plain = py.mx_quantize(x)
    assert torch.equal(p[0], plain[0]) and torch.equal(p[1], plain[1])


def test_results_beyond_32_bits():
    """An output of more than 2^32 elements: its last rows."""
    from fastmoe_amd import mx

    rows, k, n = 66000, 64, 65536
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, k, device="cuda", generator=g).bfloat16()
    w = mx.quantize(torch.randn(1, n, k, device="cuda", generator=g))
    y = mx.linear(x, torch.tensor([rows]), w)
    last = mx.linear(x[-300:], torch.tensor([300]), w)
    assert torch.equal(y[-300:], last)


def test_rows_without_an_expert_stay_as_they_are():
    from fastmoe_amd import fmoe_cuda, mx

    x, w, _ = _problem([20, 30], 128, 48, "bf16", 3)
    xq, wq = mx.quantize(x.cuda()), mx.quantize(w.view(2, 48, 128).cuda())
    seg = torch.tensor([0, 7, 19], dtype=torch.int32).cuda()
    out = torch.full((50, 48), 7.0, dtype=torch.bfloat16).cuda()
    fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, 128, None, seg, out)
    assert (out[19:] == 7).all() and (out[:19] != 7).any()
    out.fill_(7.0)
    fmoe_cuda.mx_linear_fwd(xq.codes, xq.scales, wq.codes, wq.scales, 128, None,
                            torch.zeros(3, dtype=torch.int32).cuda(), out)
    assert (out == 7).all()
    empty = mx.linear(x[:0].cuda(), torch.tensor([0, 0]), wq)
    assert empty.shape == (0, 48)


@pytest.mark.parametrize("rows", [3, 200])
def test_nan_stays_in_its_row_and_its_feature(rows):
    from fastmoe_amd import mx

    x, w, _ = _problem([rows], 256, 64, "f32", 4)
    x[1, 40] = float("nan")
    x[2, 200] = float("inf")
    w[5, 3] = float("nan")
    y = mx.linear(x.cuda(), torch.tensor([rows]), mx.quantize(w.view(1, 64, 256).cuda())).cpu()
    bad = torch.zeros(rows, 64, dtype=torch.bool)
    bad[1], bad[2], bad[:, 5] = True, True, True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_gradients_in_front_of_frozen_weights(dt):
    from fastmoe_amd import mx

    for counts, k, n in [([5, 0, 20], 64, 96), ([100, 40], 300, 130), ([300], 512, 256)]:
        x, w, b = _problem(counts, k, n, dt, k)
        wq = mx.quantize(w.view(len(counts), n, k).cuda())
        xg, bg = x.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
        y = mx.linear(xg, torch.tensor(counts), wq, bg)
        dy = _rows(sum(counts), n, dt, 9)
        y.backward(dy.cuda())
        we = R.round_trip(w.double().numpy()).reshape(len(counts), n, k)
        at = 0
        for e, c in enumerate(counts):
            g = dy[at:at + c].double().numpy()
            want, mag = g @ we[e], np.abs(g) @ np.abs(we[e])
            tol = UNIT[dt] * np.abs(want) + 2.0 ** -22 * (n / 16 + 4) * mag
            assert (np.abs(xg.grad[at:at + c].double().cpu().numpy() - want) <= tol).all()
            want, mag = g.sum(0), np.abs(g).sum(0)
            tol = UNIT[dt] * np.abs(want) + 2.0 ** -22 * (c + 4) * mag + 1e-30
            assert (np.abs(bg.grad[e].double().cpu().numpy() - want) <= tol).all()
            at += c


def test_gradient_against_differences():
    """Rows on the grid of the format itself, moved by steps that keep them on it: there the
    product is linear in them and the straight-through gradient is its slope."""
    from fastmoe_amd import mx

    rng = np.random.default_rng(2)
    k, n = 64, 40
    x = torch.from_numpy(R.E2M1[rng.integers(0, 4, (3, k))]).float()
    x[:, ::32] = 4.0                            # every block keeps the scale 1
    w = mx.quantize(torch.from_numpy(rng.standard_normal((1, n, k))).float().cuda())
    dy = torch.from_numpy(rng.standard_normal((3, n))).float()
    xg = x.cuda().requires_grad_(True)
    mx.linear(xg, torch.tensor([3]), w).backward(dy.cuda())
    for col in (1, 17, 33, 63):
        side = []
        for step in (0.5, -0.5):
            moved = x.clone()
            moved[:, col] += step
            side.append((mx.linear(moved.cuda(), torch.tensor([3]), w).cpu() * dy).sum(1))
        assert torch.allclose(side[0] - side[1], xg.grad[:, col].cpu(), rtol=1e-4, atol=1e-5)


def test_refusals():
    from fastmoe_amd import fmoe_cuda, mx

    x = torch.randn(6, 64).cuda()
    w = mx.quantize(torch.randn(2, 32, 64).cuda())
    for bad in (lambda: mx.quantize(x.double()), lambda: mx.quantize(x.cpu()),
                lambda: mx.quantize(x.int()), lambda: w.dequantize(torch.float64),
                lambda: mx.linear(x[:, :32], torch.tensor([3, 3]), w),
                lambda: mx.linear(x, torch.tensor([3, 4]), w),
                lambda: mx.linear(x, torch.tensor([7, -1]), w),
                lambda: mx.linear(x, torch.tensor([3, 3, 0]), w),
                lambda: mx.linear(x, torch.tensor([3, 3]), w, torch.zeros(2, 31).cuda()),
                lambda: mx.linear(x, torch.tensor([3, 3]), w, torch.zeros(2, 32).half().cuda()),
                lambda: mx.linear(x.cpu(), torch.tensor([3, 3]), w),
                lambda: mx.linear(x.double(), torch.tensor([3, 3]), w),
                lambda: mx.linear(x, torch.tensor([3, 3]),
                                  mx.MXTensor(w.codes, w.scales[..., :8], 64)),
                lambda: mx.linear(x, torch.tensor([3, 3]), mx.MXTensor(w.codes, w.scales, 200)),
                lambda: fmoe_cuda.mx_quantize_tokens(x, torch.zeros(5, dtype=torch.int32).cuda(), 1)):
        with pytest.raises(RuntimeError):
            bad()
    y = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):                  # no gradient of a gradient
        g, = torch.autograd.grad(mx.linear(y, torch.tensor([3, 3]), w).sum(), y, create_graph=True)
        g.sum().backward()


def test_both_bindings_agree():
    from fastmoe_amd import _ext, fmoe_cuda, mx

    py, cx = fmoe_cuda.ctypes_ops, _ext.load()
    x, w, b = _problem([20, 0, 13], 200, 72, "bf16", 6)
    x, b = x.cuda(), b.cuda()
    wq = mx.quantize(w.view(3, 72, 200).cuda())
    seg = torch.tensor([0, 20, 20, 33], dtype=torch.int32).cuda()
    inv = torch.randperm(33).int().cuda()
    same = lambda p, q: all((a is None and b is None) or torch.equal(a, b) for a, b in zip(p, q))
    assert same(py.mx_quantize(x), cx.mx_quantize(x))
    assert same(py.mx_quantize_tokens(x, inv, 1), cx.mx_quantize_tokens(x, inv, 1))
    xc, xs = py.mx_quantize(x)
    assert torch.equal(py.mx_dequantize(xc, xs, torch.empty_like(x)),
                       cx.mx_dequantize(xc, xs, torch.empty_like(x)))
    out = lambda: torch.empty(33, 72, dtype=torch.bfloat16).cuda()
    assert torch.equal(py.mx_linear_fwd(xc, xs, wq.codes, wq.scales, 200, b, seg, out()),
                       cx.mx_linear_fwd(xc, xs, wq.codes, wq.scales, 200, b, seg, out()))
    p = py.mx_linear_act_fwd(xc, xs, wq.codes, wq.scales, 200, b, seg, 1)
    c = cx.mx_linear_act_fwd(xc, xs, wq.codes, wq.scales, 200, b, seg, 1)
    assert torch.equal(p[0], c[0]) and torch.equal(p[1][:, :4], c[1][:, :4])
    dy = torch.randn(33, 72).bfloat16().cuda()
    assert same(py.mx_linear_bwd(dy, seg, wq.codes, wq.scales, 200, True, True),
                cx.mx_linear_bwd(dy, seg, wq.codes, wq.scales, 200, True, True))


def test_offsets_beyond_32_bits():
    """Weights of more than 2^32 code bytes: the last expert's rows."""
    from fastmoe_amd import mx

    k, n, e = 8192, 8192, 130                     # 4.36e9 bytes of codes
    g = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(0, 256, (e, n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.full((e, n, k // 32), 120, dtype=torch.uint8, device="cuda")
    w = mx.MXTensor(codes, scales, k)
    x = torch.randn(3, k, device="cuda", generator=g)
    counts = torch.zeros(e, dtype=torch.int64)
    counts[-1] = 3
    y = mx.linear(x, counts, w)
    last = mx.MXTensor(codes[-1], scales[-1], k).dequantize(torch.float32)
    want = mx.quantize(x).dequantize(torch.float32).double() @ last.double().T
    assert ((y.double() - want).abs() <= 1e-5 * want.abs().max()).all()


# ------------------------------------------------------------------ the experts of a layer
def _layer_reference(x, idx, score, w1, b1, w2, b2, act):
    """The fused path in 64 bits: x, score and biases as they are, weights' values."""
    from scipy.special import erfc

    y = np.zeros((x.shape[0], w2.shape[1]))
    xq = R.round_trip(x)
    for t in range(x.shape[0]):
        for j, e in enumerate(idx[t]):
            if e < 0:
                continue
            h = xq[t] @ w1[e].T + b1[e]
            h = 0.5 * h * erfc(-h * np.sqrt(0.5)) if act == "gelu" else np.maximum(h, 0)
            y[t] += score[t, j] * (R.round_trip(h[None])[0] @ w2[e].T + b2[e])
    return y


def _layer_inputs(t, k, e, d, h, dt, seed, drop=0.1):
    from fastmoe_amd import mx

    rng = np.random.default_rng(seed)
    put = lambda a: torch.from_numpy(a).to(DTYPES[dt])
    x, score = put(rng.standard_normal((t, d))), put(rng.random((t, k)))
    w1, w2 = (torch.from_numpy(rng.standard_normal(s) * 0.1).float() for s in ((e, h, d), (e, d, h)))
    b1, b2 = put(rng.standard_normal((e, h)) * 0.1), put(rng.standard_normal((e, d)) * 0.1)
    idx = make_gate(t, k, e, drop=drop, seed=seed)
    if t > 2:
        idx[1] = -1                                # a token that nobody serves
    return x, idx, score, mx.quantize(w1.cuda()), b1, mx.quantize(w2.cuda()), b2


@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("t,k,e,d,h,dt", [
    (1, 1, 4, 64, 128, "bf16"), (7, 2, 3, 100, 60, "f16"), (60, 8, 16, 128, 96, "bf16"),
    (130, 2, 2, 160, 544, "f16"), (40, 1, 80, 96, 130, "f32"), (3, 2, 5, 1030, 520, "bf16")])
def test_expert_layer(act, t, k, e, d, h, dt):
    from fastmoe_amd import mx

    x, idx, score, w1, b1, w2, b2 = _layer_inputs(t, k, e, d, h, dt, t + d)
    module = torch.nn.GELU() if act == "gelu" else torch.nn.ReLU()
    got = mx.expert_layer(x.cuda(), torch.from_numpy(idx).cuda(), score.cuda(), w1, b1.cuda(), w2,
                          b2.cuda(), module)
    assert got.dtype == DTYPES[dt] and got.shape == (t, d)
    f = lambda a: a.double().cpu().numpy()
    want = _layer_reference(f(x), idx, f(score), f(w1.dequantize(torch.float32)), f(b1),
                            f(w2.dequantize(torch.float32)), f(b2), act)
    if t > 2:
        assert not got[1].any()
    # two roundings of the result's type on the way out (experts, combine) and hidden values
    # that fall on the other side of a rounding boundary: about one in 10^4, each worth at most
    # half a step (a sixth of its value) of one of h terms
    err = np.abs(f(got) - want)
    scale = np.abs(want).max()
    assert err.max() <= scale * (8 * UNIT[dt] + 0.5 / np.sqrt(h))
    assert np.sqrt((err ** 2).mean()) <= scale * (2 * UNIT[dt] + 3e-3)


def test_expert_layer_trains_what_stands_in_front():
    from fastmoe_amd import mx

    x, idx, score, w1, b1, w2, b2 = _layer_inputs(50, 2, 4, 96, 160, "f32", 3)
    leaves = [a.cuda().requires_grad_(True) for a in (x, score, b1, b2)]
    y = mx.expert_layer(leaves[0], torch.from_numpy(idx).cuda(), leaves[1], w1, leaves[2], w2,
                        leaves[3], torch.nn.GELU())
    dy = torch.randn(50, 96).cuda()
    y.backward(dy)
    # the same arithmetic by autograd, the rounding passed straight through
    ref = [a.double().cuda().requires_grad_(True) for a in (x, score, b1, b2)]
    v1, v2 = w1.dequantize(torch.float32).double(), w2.dequantize(torch.float32).double()

    def q(a):
        return a + (mx.quantize(a.detach().float()).dequantize(torch.float32).double() - a).detach()

    want = torch.zeros(50, 96, dtype=torch.float64, device="cuda")
    gate = torch.from_numpy(idx).cuda()
    for e in range(4):
        tok, slot = torch.nonzero(gate == e, as_tuple=True)
        hid = torch.nn.functional.gelu(q(ref[0][tok]) @ v1[e].T + ref[2][e])
        want = want.index_add(0, tok, (q(hid) @ v2[e].T + ref[3][e]) * ref[1][tok, slot, None])
    want.backward(dy.double())
    for a, b in zip([y] + [l.grad for l in leaves], [want] + [r.grad for r in ref]):
        err = (a.double() - b).norm() / b.norm()
        assert err < 2e-3          # a few hidden values on the other side of a boundary


def _same_twice(fn):
    a, b = fn(), fn()
    return torch.equal(a, b)


def test_layer_with_a_scored_gate_on_other_streams_and_in_a_graph():
    import fastmoe_amd as fm
    from fastmoe_amd import fmoe_cuda, mx

    torch.manual_seed(1)
    layer = fm.FMoETransformerMLP(num_expert=16, d_model=128, d_hidden=192, top_k=4,
                                  gate=fm.ScoreGate.configured(n_group=4, top_group=2))
    layer = layer.bfloat16().cuda().eval()
    x = torch.randn(70, 128).bfloat16().cuda()
    with torch.no_grad():
        full = layer(x)
        mx.quantize_experts(layer)
        assert isinstance(layer.experts, mx.MXExpert) and len(layer.experts) == 16
        y = layer(x)
        assert _same_twice(lambda: layer(x))
        # 4-bit weights and rows: near the 16-bit layer, not equal to it
        rel = ((y - full).float().norm() / full.float().norm()).item()
        assert 0.01 < rel < 0.5
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            z = layer(x)
        side.synchronize()
        assert torch.equal(y, z)
        fmoe_cuda.init()
        static = x.clone()
        with torch.cuda.stream(side):
            layer(static)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(static)
        for seed in range(4):
            new = torch.randn(70, 128).bfloat16().cuda()
            static.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer(new))
    # the state dict goes round
    other = fm.FMoETransformerMLP(num_expert=16, d_model=128, d_hidden=192, top_k=4,
                                  gate=fm.ScoreGate.configured(n_group=4, top_group=2))
    other = mx.quantize_experts(other.bfloat16().cuda()).eval()
    other.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), y)
    # a layer in front of which something learns
    xg = x.clone().requires_grad_(True)
    layer(xg).float().sum().backward()
    assert torch.isfinite(xg.grad).all() and xg.grad.abs().sum() > 0
    assert layer.experts.b1.grad is not None
    with pytest.raises(TypeError):
        mx.quantize_experts(layer)
