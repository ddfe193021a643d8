"""8-bit rows and routing maps, what needs no GPU: sizes and pointers that are refused before any
launch, tensors that are refused, and how 8-bit experts are kept."""
import pytest
import torch

from fastmoe_amd import FMoETransformerMLP, _lib, functions, i8

lib = _lib.load()
P = 1 << 20          # an address that is aligned and never read: every call here is refused first


def refused(rc, text=b""):
    assert rc < 0 and text in lib.fmoe_last_error()


def test_rows_that_do_not_fit_are_refused():
    assert [lib.fmoe_i8_row_bytes(k) for k in (0, 1, 128, 129, 131072)] == [0, 128, 128, 256, 131072]
    refused(lib.fmoe_i8_row_bytes(-1), b"feature count")
    refused(lib.fmoe_i8_row_bytes(131073), b"feature count")
    for rows, k, dtype in ((-1, 8, 0), (1 << 31, 8, 0), (4, 0, 0), (4, 131073, 0), (4, 8, 1), (4, 8, 7)):
        refused(lib.fmoe_i8_quantize(P, rows, k, None, P, P, dtype, None), b"i8_quantize")
        if rows < 1 << 31:
            refused(lib.fmoe_i8_dequantize(P, P, rows, k, P, dtype, None), b"i8_dequantize")
    for x, codes, scales in ((None, P, P), (P, None, P), (P, P, None), (P, P + 8, P)):
        refused(lib.fmoe_i8_quantize(x, 4, 8, None, codes, scales, 0, None))
    refused(lib.fmoe_i8_quantize_counted(P, 4, 8, None, 2, P, P, P, 0, None), b"bad counts")
    refused(lib.fmoe_i8_quantize_counted(P, 4, 8, P, 2, None, P, P, 0, None), b"bad counts")
    refused(lib.fmoe_i8_quantize_tokens(P, None, 4, 2, 8, P, P, 0, None), b"null")
    refused(lib.fmoe_i8_quantize_tokens(P, P, 1 << 30, 2, 8, P, P, 0, None), b"bad sizes")
    refused(lib.fmoe_i8_dequantize_bwd(P, P, None, P, P, 4, 8, 8, 2, 0, None), b"null")
    assert lib.fmoe_i8_quantize(None, 0, 8, None, None, None, 0, None) == 0


def test_products_that_do_not_fit_are_refused():
    def call(x=P, xs=P, w=P, ws=P, seg=P, y=P, rows=4, k=8, n=8, e=2, dtype=0):
        return lib.fmoe_i8_linear_fwd(x, xs, w, ws, None, seg, y, rows, k, n, e, dtype, None)

    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(k=0), dict(k=131073), dict(n=0),
                dict(n=131073), dict(e=0), dict(dtype=1), dict(x=None), dict(xs=None), dict(w=None),
                dict(ws=None), dict(seg=None), dict(y=None), dict(x=P + 4), dict(w=P + 8),
                dict(xs=P + 2), dict(ws=P + 1)):
        refused(call(**bad), b"i8_linear")
    assert call(rows=0) == 0

    def grad(dy=P, w=P, ws=P, seg=P, dx=P, rows=4, k=8, n=8, e=2, work=P, size=1 << 30, dtype=0):
        return lib.fmoe_i8_linear_dx(dy, w, ws, seg, dx, rows, k, n, e, work, size, dtype, None)

    for bad in (dict(rows=-1), dict(k=0), dict(n=131073), dict(e=0), dict(dtype=1), dict(dy=None),
                dict(w=None), dict(ws=None), dict(seg=None), dict(dx=None), dict(w=P + 4),
                dict(ws=P + 2)):
        refused(grad(**bad), b"i8_linear_dx")
    assert grad(rows=0) == 0
    # one expert, 5 column tiles: 8 blocks share the summed axis
    assert lib.fmoe_i8_dx_workspace_bytes(20, 520, 4096, 1, 0) == 8 * 20 * 520 * 4
    for bad in (dict(work=None), dict(size=8 * 20 * 520 * 4 - 1), dict(work=P + 4)):
        refused(grad(rows=20, k=520, n=4096, e=1, **bad), b"workspace")
    assert lib.fmoe_i8_dx_workspace_bytes(5000, 4096, 4096, 8, 3) == 0
    assert lib.fmoe_i8_few_rows(192, 2, 3) == 1 and lib.fmoe_i8_few_rows(193, 2, 3) == 0
    assert lib.fmoe_i8_few_rows(100000, 2, 0) == 1


def test_plans_and_moves_that_do_not_fit_are_refused():
    assert lib.fmoe_map_workspace_bytes(64, 128) == 0
    assert lib.fmoe_map_workspace_bytes(16384, 128) == 256 * 128 * 2
    for t, e in ((-1, 4), (4, 0), (4, 1025), (1 << 23, 256), ((1 << 23) + 1, 1)):
        refused(lib.fmoe_map_workspace_bytes(t, e), b"bad sizes")

    def plan(m=P, t=100, e=4, rows=8, counts=P, pairs=P, ws=P, size=1 << 20):
        return lib.fmoe_map_plan(m, t, e, rows, counts, P, P, pairs, ws, size, None)

    for bad in (dict(m=None), dict(t=0), dict(rows=-1), dict(rows=1 << 31), dict(counts=None),
                dict(pairs=None), dict(pairs=P + 4), dict(ws=None), dict(size=8), dict(ws=P + 8)):
        refused(plan(**bad))

    def expand(tokens=P, given=None, weight=P, off=P, pairs=P, rows=P, dw=None, t=4, d=8, e=4,
               most=8, dtype=3, wdtype=0):
        return lib.fmoe_map_expand(tokens, given, weight, off, pairs, None, rows, dw, t, d, e, most,
                                   dtype, wdtype, None)

    def reduce(rows=P, given=None, weight=P, off=P, pairs=P, tokens=P, dw=None, t=4, d=8, e=4,
               most=8, dtype=3, wdtype=0):
        return lib.fmoe_map_reduce(rows, given, weight, off, pairs, tokens, dw, t, d, e, most, dtype,
                                   wdtype, None)

    for f in (expand, reduce):
        for bad in (dict(tokens=None), dict(rows=None), dict(off=None), dict(pairs=None), dict(t=-1),
                    dict(d=0), dict(e=0), dict(e=1025), dict(most=-1), dict(dtype=1),
                    dict(wdtype=2), dict(dw=P), dict(dw=P, given=P, weight=None),
                    dict(t=1 << 23, d=1 << 14)):
            refused(f(**bad))
        assert f(t=0) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(4, 8)
    w = i8.I8Tensor(torch.zeros(2, 8, 128, dtype=torch.int8), torch.zeros(2, 8), 8)
    m = torch.ones(4, 2, dtype=torch.bool)
    for call in (lambda: i8.quantize(x), lambda: w.dequantize(),
                 lambda: i8.linear(x, torch.tensor([2, 2]), w),
                 lambda: functions.MapPlan(m, 8), lambda: functions.MapPlan(m.float(), 8),
                 lambda: functions.MapPlan(m[None], 8)):
        with pytest.raises(RuntimeError):
            call()


def test_checkpoint_layouts():
    codes = torch.randint(-127, 128, (3, 5, 200), dtype=torch.int8)
    scales = torch.rand(3, 5, 1, dtype=torch.float16)
    w = i8.I8Tensor.from_codes(codes, scales)
    assert w.shape == (3, 5, 200) and w.codes.shape == (3, 5, 256) and w.scales.shape == (3, 5)
    assert torch.equal(w.codes[..., :200], codes) and not w.codes[..., 200:].any()
    assert w.scales.dtype == torch.float32 and torch.equal(w.scales, scales[..., 0].float())
    for bad in ((codes.short(), scales), (codes, scales[:, :4]), (codes[..., :0], scales)):
        with pytest.raises(ValueError):
            i8.I8Tensor.from_codes(*bad)


@pytest.fixture
def quantised(monkeypatch):
    """An 8-bit layer on the CPU, its weights quantised by hand."""
    def quantize(x):
        top = x.detach().abs().amax(-1)
        return i8.I8Tensor.from_codes(torch.round(127 * x.detach() / top[..., None]).to(torch.int8),
                                      top / 127)

    monkeypatch.setattr(i8, "quantize", quantize)
    layer = FMoETransformerMLP(num_expert=3, d_model=16, d_hidden=24, activation=torch.nn.ReLU())
    layer.experts.htoh4.bias.some_tag = "kept"
    return i8.quantize_experts(layer)


def test_experts_in_8_bits_keep_what_they_should(quantised):
    experts = quantised.experts
    assert isinstance(experts, i8.I8Expert) and len(experts) == 3
    assert experts.b1.some_tag == "kept" and experts.b1.requires_grad
    assert {n for n, _ in experts.named_buffers()} == {"w1_codes", "w1_scales", "w2_codes", "w2_scales"}
    assert experts.w1.shape == (3, 24, 16) and experts.w2.shape == (3, 16, 24)
    scales = experts.w1_scales.clone()
    for cast in (quantised.half, quantised.bfloat16, quantised.float):
        cast()
        assert experts.w1_scales.dtype == torch.float32 and torch.equal(experts.w1_scales, scales)
        assert experts.w1_codes.dtype == torch.int8
    assert experts.b1.dtype == torch.float32
    view = experts[-1]
    assert view.w1.shape == (1, 24, 16) and view.b2.shape == (1, 16)
    assert torch.equal(view.w2.codes[0], experts.w2_codes[2])
    with pytest.raises(IndexError):
        experts[3]
    with pytest.raises(TypeError):
        i8.quantize_experts(quantised)
    state = quantised.state_dict()
    assert state["experts.w2_codes"].dtype == torch.int8 and "experts.w1_scales" in state


def test_gradients_of_many_rows_that_do_not_fit_are_refused():
    size = lib.fmoe_i8_dx_many_workspace_bytes

    def grad(dy=P, w=P, ws=P, seg=P, dx=P, rows=400, k=8, n=24, e=2, work=P, room=1 << 30, dtype=3):
        return lib.fmoe_i8_linear_dx_many(dy, w, ws, seg, dx, rows, k, n, e, work, room, dtype, None)

    # rows, weights and a float a row, each to whole 256 bytes; twice the first two in f16
    assert size(400, 8, 24, 2, 3) == 400 * 24 * 2 + 2 * 24 * 8 * 2 + 1792
    assert size(400, 8, 24, 2, 2) == 2 * 400 * 24 * 2 + 2 * 2 * 24 * 8 * 2 + 1792
    assert size(0, 8, 24, 2, 3) == 0
    # (sizes past 32 bits)
    assert size(1 << 20, 4096, 14336, 8, 2) > 2 * 2 * ((1 << 20) + 8 * 4096) * 14336
    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(k=0), dict(k=131073), dict(n=131073),
                dict(e=0), dict(e=65536), dict(dtype=0), dict(dtype=1), dict(dy=None), dict(w=None),
                dict(ws=None), dict(seg=None), dict(dx=None), dict(w=P + 4), dict(ws=P + 2)):
        refused(grad(**bad), b"i8_linear_dx_many")
    for bad in (dict(work=None), dict(room=size(400, 8, 24, 2, 3) - 1), dict(work=P + 4)):
        refused(grad(**bad), b"workspace")
    assert grad(rows=0) == 0


def test_the_most_tokens_and_features_of_a_move():
    """Sizes are looked at before pointers: what passes them is refused for its missing offsets."""
    def expand(t, d, dw=None):
        return lib.fmoe_map_expand(P, dw, P, None, P, None, P, dw, t, d, 4, 8, 3, 0, None)

    def reduce(t, d, dw=None):
        return lib.fmoe_map_reduce(P, dw, P, None, P, P, dw, t, d, 4, 8, 3, 0, None)

    for f in (expand, reduce):
        for t, d in ((1 << 23, 3585), (1 << 22, 7681), ((1 << 23) - 1, 5000)):
            refused(f(t, d), b"tokens times ceil(features / 512) must be below 2^26")
            refused(f(t, d, P), b"null pointer")        # (a block per token, whatever its length)
        for t, d in ((1 << 23, 3584), ((1 << 22) - 1, 8192)):
            refused(f(t, d), b"null pointer")
