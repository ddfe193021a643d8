"""Segment tables that name more rows than a buffer has: what lies beyond is in no product."""
import pytest
import torch

from fastmoe_amd import FMoELinear, functions, i8, mx
from fastmoe_amd.functions import SegmentTable, bounds_within, segments_for
from helpers import randn


def test_bounds_stay_within_the_rows_and_ascend():
    g = torch.Generator().manual_seed(1)
    for _ in range(200):
        e, n = (int(torch.randint(1, m, (1,), generator=g)) for m in (9, 50))
        counts = torch.randint(0, 12, (e,), generator=g)
        seg = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0))).int()
        cut = bounds_within(seg, n)
        assert cut.dtype == torch.int32 and torch.equal(cut, seg.clamp(max=n))
        wild = torch.randint(-20, 80, (e + 1,), generator=g, dtype=torch.int32)
        cut = bounds_within(wild, n)
        assert (cut[1:] >= cut[:-1]).all() and 0 <= cut.min() and cut.max() <= n
        # (a model of how products cut segments into tiles: no row of any is past the buffer's end)
        for tm in (16, 64, 128):
            for a, b in zip(cut[:-1].tolist(), cut[1:].tolist()):
                assert all(r + min(tm, b - r) <= n for r in range(a, b, tm))
    empty = torch.zeros(0, dtype=torch.int32)
    assert bounds_within(empty, 4) is empty


def test_tables_that_know_their_rows_are_handed_on():
    seg, counts = torch.tensor([0, 3, 7], dtype=torch.int32), torch.tensor([3, 4])
    table = SegmentTable(seg, counts, 9)
    assert table.bounds(torch.empty(9, 2)) is seg and segments_for(table, torch.empty(12, 2)) is seg
    assert table.bounds(torch.empty(5, 2)).tolist() == [0, 3, 5]
    by_hand = SegmentTable(seg, counts)
    assert by_hand.bounds(torch.empty(9, 2)).tolist() == [0, 3, 7]
    assert by_hand.bounds(torch.empty(2, 2)).tolist() == [0, 2, 2]
    assert by_hand.bounds(torch.empty(())).tolist() == [0, 0, 0]
    assert segments_for(seg, torch.empty(5, 2)).tolist() == [0, 3, 5]
    assert segments_for(counts, torch.empty(5, 2)) is counts and segments_for(None, seg) is None


def plan_of(t, e, top_k):
    g = torch.Generator().manual_seed(t)
    best = torch.rand(t, e, generator=g).topk(top_k, dim=1)[1]
    taken = torch.zeros(t, e, dtype=torch.bool).scatter_(1, best, True)
    return functions.MapPlan(taken.cuda(), t * top_k + 5)


def products(e, k, n, dtype):
    """linear(x, segments) of every kind of weights, and one whose rows need a gradient."""
    w = randn((e, n, k), torch.float32, 2, 0.05).cuda()
    eight, four, bias = i8.quantize(w), mx.quantize(w), randn((e, n), dtype, 3).cuda()
    wide = FMoELinear(e, k, n).cuda().to(dtype)
    return [lambda x, s: i8.linear(x, s, eight, bias), lambda x, s: mx.linear(x, s, four, bias), wide]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,e", [(40, 4), (1500, 3), (300, 80)])
def test_products_of_fewer_rows_than_a_plan_names(t, e, dtype):
    plan = plan_of(t, e, 2)
    k, n = 128, 264
    x = randn((t, k), dtype, 1).cuda()
    sorted_rows = functions.sort_tokens(x, plan)
    seg = plan.segments.seg_off
    for linear in products(e, k, n, dtype):
        for rows in (x, sorted_rows[:t + 3], sorted_rows[:1], sorted_rows[:0]):
            have = rows.shape[0]
            counts = bounds_within(seg, have).diff().long()
            z, v = (rows.detach().clone().requires_grad_() for _ in range(2))
            y, want = linear(z, plan.segments), linear(v, counts.cpu())
            assert y.shape == (have, n)
            live = int(counts.sum())
            assert torch.equal(y[:live], want[:live])
            dy = randn((have, n), dtype, 4).cuda()
            y.backward(dy)
            want.backward(dy)
            assert torch.equal(z.grad[:live], v.grad[:live])


@pytest.mark.gpu
def test_tables_made_by_hand():
    e, k, n, rows = 4, 64, 136, 50
    x = randn((rows, k), torch.bfloat16, 1).cuda()
    counts = torch.tensor([3, 0, 40, 7], device="cuda")
    for linear in products(e, k, n, torch.bfloat16):
        want = linear(x, counts.cpu())
        good = torch.tensor([0, 3, 3, 43, 50], dtype=torch.int32, device="cuda")
        assert torch.equal(linear(x, SegmentTable(good, counts)), want)
        wild = torch.tensor([-7, 3, 2, 43, 1 << 30], dtype=torch.int32, device="cuda")
        assert torch.equal(linear(x, SegmentTable(wild, counts)), want)
    for linear in products(e, k, n, torch.bfloat16)[:2]:
        want = linear(x, counts.cpu())
        assert torch.equal(linear(x, wild), want)


@pytest.mark.gpu
def test_a_cut_table_in_a_graph():
    plan = plan_of(40, 4, 2)
    w = i8.quantize(randn((4, 136, 64), torch.float32, 2, 0.05).cuda())
    x = functions.sort_tokens(randn((40, 64), torch.bfloat16, 1).cuda(), plan)[:50].contiguous()
    want = i8.linear(x, plan.segments, w)
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        y = i8.linear(held, plan.segments, w)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, i8.linear(held, plan.segments, w)) and torch.equal(y, want)
