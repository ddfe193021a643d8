r"""Autograd functions of the MoE dispatch, mirroring fmoe/functions.py of the
reference (same names and argument lists), plus the fused variants this
package's own layer uses: they keep every count on the device, so a forward
pass needs no device-to-host copy.
"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import fmoe_cuda


# --------------------------------------------------------------------------
# Reference-shaped helpers (fmoe/functions.py:28-193), world_size == 1 only
# --------------------------------------------------------------------------
def _single_worker(world_size):
    if world_size != 1:
        raise NotImplementedError(
            "this build covers the single-GPU path (world_size == 1); "
            "expert exchange across workers is out of scope")


def count_by_gate(gate, num_expert, world_size, require_pos=True):
    """(pos, local_expert_count, global_expert_count) as fmoe/functions.py:28-49
    returns them: pos int64[N_valid] on the device (None if not required), the
    counts int64[E] on the device (one tensor for both at world_size 1).

    Without positions this is one histogram launch; with them, one fused
    routing call plus the single host read that sizes `pos`."""
    _single_worker(world_size)
    gate = gate.contiguous()
    with torch.no_grad():
        if not require_pos:
            hist = torch.zeros(num_expert, device=gate.device, dtype=torch.int32)
            fmoe_cuda.expert_count(gate, hist)
            counts = hist.long()
            return None, counts, counts
        pos, counts, seg_off, _ = fmoe_cuda.route(gate, num_expert, want_inv=False)
        n_valid = int(seg_off[-1].item())
    return pos[:n_valid], counts, counts


def prepare_forward(gate, num_expert, world_size):
    """(pos, local_expert_count, global_expert_count, fwd_expert_count,
    fwd_batch_size) with the three counts on the host, as
    fmoe/functions.py:52-75 hands them to the dispatch.

    ONE device-to-host copy (the E counts; the reference makes five,
    functions.py:46,68,71-73): the number of live rows that sizes `pos` is their
    sum, taken on the host."""
    _single_worker(world_size)
    with torch.no_grad():
        pos, counts, _seg_off, _ = fmoe_cuda.route(gate.contiguous(), num_expert, want_inv=False)
    host = counts.cpu()
    n_valid = int(host.sum())
    return pos[:n_valid], host, host, host.clone(), n_valid


def _local_scatter(inp, pos):
    return fmoe_cuda.local_scatter(inp.contiguous(), pos)


def _local_gather(inp, pos, out_batch_size, maybe_overlap=True):
    return fmoe_cuda.local_gather(inp.contiguous(), pos, out_batch_size,
                                  maybe_overlap)


class MOEScatter(Function):
    r"""Rows of `inp` gathered into expert order; fmoe/functions.py:93-142."""

    @staticmethod
    def forward(ctx, inp, pos, local_expert_count, global_expert_count,
                fwd_batch_size, world_size):
        _single_worker(world_size)
        local_input_buf = _local_scatter(inp, pos)
        ctx.moe_args = inp.shape[0], pos.shape[0], world_size
        ctx.save_for_backward(pos, local_expert_count, global_expert_count)
        return local_input_buf

    @staticmethod
    def backward(ctx, global_grad_in):
        (pos, _lec, _gec) = ctx.saved_tensors
        (inp_batch_size, _buf_batch_size, _world_size) = ctx.moe_args
        grad_in = _local_gather(global_grad_in, pos, inp_batch_size)
        return grad_in, None, None, None, None, None


class MOEGather(Function):
    r"""Expert-ordered rows put back at their slots; fmoe/functions.py:144-193."""

    @staticmethod
    def forward(ctx, global_output_buf, pos, local_expert_count,
                global_expert_count, local_batch_size, world_size):
        _single_worker(world_size)
        output = _local_gather(global_output_buf, pos, local_batch_size,
                               maybe_overlap=False)
        ctx.moe_args = (global_output_buf.shape[0], world_size)
        ctx.save_for_backward(pos, local_expert_count, global_expert_count)
        return output

    @staticmethod
    def backward(ctx, grad_out):
        pos, _lec, _gec = ctx.saved_tensors
        grad_out_buf = _local_scatter(grad_out.contiguous(), pos)
        return grad_out_buf, None, None, None, None, None


# --------------------------------------------------------------------------
# Fused, synchronisation-free path
# --------------------------------------------------------------------------
def bounds_within(seg_off: torch.Tensor, n_rows: int) -> torch.Tensor:
    """Segment bounds nobody has looked at, for a buffer of n_rows rows: what lies beyond the rows
    there are is cut off, and bounds below the one before are that one.  (The products take their
    rows from the bounds alone.)"""
    if not seg_off.numel():
        return seg_off
    return seg_off.clamp(0, min(n_rows, 2 ** 31 - 1)).cummax(0)[0]


class SegmentTable:
    """Per-expert row segments kept on the device.

    seg_off  int32[E+1]  exclusive prefix of the row counts
    counts   int64[E]    rows per expert (what the reference calls
                         fwd_expert_count, fmoe/functions.py:66-67)
    n_rows   rows that the bounds are known to stay within (None: not known)
    """

    def __init__(self, seg_off: torch.Tensor, counts: torch.Tensor, n_rows=None):
        self.seg_off = seg_off
        self.counts = counts
        self.n_rows = n_rows
        self._host = None

    def bounds(self, x: torch.Tensor) -> torch.Tensor:
        """seg_off for the rows of x, cut off where x has fewer than the table may name."""
        rows = x.shape[0] if x.dim() else 0
        if self.n_rows is not None and rows >= self.n_rows:
            return self.seg_off
        return bounds_within(self.seg_off, rows)

    @property
    def num_expert(self) -> int:
        return self.counts.numel()

    def cpu(self) -> torch.Tensor:
        """Host int64 counts (one device-to-host copy, cached)."""
        if self._host is None:
            self._host = self.counts.cpu()
        return self._host


def segments_for(counts, x: torch.Tensor):
    """What a product takes for the rows of x: a table's bounds, or bounds themselves, within x; row
    counts (int64, or none) as they are."""
    if isinstance(counts, SegmentTable):
        return counts.bounds(x)
    if isinstance(counts, torch.Tensor) and counts.dtype == torch.int32:
        return bounds_within(counts, x.shape[0] if x.dim() else 0)
    return counts


class RoutePlan:
    """Everything the dispatch needs about one routing decision; `routed` is what
    fmoe_cuda.route made of it, where that is at hand."""

    def __init__(self, gate: torch.Tensor, num_expert: int, routed=None):
        self.top_k = gate.shape[-1] if gate.dim() >= 2 else 1
        self.n_slots = gate.numel()
        self.n_tokens = self.n_slots // max(self.top_k, 1)
        if routed is None:
            with torch.no_grad():
                routed = fmoe_cuda.route(gate.contiguous(), num_expert)
        pos, counts, seg_off, inv = routed
        self.pos = pos
        self.inv = inv
        self.segments = SegmentTable(seg_off, counts, self.n_slots)

    @property
    def n_rows_dev(self) -> torch.Tensor:
        """Device int32 holding the number of live rows (= seg_off[E])."""
        return self.segments.seg_off[-1:]


class FusedScatter(Function):
    r"""buf[r] = inp[pos[r] // k]; backward sums a token's k rows in a fixed
    order (no float atomics).  Replaces MOEScatter at world_size 1."""

    @staticmethod
    def forward(ctx, inp, plan: RoutePlan):
        ctx.plan = plan
        if 4 <= plan.top_k <= 64:
            # token order: a row is read once for its k copies (measured: 62 vs 81 us
            # at k = 8 on 8192 x 2048 bf16; at k = 2 the row order is the faster one)
            return fmoe_cuda.scatter_tokens(inp.contiguous(), plan.inv, plan.top_k)
        return fmoe_cuda.local_scatter(inp.contiguous(), plan.pos, plan.top_k,
                                       plan.n_rows_dev)

    @staticmethod
    def backward(ctx, grad_buf):
        plan = ctx.plan
        return fmoe_cuda.scatter_reduce(grad_buf.contiguous(), plan.inv,
                                        plan.n_tokens, plan.top_k), None


class FusedGatherCombine(Function):
    r"""y[t] = sum_j score[t, j] * buf[row of slot (t, j)]: MOEGather followed
    by the bmm of fmoe/layers.py:288-295 in one pass over the rows."""

    @staticmethod
    def forward(ctx, buf, score, plan: RoutePlan):
        buf = buf.contiguous()
        score = score.contiguous().to(buf.dtype)
        ctx.plan = plan
        ctx.save_for_backward(buf, score)
        return fmoe_cuda.gather_combine_fwd(buf, plan.inv, score, plan.n_tokens,
                                            plan.top_k)

    @staticmethod
    def backward(ctx, grad_y):
        buf, score = ctx.saved_tensors
        plan = ctx.plan
        dbuf, dscore = fmoe_cuda.gather_combine_bwd(
            grad_y.contiguous(), buf, plan.inv, score, plan.n_tokens, plan.top_k)
        return dbuf, dscore.view_as(score), None


class MapPlan:
    r"""Which rows tokens become where `routing_map` (bool [tokens, experts], on the GPU) says which
    expert takes which token: any number of experts per token, as with experts that choose their
    tokens or with thresholds.  Rows are numbered expert by expert, an expert's in token order.

    `max_rows`: rows of the sorted buffers, e.g. experts * capacity; what the map has beyond is cut
    off (the last experts' last tokens), and rows it does not fill stay as they were allocated.
    Without it the map's entries are counted and read back to the host.

    counts    int64[E]   rows per expert, on the device
    segments  SegmentTable of them, as the expert layers take it
    """

    def __init__(self, routing_map: torch.Tensor, max_rows=None):
        if routing_map.dim() != 2 or routing_map.dtype != torch.bool:
            raise RuntimeError("routing_map must be bool [tokens, experts]")
        if max_rows is None:
            max_rows = int(routing_map.sum())
        self.counts, seg_off, self.token_off, self.pairs = fmoe_cuda.map_plan(
            routing_map.contiguous(), int(max_rows))
        self.n_tokens, self.num_expert = routing_map.shape
        self.max_rows = int(max_rows)
        self.segments = SegmentTable(seg_off, self.counts, self.max_rows)

    @property
    def n_rows_dev(self) -> torch.Tensor:
        """Device int32 holding the number of live rows (= seg_off[E])."""
        return self.segments.seg_off[-1:]

    def _tensors(self):
        return self.segments.seg_off, self.token_off, self.pairs


class _MapExpand(Function):
    r"""sort_tokens operator by operator; map_reduce is its gradient."""

    @staticmethod
    def forward(ctx, x, weight, *plan):
        x = x.contiguous()
        weight = None if weight is None else weight.contiguous()
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight, *plan)
        return fmoe_cuda.map_expand(x, weight, *plan)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, *plan = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        dx, dw = fmoe_cuda.map_reduce(grad.contiguous(), weight, *plan, x if need_dw else None,
                                      need_dx)
        return dx, dw, None, None, None


class _MapReduce(Function):
    r"""unsort_tokens operator by operator; map_expand is its gradient."""

    @staticmethod
    def forward(ctx, rows, weight, *plan):
        rows = rows.contiguous()
        weight = None if weight is None else weight.contiguous()
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weight, *plan)
        return fmoe_cuda.map_reduce(rows, weight, *plan)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weight, *plan = ctx.saved_tensors
        need_drows, need_dw = ctx.needs_input_grad[:2]
        drows, dw = fmoe_cuda.map_expand(grad.contiguous(), weight, *plan,
                                         rows if need_dw else None, True, need_drows)
        return drows, dw, None, None, None


def _no_trace(name):
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{name}: a MapPlan would be a constant of the trace")


def sort_tokens(x: torch.Tensor, plan: MapPlan, weight=None) -> torch.Tensor:
    r"""rows [plan.max_rows, d]: weight[t, e] * x[t] for every token t that expert e takes, in the
    order of `plan`.  x [tokens, d] float32, float16 or bfloat16; weight [tokens, experts] float32
    or of x's dtype (None: ones), read where the map is true; both get gradients, the weight's zero
    elsewhere."""
    native = fmoe_cuda.native()
    if native is not None:
        return native.sort_tokens(x, weight, *plan._tensors())
    _no_trace("sort_tokens")
    return _MapExpand.apply(x, weight, *plan._tensors())


def unsort_tokens(rows: torch.Tensor, plan: MapPlan, weight=None) -> torch.Tensor:
    r"""y [tokens, d]: the sum over the experts e that take token t of weight[t, e] * (t's row of
    e's), summed in float32 in the order of the experts; zero for a token that nobody takes.  Types
    and gradients as of sort_tokens; rows behind the last of the map's get a gradient of zero."""
    native = fmoe_cuda.native()
    if native is not None:
        return native.unsort_tokens(rows, weight, *plan._tensors())
    _no_trace("unsort_tokens")
    return _MapReduce.apply(rows, weight, *plan._tensors())


class TopKSoftmax(Function):
    r"""(idx, score) = top-k of the logits and the softmax over the k values,
    the two torch calls of fmoe/gates/naive_gate.py:31-38 as one kernel each
    way.  idx is ordered by descending logit and carries no gradient."""

    @staticmethod
    def forward(ctx, logits, top_k: int):
        idx, score = fmoe_cuda.topk_softmax_fwd(logits.contiguous(), top_k)
        ctx.n_expert = logits.shape[1]
        ctx.save_for_backward(idx, score)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)   # no zero tensor for idx's "gradient"
        return idx, score

    @staticmethod
    def backward(ctx, _grad_idx, grad_score):
        if grad_score is None:
            return None, None
        idx, score = ctx.saved_tensors
        return fmoe_cuda.topk_softmax_bwd(grad_score.contiguous(), score, idx,
                                          ctx.n_expert), None


SCORES = {"sigmoid": 0, "softmax": 1}      # FMOE_SCORE_* of the C ABI


class ScoreTopK(Function):
    r"""(idx, weight) of scored routing, one kernel each way; idx carries no gradient."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, n_group, top_group, group_best, score, renormalize,
                scale):
        logits = logits.contiguous()
        idx, weight = fmoe_cuda.score_topk_fwd(logits, bias, top_k, n_group, top_group,
                                               group_best, score, renormalize, scale)
        ctx.args = score, renormalize, scale
        ctx.save_for_backward(logits, idx)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return idx, weight

    @staticmethod
    @once_differentiable
    def backward(ctx, _grad_idx, grad_weight):
        if grad_weight is None:
            return (None,) * 9
        logits, idx = ctx.saved_tensors
        return (fmoe_cuda.score_topk_bwd(grad_weight.contiguous(), logits, idx, *ctx.args),
                ) + (None,) * 8


def score_topk(logits, top_k: int, bias=None, score: str = "sigmoid", n_group: int = 1,
               top_group: int = 1, group_best: int = 2, renormalize: bool = True,
               scale: float = 1.0):
    r"""Scored routing of logits [..., E] on the GPU: `(idx [T, k] int64, weight [T, k])`.

    The scores s are the sigmoid or the softmax of the logits.  Experts are chosen by
    v = s + bias (`bias`: float32 [E], e.g. a load-balancing bias; it takes no part in the
    weights and gets no gradient) among the `top_group` best of `n_group` equal groups of
    consecutive experts, a group counting the sum of its `group_best` (1 or 2) largest v;
    ties go to the lower index.  The weights are the chosen scores, divided by their sum if
    `renormalize`, times `scale`.  An expert whose logit or bias is -inf is never chosen; a
    slot for which nobody is left is -1 (a dropped slot) with weight 0."""
    kind = SCORES.get(score)
    if kind is None:
        raise ValueError(f"score must be one of {sorted(SCORES)}, not {score!r}")
    native = fmoe_cuda.native()
    if native is not None:
        return native.score_topk(logits, bias, top_k, n_group, top_group, group_best, kind,
                                 renormalize, scale)
    flat = logits.reshape(-1, logits.shape[-1])
    if bias is not None:
        bias = bias.detach().to(torch.float32).contiguous()
    return ScoreTopK.apply(flat, bias, top_k, n_group, top_group, group_best, kind, renormalize,
                           scale)


class Gelu(Function):
    r"""The exact (erf) GELU between the two expert layers, the
    `self.activation(x)` of fmoe/transformer.py:28-30 for torch.nn.GELU(), as
    one kernel each way."""

    @staticmethod
    def forward(ctx, x, n_rows_dev=None):
        x = x.contiguous()
        ctx.save_for_backward(x)
        ctx.n_rows_dev = n_rows_dev
        return fmoe_cuda.gelu_fwd(x, n_rows_dev)

    @staticmethod
    def backward(ctx, grad_y):
        (x,) = ctx.saved_tensors
        return fmoe_cuda.gelu_bwd(grad_y.contiguous(), x, ctx.n_rows_dev), None


def apply_activation(activation, x, n_rows_dev=None):
    r"""`activation(x)`; an exact torch.nn.GELU on a GPU tensor runs as the
    library's kernel, anything else as the module itself.  `n_rows_dev` (device
    int32[1], optional): the rows of x behind that count are dead (slots a
    capacity limit dropped) and the kernel skips them."""
    if (type(activation) is torch.nn.GELU and "forward" not in activation.__dict__
            and getattr(activation, "approximate", "none") == "none"
            and x.is_cuda and x.dtype in (torch.float32, torch.float64, torch.float16,
                                          torch.bfloat16)):
        return Gelu.apply(x, n_rows_dev)
    return activation(x)


def topk_softmax(logits, top_k: int):
    r"""Top-k gate decision of logits [..., E]: `(idx [T, k] int64, score [T, k])`.
    On the GPU, for k up to fmoe_cuda.MAX_GATE_TOP_K, one fused kernel each way.
    The gate is host-side torch code in the reference (naive_gate.py:31-38), and a
    gate module may live on the CPU or ask for a larger k: those two cases keep the
    reference's own torch.topk + softmax formulation."""
    flat = logits.reshape(-1, logits.shape[-1])
    if flat.is_cuda and top_k <= fmoe_cuda.MAX_GATE_TOP_K and flat.dtype in (
            torch.float32, torch.float64, torch.float16, torch.bfloat16):
        return TopKSoftmax.apply(flat, top_k)
    val, idx = torch.topk(flat, k=top_k, dim=-1, largest=True, sorted=False)
    return idx, torch.nn.functional.softmax(val, dim=-1)
