r"""Scored top-k routing with a load-balancing bias and groups of experts.  The reference
has no such gate; this one keeps the interface of fmoe/gates/naive_gate.py."""
import torch

from .. import fmoe_cuda
from ..functions import score_topk
from .naive_gate import NaiveGate


class ScoreGate(NaiveGate):
    r"""logits = Linear(d_model, experts); `functions.score_topk` of them picks the experts and
    gives the combine weights.  Returns `(idx [..., k] int64, weight [T, k])`, plus the full
    logits when `return_all_scores`.

    * `score`: "sigmoid" or "softmax" of the logits.
    * `n_group`, `top_group`, `group_best`: experts only of the `top_group` best of `n_group`
      groups, a group counting its `group_best` best experts.
    * `renormalize`, `scale`: of the weights.
    * `balance_bias` (float32 buffer [experts], kept in float32 whatever dtype the layer is
      converted to): added to the scores for the choice alone.  In training every forward pass
      adds its choices to the buffer `load`; `update_bias(speed)` moves the bias by `speed`
      towards the experts that had less than the mean and clears the counts.  No auxiliary
      loss is involved: `get_loss()` is zero.

    Layers build their gate from the class: `FMoETransformerMLP(gate=ScoreGate.configured(
    n_group=8, top_group=3), ...)`."""

    def __init__(self, d_model, num_expert, world_size, top_k=2, gate_bias=True,
                 score="sigmoid", n_group=1, top_group=1, group_best=2, renormalize=True,
                 scale=1.0):
        super().__init__(d_model, num_expert, world_size, top_k=top_k, gate_bias=gate_bias)
        self.options = dict(score=score, n_group=n_group, top_group=top_group,
                            group_best=group_best, renormalize=renormalize, scale=scale)
        self.register_buffer("balance_bias", torch.zeros(self.tot_expert))
        self.register_buffer("load", torch.zeros(self.tot_expert, dtype=torch.int32),
                             persistent=False)

    @classmethod
    def configured(cls, **options):
        r"""A subclass whose constructor's defaults are `options`.  What it makes are instances of
        this class (the options are theirs), so that they can be pickled."""
        def init(self, *args, **kwargs):
            cls.__init__(self, *args, **{**options, **kwargs})
            if type(self) is made:
                self.__class__ = made._made_from
        made = type(cls.__name__, (cls,), {
            "__init__": init, "_made_from": cls.__dict__.get("_made_from", cls)})
        return made

    def _apply(self, fn, recurse=True):
        bias = self.balance_bias
        super()._apply(fn, recurse)
        if self.balance_bias.dtype != bias.dtype:    # converted with the layer's parameters
            self.balance_bias = bias.to(self.balance_bias.device)
        return self

    def forward(self, inp, return_all_scores=False):
        logits = self.gate(inp)
        idx, weight = score_topk(logits, self.top_k, bias=self.balance_bias, **self.options)
        if self.training:
            fmoe_cuda.expert_count(idx, self.load)
        idx = idx.view(*logits.shape[:-1], self.top_k)
        self.set_loss(torch.zeros(1, device=inp.device, requires_grad=True))
        if return_all_scores:
            return idx, weight, logits
        return idx, weight

    @torch.no_grad()
    def update_bias(self, speed=1e-3):
        r"""bias += speed * sign(mean load - load), from the choices counted since the last
        call."""
        load = self.load.float()
        self.balance_bias += speed * torch.sign(load.mean() - load)
        self.load.zero_()
