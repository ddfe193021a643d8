"""The statement of scored routing that the GPU tests compare with, against differences (no
GPU needed)."""
import copy
import io
import pickle

import numpy as np
import pytest
import torch

import mx_reference as R


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_formula_against_differences(kind, renorm):
    rng = np.random.default_rng(5)
    t, e, k = 4, 12, 3
    logits, dweight = rng.standard_normal((t, e)), rng.standard_normal((t, k))
    logits[1, :10] = -np.inf                      # fewer experts than slots
    idx, _, margin = R.score_topk(logits, None, k, kind, renorm=renorm, scale=2.5)
    assert margin.min() > 1e-3                    # the differences below keep the choice
    got = R.score_topk_backward(dweight, logits, idx, kind, renorm, 2.5)
    step = 1e-6
    for r in range(t):
        for i in range(e):
            if np.isneginf(logits[r, i]):
                assert got[r, i] == 0
                continue
            side = []
            for sign in (1, -1):
                moved = logits.copy()
                moved[r, i] += sign * step
                w = R.score_topk(moved, None, k, kind, renorm=renorm, scale=2.5)[1]
                side.append((w * dweight).sum())
            assert abs((side[0] - side[1]) / (2 * step) - got[r, i]) < 1e-8


def test_configured_gates_can_be_pickled_and_copied():
    from fastmoe_amd import FMoETransformerMLP, ScoreGate

    gate = ScoreGate.configured(score="softmax", n_group=4, top_group=2).configured(scale=2.5)
    assert issubclass(gate, ScoreGate)
    layer = FMoETransformerMLP(num_expert=8, d_model=16, d_hidden=32, gate=gate)
    layer.gate.balance_bias.copy_(torch.arange(8.0))
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    for other in (pickle.loads(pickle.dumps(layer)), copy.deepcopy(layer),
                  torch.load(file, weights_only=False)):
        assert type(other.gate) is ScoreGate and other.gate.options == layer.gate.options
        assert torch.equal(other.gate.balance_bias, layer.gate.balance_bias)
        assert torch.equal(other.gate.gate.weight, layer.gate.gate.weight)
    assert layer.gate.options == dict(score="softmax", n_group=4, top_group=2, group_best=2,
                                      renormalize=True, scale=2.5)

    class Own(gate):
        pass

    assert type(Own(16, 8, 1)) is Own and Own(16, 8, 1).options["scale"] == 2.5
