"""The statement of scored routing that the GPU tests compare with, against differences (no
GPU needed)."""
import numpy as np
import pytest

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
