"""Whose the advantages of a policy loss are, where their number does not tell."""
import numpy as np
import pytest

import adapt_common as ac
import train_common as tc

X = np.array([1.0, 2.0], np.float32)
ADV = np.array([0.5, -1.5], np.float32)


@pytest.mark.parametrize("off", [[0, 0, 2], [0, 2, 2]])
def test_as_many_lines_as_steps(rh, off):
    """Two lines of two steps, one of them empty: a call that does not say whose they are is refused."""
    with pytest.raises(rh.OcrError, match="PolicyLoss"):
        rh.policy_loss(X, X, ADV, off)


def test_numbers_that_do_not_fit(rh):
    for adv, per_step in ((ADV, False), (ADV[:1], True), (np.ones(3), None), (np.ones((2, 1)), True)):
        with pytest.raises(rh.OcrError, match="PolicyLoss"):
            rh.policy_loss(X, X, adv, [0, 2], per_step=per_step)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [[0, 0, 2], [0, 2, 2], [0, 1, 2]])
@pytest.mark.parametrize("per_step", [False, True])
def test_said(rh, off, per_step):
    got = rh.policy_loss(X, X - 0.25, ADV, off, per_step=per_step)
    want, tol = ac.policy64(X, X - np.float32(0.25), None, None, ADV, per_step, off, 0.2, 0.2, 0.0)
    for k, v in zip(("loss", "kl", "clipped", "row_grad"), got):
        tc.close(v, want[k], tol[k], f"{off} {per_step} {k}")
    if off == [0, 1, 2]:  # a line a step: either is the same, and the call may leave it open
        for a, b in zip(got, rh.policy_loss(X, X - 0.25, ADV, off)):
            assert np.array_equal(a, b)
