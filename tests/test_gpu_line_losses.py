"""Losses over lines of steps where a term, a sum or a mean leaves the numbers of 32 bits, and where only some of the
outputs are asked for."""
import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from test_gpu_sequence_loss import Policy, Preference

pytestmark = pytest.mark.gpu

# lines in one workgroup each, and lines that several share
LENGTHS = [[5, 1, 70], [900, 300], [40000, 3000, 20000]]


def outputs_of(job, keys=None):
    o = job.outputs()
    return {k: v.get() for k, v in job.run({k: o[k] for k in (keys or o)}).items()}


@pytest.mark.parametrize("lengths", LENGTHS, ids=["short", "long", "split"])
def test_divergences_without_a_weight(rh, lengths):
    """beta 0 and a reference: the divergence is reported, infinite where 32 bits do not hold it, and is no part of the
    loss and of the gradients."""
    rng = np.random.default_rng(1)
    off = ac.offsets(lengths)
    m = int(off[-1])
    loss = (rng.random(m) * 3).astype(np.float32)
    ref = (loss + rng.standard_normal(m) * 0.3).astype(np.float32)
    loss[::5] += 100
    ref[::5] = 0.5
    old = (loss + rng.standard_normal(m) * 0.2).astype(np.float32)
    job = Policy(rh, loss, old, ref, None, rng.standard_normal(len(lengths)).astype(np.float32), off, beta=0.0)
    got = outputs_of(job)
    kl = got.pop("kl")
    assert (kl[np.add.reduceat(loss > 90, off[:-1]) > 0] == np.inf).all() and not np.isnan(kl).any()
    job.check(got, "beta 0")


@pytest.mark.parametrize("lengths", LENGTHS, ids=["short", "long", "split"])
def test_means_of_large_values(rh, lengths):
    """Values whose sum passes the largest number of 32 bits, and their mean does not."""
    off = ac.offsets(lengths)
    m = int(off[-1])
    loss = np.full(m, 88.0, np.float32)
    adv = np.array([3e38, -3e38, 1e38], np.float32)[:len(lengths)]
    job = Policy(rh, loss, loss, np.full(m, 0.5, np.float32), None, adv, off, beta=1.0)  # divergences of e^87.5
    got = outputs_of(job)
    assert np.isfinite(got["kl"]).all()
    # a step's value in the second line, and its slope in the first, is 3e38 + e^87.5 = 4.0e38 itself, above the largest
    # number, 3.4028e38
    assert (np.isinf(got["loss"]) == (np.arange(len(lengths)) == 1)).all()
    want, tol = ac.policy64(loss, loss, np.full(m, 0.5, np.float32), None, adv, False, off, 0.2, 0.28, 1.0)
    want["loss"][1:2] = np.inf
    want["row_grad"][:off[1]] = got["row_grad"][:off[1]]
    for k, v in got.items():
        tc.close(v, want[k], tol[k], f"means {k}")


def test_all_smoothing_under_an_infinite_margin(rh):
    """smoothing 1 is the other line's loss alone, whatever the margin."""
    loss = np.array([3e38] * 4 + [0.5, 1.0] + [3e38] * 4, np.float32)
    off = [0, 4, 5, 6, 10]
    job = Preference(rh, loss, None, None, off, 1.0, 1.0)
    got = outputs_of(job, ("loss", "row_grad"))
    assert got["loss"][0] == 0 and got["loss"][1] == np.inf
    want, tol = ac.preference64(loss, None, None, off, 1.0, 1.0, False)
    tc.close(got["row_grad"], want["row_grad"], tol["row_grad"], "row_grad")
