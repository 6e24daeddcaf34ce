"""Rows and classes of the losses whose magnitudes lie far apart within a group of 32: the small ones
keep their bits, whatever stands next to them."""
import numpy as np
import pytest

import train_common as tc
from loss_scales import compare, reference, run, targets, without_target
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

DT = pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
SIZE = pytest.mark.parametrize("size", [1e6, 1e10, 1e30])


@pytest.mark.parametrize("kind", ["xent", "distill"])
@SIZE
@DT
def test_padding_may_hold_any_number(rh, dt, size, kind):
    """Single rows of huge values in groups of 32, without a target or with a gradient of 0: their
    neighbours' losses and all gradients are what they are without them."""
    rng = np.random.default_rng(31)
    m, n, k = 100, 500, 120
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    t = targets(kind, rng, m, n, to)
    grad = (0.5 + rng.random(m)).astype(np.float32)
    pad = np.array([3, 31, 40, 97])
    without_target(t, pad[:3])
    grad[pad[3]] = 0.0
    a[pad] = (rng.standard_normal((4, k)) * size).astype(np.float32)
    rows = np.setdiff1d(np.arange(m), pad)
    got, _ = compare(rh, a, w, b, dt, t, grad, rows, np.arange(n), f"{kind} padding {size}")
    assert (got["da"][pad] == 0).all() and (got["loss"][pad[:3]] == 0).all()


@pytest.mark.parametrize("kind", ["xent", "distill"])
@SIZE
@DT
def test_rows_next_to_a_large_one(rh, dt, size, kind):
    """The same with a target.  The large row's own probabilities are 0 or 1 to the last bit, where
    its logits differ by more than their roundings; the other rows and the classes that it does not
    lean to keep their losses and gradients."""
    rng = np.random.default_rng(32)
    m, n, k = 100, 500, 120
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    t = targets(kind, rng, m, n, to)
    grad = (0.5 + rng.random(m)).astype(np.float32)
    large = np.array([5, 70])
    a[large] = (rng.standard_normal((2, k)) * size).astype(np.float32)
    _, av = tc.typed(a, dt)
    _, wv = tc.typed(w, dt)
    z = av[large].astype(np.float64) @ wv.astype(np.float64).T
    lean = np.nonzero((z > z.max(axis=1, keepdims=True) * (1 - 1e-3)).any(axis=0))[0]
    own = to[large] if kind == "xent" else t["idx"][large].ravel()
    classes = np.setdiff1d(np.arange(n), np.concatenate([lean, own]))
    compare(rh, a, w, b, dt, t, grad, np.setdiff1d(np.arange(m), large), classes, f"{kind} large rows {size}")


@pytest.mark.parametrize("kind", ["xent", "distill"])
@pytest.mark.parametrize("mask", [False, True])
@SIZE
@DT
def test_classes_next_to_a_large_one(rh, dt, size, mask, kind):
    """Single classes of huge weights that no row takes: by the sign of their logits, or masked by
    their bias."""
    rng = np.random.default_rng(33)
    m, n, k = 70, 300, 96
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    a[:, 0] = np.abs(a[:, 0]) + 1.0
    w[:, 0] = np.abs(w[:, 0])
    large = np.array([7, 140, 141, 299])
    to = np.where(np.isin(to, large), 11, to).astype(np.int32)
    t = targets(kind, rng, m, n, to)
    if kind == "distill":
        t["idx"] = np.where(np.isin(t["idx"], large), 12, t["idx"]).astype(np.int32)
    w[large] = 0.0
    if mask:
        w[large] = rng.choice([-size, size], (4, k)).astype(np.float32)
        b[large] = -np.inf
    else:
        w[large, 0] = -size
    compare(rh, a, w, b, dt, t, None, np.arange(m), np.arange(n), f"{kind} large classes {size}")


@DT
def test_a_row_and_its_neighbours_do_not_meet(rh, dt):
    """A row's loss does not depend on the other rows of the call, but for roundings: next to rows of
    zeros, like ones and far larger ones."""
    rng = np.random.default_rng(34)
    m, n, k = 64, 400, 80
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    want, _, _ = run(rh, a, w, b, dt, {"target": to})
    for size in (0.0, 1.0, 1e4, 1e20):
        other = a.copy()
        other[1::2] = (rng.standard_normal((m // 2, k)) * size).astype(np.float32)
        got, av, wv = run(rh, other, w, b, dt, {"target": to})
        ref, z, p, dz, s, al, q, logq = reference(av, wv, b, {"target": to}, None)
        tol = tc.loss_tol(av, wv, b, z, p, dz, s, al, ref, dt, 1.0, q, logq)
        rows = np.arange(0, m, 2)
        for key in ("loss", "lse"):
            tc.close(got[key][rows], want[key][rows], 2 * tol[key][rows], f"{key} next to {size}")


@pytest.mark.parametrize("kind", ["xent", "distill"])
@pytest.mark.parametrize("m,n,k", [(300, 700, 40), (257, 300, 120), (150, 400, 180), (140, 130, 256), (1000, 2100, 64)])
@DT
def test_unlike_rows_and_classes(rh, dt, m, n, k, kind):
    """Rows and classes of ordinary sizes and of a 64th and 64 times those in every group of both."""
    rng = np.random.default_rng(m + k)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    a *= rng.choice([1 / 64, 1, 1, 1, 8], (m, 1)).astype(np.float32)
    a[::17] *= np.float32(8)
    w *= rng.choice([1 / 64, 1, 1, 4], (n, 1)).astype(np.float32)
    t = targets(kind, rng, m, n, to)
    grad = (rng.standard_normal(m) * 2.0 ** rng.integers(-12, 1, m)).astype(np.float32)
    compare(rh, a, w, b, dt, t, grad, np.arange(m), np.arange(n), f"{kind} unlike")
