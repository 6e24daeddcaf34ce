"""Classes that are improbable in every row, and rows whose classes nearly all are: their gradients are
as near to the formulas as the others', measured against themselves."""
import numpy as np
import pytest

import train_common as tc
from loss_scales import compare, reference, run, targets
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

DT = pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])


@pytest.mark.parametrize("kind", ["xent", "distill"])
@pytest.mark.parametrize("m,n,k", [(150, 300, 120), (700, 200, 64), (33, 500, 200)])
@DT
def test_improbable_classes(rh, dt, m, n, k, kind):
    """Classes of probability 1e-9 to 1e-24 in every row, among ordinary ones: dw, db."""
    rng = np.random.default_rng(m + n)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    rare = np.arange(n) % 3 == 1
    b[rare] -= (20 + 35 * rng.random(int(rare.sum()))).astype(np.float32)
    to = np.where(rare[to], to - 1, to).astype(np.int32)
    t = targets(kind, rng, m, n, to)
    if kind == "distill":
        t["idx"] = np.where(rare[t["idx"]], t["idx"] - 1, t["idx"]).astype(np.int32)
    grad = (0.5 + rng.random(m)).astype(np.float32)
    tau = np.float32(t.get("tau", 1.0))
    compare(rh, a, w * tau, b * tau, dt, t, grad, np.arange(m), np.arange(n), f"{kind} rare classes")


@DT
def test_improbable_classes_under_large_activations(rh, dt):
    """The same with activations 50 times as large and weights as much smaller, and rows among them
    whose gradient is 2^-20 of the others'."""
    rng = np.random.default_rng(41)
    m, n, k = 200, 300, 120
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    rare = np.arange(n) % 4 == 1
    b[rare] -= (20 + 20 * rng.random(int(rare.sum()))).astype(np.float32)
    to = np.where(rare[to], to - 1, to).astype(np.int32)
    grad = np.where(np.arange(m) % 5 == 0, 2.0 ** -20, 1.0).astype(np.float32)
    compare(rh, a * np.float32(50), w / np.float32(50), b, dt, {"target": to}, grad, np.arange(m), np.arange(n),
            "rare classes, large rows")


@DT
def test_a_class_that_few_rows_reach(rh, dt):
    """Classes whose probability comes from one row near the end, after many that give next to
    nothing, and from one near the start, before them: the scale a class's sums are held at moves
    once, and late."""
    rng = np.random.default_rng(42)
    m, n, k = 600, 200, 64
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    rare = np.array([3, 40, 77, 120, 160])
    to = np.where(np.isin(to, rare), 0, to).astype(np.int32)
    # a direction of its own for each, which the other rows do not have
    w[:, :5], a[:, :5], w[rare] = 0.0, 0.0, 0.0
    b[rare] = -30.0
    w[rare, np.arange(5)] = 1.0
    for j, r in enumerate((595, 2, 300, 599, 64)):
        a[r, j] = (28.0, 25.0, 20.0, 10.0, 28.0)[j]
    compare(rh, a, w, b, dt, {"target": to}, None, np.arange(m), np.arange(n), "late classes")


@pytest.mark.parametrize("size", [1e10, 1e30])
@DT
def test_rows_of_which_one_is_large(rh, dt, size):
    """Labelled rows of very different sizes far from each other: dw of the classes that only the
    small ones reach."""
    rng = np.random.default_rng(43)
    m, n, k = 160, 300, 64
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    a[96:128] = (rng.standard_normal((32, k)) * size).astype(np.float32)
    _, av = tc.typed(a, dt)
    _, wv = tc.typed(w, dt)
    z = av[96:128].astype(np.float64) @ wv.astype(np.float64).T
    lean = np.nonzero((z > z.max(axis=1, keepdims=True) * (1 - 1e-3)).any(axis=0))[0]
    classes = np.setdiff1d(np.arange(n), np.concatenate([lean, to[96:128]]))
    rows = np.r_[0:96, 128:160]
    compare(rh, a, w, b, dt, {"target": to}, None, rows, classes, f"a group of large rows {size}")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@DT
def test_gradients_that_are_no_numbers_show(rh, dt, bad):
    """An overflown loss scale: the row's da and what its classes sum are no numbers either, and the
    other rows keep theirs."""
    rng = np.random.default_rng(44)
    a, w, b, to = tc.head_inputs(rng, 70, 100, 40)
    grad = np.ones(70, np.float32)
    want, av, wv = run(rh, a, w, b, dt, {"target": to}, grad)
    grad[33] = bad
    got, _, _ = run(rh, a, w, b, dt, {"target": to}, grad)
    rest = np.arange(70) != 33
    assert not np.isfinite(got["da"][33]).any()
    assert not np.isfinite(got["dw"][to[33]]).any() and not np.isfinite(got["db"][to[33]])
    assert np.array_equal(got["loss"], want["loss"]) and np.array_equal(got["da"][rest], want["da"][rest])


@DT
def test_logits_beyond_what_32_bits_tell_apart(rh, dt):
    """Rows whose logits are so large that lse is off by more than 1: gradients stay numbers, no larger
    than a probability of 1 makes them, and rows next to them are right."""
    rng = np.random.default_rng(45)
    m, n, k = 64, 200, 48
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    large = np.arange(32, 64)
    a[large] = (rng.standard_normal((32, k)) * 1e18).astype(np.float32)
    z = a[large].astype(np.float64) @ w.astype(np.float64).T
    to[large] = z.argmax(axis=1)  # p of the label is 1, its gradient nothing
    got, av, wv = run(rh, a, w, b, dt, {"target": to})
    ref, z, p, dz, s, al, q, logq = reference(av, wv, b, {"target": to}, None)
    for key in ("da", "dw", "db"):
        assert np.isfinite(got[key]).all(), key
    assert (np.abs(got["da"][large]) <= 2.1 * np.abs(wv).max()).all()
    rows = np.arange(32)
    tol = tc.loss_tol(av, wv, b, z, p, dz, s, al, ref, dt, 1.0, q, logq)
    for key in ("loss", "lse", "da"):
        tc.close(got[key][rows], ref[key][rows], tol[key][rows], key)


@pytest.mark.parametrize("kind", ["xent", "distill"])
@DT
def test_improbable_classes_behind_rows_without_target(rh, dt, kind):
    """Every other group of 32 rows, the first among them, has no target: the groups that set the scales
    are the others."""
    rng = np.random.default_rng(46)
    m, n, k = 700, 200, 64
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    rare = np.arange(n) % 3 == 1
    b[rare] -= (20 + 20 * rng.random(int(rare.sum()))).astype(np.float32)
    to = np.where(rare[to], to - 1, to).astype(np.int32)
    t = targets(kind, rng, m, n, to)
    if kind == "distill":
        t["idx"] = np.where(rare[t["idx"]], t["idx"] - 1, t["idx"]).astype(np.int32)
    none = (np.arange(m) // 32) % 2 == 0
    t["target" if kind == "xent" else "idx"][none] = -1
    tau = np.float32(t.get("tau", 1.0))
    got, _ = compare(rh, a, w * tau, b * tau, dt, t, None, np.arange(m), np.arange(n), f"{kind} rare classes, groups of padding")
    assert (got["da"][none] == 0).all()
