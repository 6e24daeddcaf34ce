"""The losses at sizes that choose other kernels and chunks than the small ones: labels of more than 4096
rows, and rows and classes whose numbers are far apart (streams of more than 256 times the other's
length, which are cut by a rule of their own)."""
import numpy as np
import pytest

import train_common as tc
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

DT = pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])


@pytest.mark.parametrize("m,n,k", [(4097, 40, 24), (4111, 300, 33), (5000, 129, 120), (9001, 70, 256)])
@DT
def test_labels_of_many_rows(rh, m, n, k, dt):
    rng = np.random.default_rng(m + n)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    target = np.where(rng.random(m) < 0.3, rng.integers(0, n, m), to).astype(np.int32)
    target[rng.random(m) < 0.1] = -1
    target[[0, 31, m - 1]] = -1, n, -7  # the device form takes n and above as no label
    grad = rng.standard_normal(m).astype(np.float32)
    got, _ = tc.check_step(rh, a, w, b, dt, "many labels", target=target, grad=grad)
    none = (target < 0) | (target >= n)
    assert (got["loss"][none] == 0).all() and (tc.values(got["da"])[none] == 0).all()


@DT
def test_labels_of_many_unaligned_rows(rh, dt):
    """Many labels of rows that start one value past a vector boundary: the same bits."""
    from ppocr_rechead.hip import synchronize
    import ctypes
    rng = np.random.default_rng(51)
    m, n, k = 4200, 64, 40
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    ar, wr = tc.typed(a, dt)[0], tc.typed(w, dt)[0]
    job = tc.Loss(rh, ar, wr, b, dt, to)
    want = job.step()
    size = ar.itemsize

    class Past:
        def __init__(self, x):
            self.d = tc.up(np.concatenate([np.zeros(1, x.dtype), x.ravel()]))
            self.p = ctypes.c_void_p(self.d.p.value + size)

    job.a, job.w = Past(ar), Past(wr)
    o = job.outputs()
    job.forward(o)
    job.backward(o)
    synchronize()
    for key, v in o.items():
        assert np.array_equal(v.get().view(np.uint8), want[key].view(np.uint8)), key


@pytest.mark.parametrize("kind", ["xent", "distill"])
@pytest.mark.parametrize("m,n,k", [(1, 33000, 40), (33, 36001, 64), (128, 40000, 24), (40001, 31, 16), (33333, 90, 8)])
@DT
def test_few_of_one_and_many_of_the_other(rh, m, n, k, kind, dt):
    rng = np.random.default_rng(m + n + k)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    grad = (0.5 + rng.random(m)).astype(np.float32)
    if kind == "xent":
        target = to.copy()
        target[m // 2:m // 2 + (m > 1)] = -1
        tc.check_step(rh, a, w, b, dt, "far apart", target=target, grad=grad)
    else:
        idx, z = tc.teacher_inputs(rng, m, n, 7, to)
        idx[:, 3] = n - 1 - (np.arange(m) % min(n, 200))  # the last classes' records too
        tc.check_step(rh, a, w, b, dt, "far apart", idx=idx, z=z, tau=2.0, grad=grad)
