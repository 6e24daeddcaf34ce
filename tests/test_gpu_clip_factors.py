"""Gradient clipping by factors that 32 bits hold in few bits or not at all."""
import numpy as np
import pytest

import train_common as tc
from test_gpu_grad_clip import Clip, tensors
from train_common import F32, HALF, LEAST, U24

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("size,most", [(1e37, 1e-3), (1e37, 1e-8), (1e36, 1e-30), (1e30, 3e-9)])
def test_tiny_factors(rh, size, most, shift):
    """The factor is rounded once at most, the product once, and the stored value."""
    rng = np.random.default_rng(1)
    job = Clip(rh, tensors(rng, [500, 3001, 9, 20000], scale=size), shift)
    out, norm = job.run(most)
    total = np.sqrt(sum(float((v.astype(np.float64) ** 2).sum()) for v in job.val))
    with np.errstate(over="ignore"):
        assert norm.get()[0] in (np.float32(total), np.nextafter(np.float32(total), np.float32(0)),
                                 np.nextafter(np.float32(total), np.float32(np.inf)))
    factor = float(np.float32(most)) / total
    for i, (o, v, dt) in enumerate(zip(out, job.val, job.dts)):
        w = v.astype(np.float64) * factor
        e = np.abs(w) * 3 * U24
        # (bf16 from fp32: numbers of 32 bits first, whose least step is 2^-149)
        tc.close(o.get(), w, e + HALF[dt] * (np.abs(w) + e) + LEAST[dt] + LEAST[F32], f"{size} {most} {i}")
    want = [o.get() for o in out]
    job.run(most, in_place=True)
    for w, d in zip(want, job.dev):
        assert np.array_equal(d.numpy()[shift:], w)


def test_a_norm_beyond_32_bits(rh):
    """It is held in 64 bits and scales the gradients; what is written of it is infinity."""
    x = np.full(1000, 3e38, np.float32)
    job = Clip(rh, [(x, F32)])
    out, norm = job.run(1.0)
    assert norm.get()[0] == np.inf
    tc.close(out[0].get(), np.full(1000, 1000 ** -0.5), np.full(1000, 4 * U24 * 1000 ** -0.5), "scaled")
