"""Adapters beside heads whose classes have scales far apart, classes without any weight among them: what is kept of
each class's products."""
import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from train_common import U24

pytestmark = pytest.mark.gpu

N, K, RANK = 96, 120, 4


def adapted(rh, rng, w, quant, up):
    """A head of weights w, and an adapter of the sizes `up` [n, 1] in slot 0."""
    h = ac.Head(rh, rng, N, K, quant, 1, RANK, ranks=[0])
    h.bias = np.zeros(N, np.float32)
    if quant:
        qw = rh.QuantizedWeight.from_f32_transposed(w)
        h.base = rh.RecHead(qw=qw, bias=h.bias)
        h.w = qw.data.astype(np.float64) * qw.scales.astype(np.float64)[:, None]
    else:
        h.base = rh.RecHead(w_t=w, bias=h.bias)
        h.w = w.astype(np.float64)
    h.head = rh.AdaptedHead(h.base, 1, RANK)
    sign = lambda shape: np.where(rng.random(shape) < 0.5, -1.0, 1.0)
    down = (rng.uniform(0.5, 1, (RANK, K)) * sign((RANK, K)) / np.sqrt(K)).astype(np.float32)
    h.set(0, down, (rng.uniform(0.5, 1, (N, RANK)) * sign((N, RANK)) * up).astype(np.float32), 1.0)
    return h


def check(h, rng, label):
    """Rows of one value each, so that few roundings hide what the operands lost.  Halves keep 2^-22: of the row, down
    and u each once, of up once, and the two products of low halves left out: 6 for an adapter's product, one more for the
    row's value in u; 3 for the head's (relative to the class's largest weight).  Sums of 3 products a rank and of 3 of the
    head's, u's 3, up's two roundings and some of the epilogue: 3 rank + 12 half steps."""
    m = 40
    a = np.zeros((m, K), np.float32)
    a[np.arange(m), rng.integers(0, K, m)] = (2.0 ** 13 * rng.uniform(1, 2, m)).astype(np.float32)
    down, up, scale = h.adapters[0]
    a64 = a.astype(np.float64)
    z = a64 @ h.w.T + (a64 @ down.T) @ up.T
    mag = (np.abs(a64) @ np.abs(down).T) @ np.abs(up).T
    head = np.abs(a64).max(axis=1, keepdims=True) * np.abs(h.w).max(axis=1)
    e = mag * (7 * 2.0 ** -22 + (3 * RANK + 12) * U24) + head * (3 * 2.0 ** -22 + (3 * RANK + 12) * U24)
    off, slot = [0, m], [0]
    tc.close(ac.Call(h, a, off, slot).logits().get(), z, e, label)
    o = ac.Call(h, a, [0, m // 2, m], [0, 0]).decode()
    top = z.max(axis=1)
    assert (z[np.arange(m), o["idx"].get()] >= top - 2 * e.max(axis=1)).all(), label


@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-5, 1e-7, 1e-8])
@pytest.mark.parametrize("quant", [True, False], ids=["q", "w"])
def test_classes_of_zeros(rh, quant, size):
    """Unused classes do not cost the others' adapters any bits, and keep their own."""
    rng = np.random.default_rng(1)
    w = (rng.standard_normal((N, K)) * size).astype(np.float32)
    w[[0, 7, 40, N - 1]] = 0.0
    h = adapted(rh, rng, w, quant, size)
    check(h, rng, f"zeros beside weights of {size}")
    a = (rng.standard_normal((9, K)) * 2).astype(np.float32)
    assert np.array_equal(h.head.logits(a), h.base.logits(a))


def test_nothing_but_zeros(rh):
    for quant in (True, False):
        rng = np.random.default_rng(2)
        check(adapted(rh, rng, np.zeros((N, K), np.float32), quant, 0.05), rng, f"zeros, INT8 {quant}")


def test_zeros_of_any_scale(rh):
    """A head of zeros whose scales lie further apart than any units may."""
    rng = np.random.default_rng(4)
    h = adapted(rh, rng, np.zeros((N, K), np.float32), True, 0.05)
    qw = rh.QuantizedWeight.from_f32_transposed(np.zeros((N, K), np.float32))
    qw.scales[:] = 2.0 ** rng.integers(-34, 90, N)
    h.base = rh.RecHead(qw=qw, bias=h.bias)
    h.head = rh.AdaptedHead(h.base, 1, RANK)
    h.set(0, *(v.astype(np.float32) for v in h.adapters[0][:2]), 1.0)
    check(h, rng, "zeros of any scale")


@pytest.mark.parametrize("common", [False, True], ids=["own", "common"])
@pytest.mark.parametrize("quant,size", [(True, 1e-3), (True, 1e-5), (True, 1e-6), (True, 1e-7), (False, 1e-3), (False, 1e-5)])
def test_scales_far_apart(rh, quant, size, common):
    """One class of weights far above the others', the adapter in proportion to each class's weights or the same in
    all."""
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((N, K)) * size).astype(np.float32)
    w[11] = (rng.standard_normal(K) * 0.5).astype(np.float32)
    up = np.full((N, 1), 0.5 if common else size)
    up[11] = 0.5
    check(adapted(rh, rng, w, quant, up), rng, f"one class above {size}")


@pytest.mark.parametrize("apart", range(8, 15))
def test_zeros_keep_22_bits(rh, apart):
    """A class of zeros beside scales of 2^-apart: with a row, a down and a scale of powers of two its logit is the product
    of the row's value and up, exactly, if 22 bits of up are kept (24 hold the sum of both halves' products)."""
    rng = np.random.default_rng(5)
    w = rng.integers(-126, 127, (N, K)) * 2.0 ** -apart
    w[:, 3] = 127 * 2.0 ** -apart  # the largest value: the scale
    w[[7, 40]] = 0.0
    h = adapted(rh, rng, w.astype(np.float32), True, 0.0)
    down = np.zeros((1, K), np.float32)
    down[0, 5] = 1.0
    up = ((2 ** 21 + 2 * rng.integers(0, 2 ** 20, (N, 1)) + 1) * 2.0 ** (6 - apart - 21)).astype(np.float32)  # half the weights' size
    h.set(0, down, up, 1.0)
    a = np.zeros((1, K), np.float32)
    a[0, 5] = 2.0 ** 13
    z = h.head.logits_lines(a, [0, 1], [0])
    assert np.array_equal(z[0, [7, 40]], 2.0 ** 13 * up[[7, 40], 0])


def bits22(rng, n, power):
    """Odd numbers of 22 bits in [2^power, 2^(power + 1)), of either sign."""
    v = (2 ** 21 + 2 * rng.integers(0, 2 ** 20, n) + 1) * 2.0 ** (power - 21)
    return (v * np.where(rng.random(n) < 0.5, -1, 1)).astype(np.float32)


@pytest.mark.parametrize("apart", [0, 4, 11, 12, 13, 14, 17, 21])
def test_22_bits_of_int8_classes_far_apart(rh, apart):
    """Half of the classes 2^apart below the others, the adapter in proportion: its products are exact, as those of zeros."""
    rng = np.random.default_rng(6)
    power = np.where(np.arange(N) % 2 == 0, -8, -8 - apart)
    w = rng.integers(-126, 127, (N, K)) * 2.0 ** power[:, None]
    w[:, 3], w[:, 5] = 127 * 2.0 ** power, 0.0
    h = adapted(rh, rng, w.astype(np.float32), True, 0.0)
    # a down whose sum all but fills its power of two: half of it where the row is
    down = np.full((1, K), 0.499 / (K - 1), np.float32)
    down[0, 5] = 0.5
    up = (bits22(rng, N, 6) * 2.0 ** power).astype(np.float32)[:, None]
    h.set(0, down, up, 1.0)
    a = np.zeros((1, K), np.float32)
    a[0, 5] = 2.0 ** 13
    assert np.array_equal(h.head.logits_lines(a, [0, 1], [0])[0], 2.0 ** 12 * up[:, 0])


@pytest.mark.parametrize("apart", [0, 4, 8, 9, 11, 12, 13, 14])
def test_22_bits_of_fp32_classes_far_apart(rh, apart):
    """The same beside an FP32 head, whose own weights keep their bits as well."""
    rng = np.random.default_rng(7)
    power = np.where(np.arange(N) % 2 == 0, -3, -3 - apart)
    w = (rng.uniform(-1, 1, (N, K)) * 2.0 ** power[:, None]).astype(np.float32)
    w[:, 3], w[:, 5] = bits22(rng, N, -1) * 2.0 ** power, 0.0
    h = adapted(rh, rng, w, False, 0.0)
    down = np.full((1, K), 0.499 / (K - 1), np.float32)
    down[0, 5] = 0.5
    up = (bits22(rng, N, -1) * 2.0 ** power).astype(np.float32)[:, None]
    h.set(0, down, up, 1.0)
    a = np.zeros((2, K), np.float32)
    a[0, 5], a[1, 3] = 2.0 ** 13, 2.0 ** 13
    z = h.head.logits_lines(a, [0, 1, 2], [0, -1])
    assert np.array_equal(z[0], 2.0 ** 12 * up[:, 0])
    assert np.array_equal(z[1], 2.0 ** 13 * w[:, 3])


@pytest.mark.parametrize("quant", [True, False], ids=["q", "w"])
@pytest.mark.parametrize("apart,over", [(0, 16), (12, 16), (21, 16), (0, 28), (3, 25)])
def test_the_heads_bits_beside_large_adapters(rh, quant, apart, over):
    """An adapter 2^16 times an FP32 head's largest weight or an INT8 head's largest scale (2^28 times the least, where that
    is more): the head's products keep 22 bits of a row that the adapter does not meet."""
    rng = np.random.default_rng(8)
    power = np.where(np.arange(N) % 2 == 0, -8, -8 - apart)
    w = rng.integers(-126, 127, (N, K)) * 2.0 ** power[:, None]
    w[:, 3], w[:, 5], w[:, 7] = 127 * 2.0 ** power, 0.0, 64 * 2.0 ** power
    h = adapted(rh, rng, w.astype(np.float32), quant, 0.0)
    down = np.zeros((1, K), np.float32)
    down[0, 5] = 1.0
    largest = 2.0 ** -8 if quant else 127 * 2.0 ** -8
    h.set(0, down, np.full((N, 1), largest * 2.0 ** over, np.float32), 1.0)
    a = np.zeros((3, K), np.float32)
    a[:, 7] = bits22(rng, 3, 0) * np.array([2.0 ** 14, 2.0 ** -20, 1], np.float32)
    z = h.head.logits_lines(a, [0, 3], [0])
    assert np.array_equal(z, (a[:, 7:8].astype(np.float64) * w[:, 7]).astype(np.float32))
