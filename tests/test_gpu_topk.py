"""ppocr_topk_rows against a stable sort: values, columns, ties by column, NaN, missing places."""
import numpy as np
import pytest

import train_common as tc

pytestmark = pytest.mark.gpu


def topk_ref(x, top):
    rows, cols = x.shape
    idx = np.full((rows, top), -1, np.int32)
    val = np.full((rows, top), -np.inf, np.float32)
    for r in range(rows):
        ok = np.nonzero(~np.isnan(x[r]))[0]
        order = ok[np.argsort(-x[r, ok].astype(np.float64), kind="stable")][:top]
        idx[r, :order.size], val[r, :order.size] = order, x[r, order]
    return idx, val


def run(rh, x, top):
    from ppocr_rechead.hip import synchronize
    rows, cols = x.shape
    dx, oi, ov = tc.up(x), tc.Out((rows, top), np.int32), tc.Out((rows, top), np.float32)
    rh._check(rh._lib.lib().ppocr_topk_rows_dev(dx.p, rows, cols, top, oi.p, ov.p, None))
    synchronize()
    return oi.get(), ov.get()


def check(rh, x, top, label):
    print(f"topk {label} {x.shape} top={top}", flush=True)
    idx, val = run(rh, x, top)
    ri, rv = topk_ref(x, top)
    assert np.array_equal(idx, ri), label
    assert np.array_equal(val, rv), label


@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (3, 5, 5), (2, 7, 16), (5, 64, 1), (4, 255, 64), (3, 257, 64), (7, 1000, 17),
                                           (33, 6906, 32), (20, 18710, 16), (3, 20480, 64), (3, 20481, 64), (2, 70001, 64)])
def test_random_rows(rh, rows, cols, top):
    rng = np.random.default_rng(rows + cols + top)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    check(rh, x, top, "random")
    check(rh, np.round(x * 2) / 2, top, "ties")
    x[rng.random((rows, cols)) < 0.3] = np.nan
    x[rng.random((rows, cols)) < 0.1] = np.inf
    x[rng.random((rows, cols)) < 0.3] = -np.inf
    check(rh, x, top, "nan and infinities")


def test_special_rows(rh):
    cols = 3001
    rows = [np.full(cols, 2.5), np.full(cols, np.nan), np.full(cols, -np.inf), np.arange(cols), np.arange(cols)[::-1],
            np.where(np.arange(cols) % 2, 0.0, -0.0), np.where(np.arange(cols) == 1500, -3.4e38, np.nan),
            np.full(cols, np.inf), np.where(np.arange(cols) % 64 == 5, 100.0 + np.arange(cols), 0.0),
            np.float32(1e-45) * (np.arange(cols) % 5)]
    check(rh, np.stack([np.asarray(r, np.float32) for r in rows]), 64, "special")


def test_all_large_values_in_one_threads_columns(rh):
    """A thread sees every 256th (or 512th, 1024th) column: rows whose largest values all lie there, more of them than
    the candidates' memory holds."""
    rng = np.random.default_rng(2)
    cols = 400000
    x = rng.random((3, cols)).astype(np.float32)
    for i, step in enumerate((64, 256, 1024)):
        x[i, 5::step] += 10.0
    x[1, 6::256] += 20.0
    x[1, 70::256] += 20.0
    check(rh, x, 64, "columns")
    wide = np.zeros((1, 1 << 20), np.float32)
    for t in range(64):
        wide[0, t::4096] = 1.0 + rng.random(wide[0, t::4096].size)
    check(rh, wide, 64, "many candidates")


def test_more_rows_than_workgroups(rh):
    rng = np.random.default_rng(3)
    x = rng.standard_normal(((1 << 20) + 5, 3)).astype(np.float32)
    idx, val = run(rh, x, 2)
    order = np.argsort(-x, axis=1, kind="stable")[:, :2]
    assert np.array_equal(idx, order) and np.array_equal(val, np.take_along_axis(x, order, 1))


def test_unaligned_rows_and_host_form(rh):
    from ppocr_rechead.hip import synchronize
    import ctypes
    rng = np.random.default_rng(4)
    x = rng.standard_normal((9, 1003)).astype(np.float32)
    d = tc.up(np.concatenate([np.zeros(1, np.float32), x.ravel()]))
    oi, ov = tc.Out((9, 11), np.int32), tc.Out((9, 11), np.float32)
    rh._check(rh._lib.lib().ppocr_topk_rows_dev(ctypes.c_void_p(d.p.value + 4), 9, 1003, 11, oi.p, ov.p, None))
    synchronize()
    ri, rv = topk_ref(x, 11)
    assert np.array_equal(oi.get(), ri) and np.array_equal(ov.get(), rv)
    hi, hv = rh.topk(x, 11)
    assert np.array_equal(hi, ri) and np.array_equal(hv, rv)
