"""An adapter merged into a weight and its gradients against the formulas in 64 bits."""
import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from train_common import BF16, F32

pytestmark = pytest.mark.gpu


class Merge:
    def __init__(self, rh, rng, n, k, rank, dt, scale=1.5, shift=0):
        self.rh, self.L, self.dt, self.scale = rh, rh._lib.lib(), dt, scale
        self.shape = (n, k, rank)
        self.host, self.val = {}, {}
        for key, shape, s in (("w", (n, k), 0.05), ("dw", (n, k), 1e-3), ("down", (rank, k), 0.1), ("up", (n, rank), 0.02)):
            x = rng.standard_normal(shape) * s
            if key == "dw":
                x *= np.exp(rng.standard_normal((n, 1)))
            self.host[key], self.val[key] = tc.typed(x.astype(np.float32), dt)
        # tensors at addresses that are aligned to their type only
        pad = {k_: np.concatenate([np.zeros(shift, v.dtype), v.ravel()]) for k_, v in self.host.items()}
        self.dev = {k_: tc.up(v) for k_, v in pad.items()}
        width = 4 if dt == F32 else 2
        import ctypes
        self.p = {k_: ctypes.c_void_p(v.p.value + shift * width) for k_, v in self.dev.items()}
        self.tdt = np.float32 if dt == F32 else np.uint16
        self.bytes = self.L.ppocr_ra_merge_workspace_bytes(n, k, rank)
        self.ws = tc.Out((self.bytes,), np.uint8)

    def outputs(self):
        n, k, rank = self.shape
        return {"w": tc.Out((n, k), self.tdt), "ddown": tc.Out((rank, k), self.tdt), "dup": tc.Out((n, rank), self.tdt)}

    def run(self, o, stream=None, ws=True):
        n, k, rank = self.shape
        shape = (n, k, rank, self.scale, self.dt)
        if "w" in o:
            self.rh._check(self.L.ppocr_ra_merge_dev(self.p["w"], self.p["down"], self.p["up"], *shape, o["w"].p, stream))
        self.rh._check(self.L.ppocr_ra_merge_backward_dev(self.p["dw"], self.p["down"], self.p["up"], *shape,
                                                          tc.ptr(o.get("ddown")), tc.ptr(o.get("dup")),
                                                          self.ws.p if ws else None, self.bytes if ws else 0, stream))
        return o

    def check(self, got, label):
        v = self.val
        ref, tol = ac.merge64(v["w"], v["dw"], v["down"], v["up"], self.scale, self.dt)
        for key in got:
            tc.close(got[key], ref[key], tol[key], f"{label} {key}")


SHAPES = [(1, 1, 1), (5, 3, 2), (33, 120, 16), (100, 80, 64), (300, 256, 17), (257, 255, 33), (31, 8, 63), (64, 33, 31),
          (2000, 120, 8), (6906, 80, 32), (18710, 120, 16), (9000, 256, 64),
          (3001, 2, 3), (5003, 1, 64), (777, 13, 35), (40001, 7, 17), (20011, 185, 59)]


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_merge_and_gradients(rh, shape, dt):
    print(shape, dt, flush=True)
    job = Merge(rh, np.random.default_rng(sum(shape)), *shape, dt)
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    job.ws.get()
    job.check(got, "merge")
    again = {k: v.get() for k, v in job.run(job.outputs(), ws=False).items()}
    for key in got:
        assert np.array_equal(got[key], again[key]), key


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_addresses_and_single_outputs(rh, dt):
    for shift in (1, 3):
        job = Merge(rh, np.random.default_rng(shift), 400, 120, 16, dt, scale=-0.7, shift=shift)
        job.check({k: v.get() for k, v in job.run(job.outputs()).items()}, f"shift {shift}")
    for key in ("ddown", "dup"):
        o = {key: job.outputs()[key]}
        job.check({key: job.run(o)[key].get()}, "alone")


def test_in_place_and_host_forms(rh):
    rng = np.random.default_rng(3)
    job = Merge(rh, rng, 700, 120, 16, F32)
    v = job.val
    want = {k: x.get() for k, x in job.run(job.outputs()).items()}
    n, k, rank = job.shape
    rh._check(job.L.ppocr_ra_merge_dev(job.p["w"], job.p["down"], job.p["up"], n, k, rank, job.scale, F32, job.p["w"], None))
    assert np.array_equal(job.dev["w"].numpy().reshape(n, k), want["w"])
    assert np.array_equal(rh.merge_adapter(v["w"], v["down"], v["up"], job.scale), want["w"])
    ddown, dup = rh.merge_adapter_backward(v["dw"], v["down"], v["up"], job.scale)
    assert np.array_equal(ddown, want["ddown"]) and np.array_equal(dup, want["dup"])


def test_gradient_by_differences(rh):
    """The gradients of sum(c * merged) by down and up, against differences of the merged weight in 64 bits."""
    rng = np.random.default_rng(4)
    n, k, rank, s = 20, 12, 3, 1.25
    w, c = rng.standard_normal((n, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    down, up = rng.standard_normal((rank, k)).astype(np.float32), rng.standard_normal((n, rank)).astype(np.float32)
    ddown, dup = rh.merge_adapter_backward(c, down, up, s)

    def value(d, u):
        return (c * (w.astype(np.float64) + s * (u @ d))).sum()

    for got, x, which in ((ddown, down, 0), (dup, up, 1)):
        x = x.astype(np.float64)
        for at in [(0, 0), (x.shape[0] - 1, x.shape[1] - 1), (1, 2)]:
            step = np.zeros_like(x)
            step[at] = 1e-3
            pair = [(down.astype(np.float64) + t * step, up.astype(np.float64)) if which == 0 else
                    (down.astype(np.float64), up.astype(np.float64) + t * step) for t in (1, -1)]
            diff = (value(*pair[0]) - value(*pair[1])) / 2e-3
            assert abs(got[at] - diff) < 1e-4 * (1 + abs(diff))


def test_infinities_and_nan_stay_in_their_rows(rh):
    """A row of dw that holds a NaN: its row of dup, and ddown (which sums over all rows); the rest is as it was."""
    rng = np.random.default_rng(5)
    w, dw = rng.standard_normal((50, 20)).astype(np.float32), rng.standard_normal((50, 20)).astype(np.float32)
    down, up = rng.standard_normal((4, 20)).astype(np.float32), rng.standard_normal((50, 4)).astype(np.float32)
    clean = rh.merge_adapter_backward(dw, down, up)[1]
    dw[7, 3] = np.nan
    ddown, dup = rh.merge_adapter_backward(dw, down, up)
    assert np.isnan(ddown[:, 3]).all() and np.isfinite(np.delete(ddown, 3, axis=1)).all()
    assert np.isnan(dup[7]).all() and np.array_equal(np.delete(dup, 7, axis=0), np.delete(clean, 7, axis=0))
    up[9, 1] = np.inf
    out = rh.merge_adapter(w, down, up)
    assert not np.isfinite(out[9]).any() and np.isfinite(np.delete(out, 9, axis=0)).all()
