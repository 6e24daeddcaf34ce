"""The global norm of many gradients and their clipping against the formula in 64 bits."""
import ctypes

import numpy as np
import pytest

import train_common as tc
from train_common import BF16, F32, HALF, LEAST, U24

pytestmark = pytest.mark.gpu


class Clip:
    def __init__(self, rh, tensors, shift=0):
        """tensors: (values, type); shift: their first element lies that many elements behind an allocation's start."""
        self.rh, self.L = rh, rh._lib.lib()
        self.dts = [dt for _, dt in tensors]
        self.val = []
        self.dev, self.src = [], []
        for x, dt in tensors:
            raw, v = tc.typed(np.asarray(x, np.float32), dt)
            self.val.append(v)
            d = tc.up(np.concatenate([np.zeros(shift, raw.dtype), raw]))
            self.dev.append(d)
            self.src.append(d.p.value + shift * raw.itemsize)
        self.count = len(tensors)
        self.sizes = (ctypes.c_int64 * self.count)(*[v.size for v in self.val])
        self.types = (ctypes.c_int32 * self.count)(*self.dts)
        self.bytes = self.L.ppocr_grad_clip_workspace_bytes(self.sizes, self.count)
        self.ws = tc.Out((self.bytes,), np.uint8)

    def run(self, most, out=None, stream=None, ws=True, in_place=False, norm=None):
        if out is None and not in_place:
            out = [tc.Out(v.shape, np.float32 if dt == F32 else np.uint16) for v, dt in zip(self.val, self.dts)]
        norm = tc.Out((1,), np.float32) if norm is None else norm
        P = ctypes.c_void_p * self.count
        self.rh._check(self.L.ppocr_grad_clip_dev(P(*self.src), None if in_place else P(*[o.p.value for o in out]), self.sizes, self.types,
                                                  self.count, most, norm.p, self.ws.p if ws else None, self.bytes if ws else 0, stream))
        return out, norm

    def expect(self, most):
        total = sum(float((v.astype(np.float64) ** 2).sum()) for v in self.val)
        norm = np.sqrt(total)
        scale = most / norm if norm > most else 1.0
        want = [v.astype(np.float64) * scale for v in self.val]
        # the factor and the product are rounded, then the stored value; unscaled gradients are copied
        tol = [np.abs(w) * 3 * U24 + HALF[dt] * np.abs(w) * (1 + 3 * U24) + LEAST[dt] for w, dt in zip(want, self.dts)]
        return want, tol, norm

    def check(self, got, norm, most, label):
        want, tol, n64 = self.expect(most)
        assert abs(norm - n64) <= 2 * U24 * n64, label
        for i, (g, w, t) in enumerate(zip(got, want, tol)):
            tc.close(g, w, t, f"{label} {i}")


def tensors(rng, sizes, kinds=(F32, BF16), scale=0.01):
    return [(rng.standard_normal(n) * scale, kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


SIZES = [[1], [0], [], [5, 0, 7], [4096, 8192, 4097, 8191], [100000, 3, 16384], [1920, 299360, 18710, 120, 120],
         [17] * 130, [1000] * 119 + [0] + [9000] * 125, [3000001]]


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}-{sum(s)}" for s in SIZES])
def test_clip(rh, sizes, shift):
    print(sizes[:5], shift, flush=True)
    rng = np.random.default_rng(len(sizes))
    job = Clip(rh, tensors(rng, sizes), shift)
    size = np.sqrt(sum(float((v.astype(np.float64) ** 2).sum()) for v in job.val))
    for most in (0.37 * size + 1e-9, 10 * size + 1):
        out, norm = job.run(most)
        got = [o.get() for o in out]
        job.ws.get()
        job.check(got, norm.get()[0], most, f"clip {most:.3g}")
        if most > size:
            for g, d, s in zip(got, job.dev, job.sizes):
                assert np.array_equal(g, d.numpy()[shift:])
        again, n2 = job.run(most, ws=False)
        assert n2.get()[0] == norm.get()[0] and all(np.array_equal(a.get(), g) for a, g in zip(again, got))
    # in place
    most = 0.37 * size + 1e-9
    want = [o.get() for o in job.run(most)[0]]
    job.run(most, in_place=True)
    for w, d in zip(want, job.dev):
        back = d.numpy()
        assert np.array_equal(back[shift:], w) and (back[:shift] == 0).all()


def test_norms_beyond_32_bits_of_squares(rh):
    """Gradients whose squares vanish or overflow in 32 bits."""
    rng = np.random.default_rng(2)
    for scale in (1e-30, 1e-38, 1e25, 1e37):
        job = Clip(rh, tensors(rng, [500, 3000], scale=scale))
        for most in (scale, scale * 1e-6, 1e30):
            out, norm = job.run(most)
            n = norm.get()[0]
            want, tol, n64 = job.expect(float(np.float32(most)))
            if n64 < 3.4e38:
                assert abs(n - n64) <= 2 * U24 * n64 + LEAST[F32]
            else:
                assert n == np.inf
            for o, w, t in zip(out, want, tol):
                # a factor below the normal numbers has an absolute error of 2^-150
                tc.close(o.get(), w, t + np.abs(w).max() / max(min(1.0, most / n64), 1e-300) * 2.0 ** -149, f"{scale} {most}")


def test_not_finite(rh):
    """A NaN or infinity: the norm shows it and the gradients stay."""
    for bad in (np.nan, np.inf, -np.inf):
        x = np.linspace(-1, 1, 5000).astype(np.float32)
        x[4999] = bad
        job = Clip(rh, [(x, F32), (np.ones(10), BF16)])
        out, norm = job.run(0.5)
        assert not np.isfinite(norm.get()[0])
        assert np.array_equal(out[0].get(), x, equal_nan=True) and (tc.values(out[1].get()) == 1).all()
        job.run(0.5, in_place=True)
        assert np.array_equal(job.dev[0].numpy(), x, equal_nan=True)
    job = Clip(rh, [(np.full(100, 2.0), F32)])
    out, norm = job.run(np.inf)  # the norm alone
    assert norm.get()[0] == 20.0 and (out[0].get() == 2).all()


def test_captured_with_its_own_tables(rh):
    """Two calls of different tensors captured into graphs, replayed in turn on new values."""
    from ppocr_rechead.hip import H2D, Stream, check, hip, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(4)
    jobs = [Clip(rh, tensors(rng, [5000, 70, 123])), Clip(rh, tensors(rng, [9] * 140))]
    st = Stream()
    synchronize()
    runs = []
    for job in jobs:
        held = {}
        def call(job=job, held=held):
            held["out"], held["norm"] = job.run(0.05, out=held["o"], stream=st.h, norm=held["n"])
        held["n"] = tc.Out((1,), np.float32)
        held["o"] = [tc.Out(v.shape, np.float32 if dt == F32 else np.uint16) for v, dt in zip(job.val, job.dts)]
        runs.append((job, held, _Graph(st, call)))
    for turn in range(3):
        for job, held, graph in runs:
            for i, dt in enumerate(job.dts):
                raw, job.val[i] = tc.typed((rng.standard_normal(job.val[i].size) * (turn + 0.01)).astype(np.float32), dt)
                check(hip().hipMemcpy(ctypes.c_void_p(job.src[i]), raw.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(raw.nbytes), H2D), "hipMemcpy")
            synchronize()
            graph.replay()
            job.check([o.get() for o in held["out"]], held["norm"].get()[0], float(np.float32(0.05)), f"replay {turn}")
    for *_, graph in runs:
        graph.close()


def test_host_form(rh):
    rng = np.random.default_rng(5)
    g = [rng.standard_normal((30, 7)).astype(np.float32), rng.standard_normal(0).astype(np.float32),
         rng.standard_normal(2000000).astype(np.float32)]
    out, norm = rh.clip_gradients(g, 3.0)
    n64 = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in g))
    assert abs(norm - n64) <= 2 * U24 * n64
    for o, x in zip(out, g):
        assert o.shape == x.shape
        tc.close(o, x * (3.0 / n64), np.abs(x) * (3.0 / n64) * 4 * U24 + LEAST[F32], "host")
    assert rh.clip_gradients([], 1.0) == ([], 0.0)
    # in place: no table of outputs
    h = g[0].copy()
    L = rh._lib.lib()
    rh._check(L.ppocr_grad_clip((ctypes.c_void_p * 1)(h.ctypes.data), None, (ctypes.c_int64 * 1)(h.size), 1, 1e-3, None))
    assert abs(np.linalg.norm(h.astype(np.float64)) - 1e-3) < 1e-8
