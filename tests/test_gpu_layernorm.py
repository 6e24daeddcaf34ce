"""ppocr_layernorm_* against their formulas in 64 bits."""
import ctypes

import numpy as np
import pytest

import train_common as tc
from train_common import BF16, F32, U24

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 120), (120, 120), (33, 80), (17, 7), (100, 128), (65, 129), (40, 512), (21, 513), (9, 1000), (7, 2048),
          (6, 2049), (5, 4096), (3, 8192), (4, 8193), (2, 16384), (5000, 16), (1030, 260)]


def norm64(x, w, b, eps, dy):
    x, w, b, dy = (v.astype(np.float64) for v in (x, w, b, dy))
    mu = x.mean(axis=1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mu) ** 2).mean(axis=1, keepdims=True) + eps)
    h = (x - mu) * rstd
    t = dy * w
    c1, c2 = t.mean(axis=1, keepdims=True), (t * h).mean(axis=1, keepdims=True)
    return {"y": h * w + b, "mean": mu[:, 0], "rstd": rstd[:, 0], "dx": rstd * (t - c1 - h * c2),
            "dw": (dy * h).sum(axis=0), "db": dy.sum(axis=0)}, h, t


def tolerances(x, w, b, dy, ref, h, t, dt):
    """Sums of d (or m) fp32 values are off by at most 8 sqrt(d) half steps of their magnitude, the
    rest a few half steps each; the mean's error moves every h of its row by as much times rstd."""
    d, m = x.shape[1], x.shape[0]
    s = 8 * np.sqrt(float(d)) * U24
    x, w, dy = np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64)), np.abs(dy.astype(np.float64))
    mean = s * x.mean(axis=1) + 2 * U24 * np.abs(ref["mean"])
    emu = (mean + 2 * U24 * x.max(axis=1)) * ref["rstd"]  # in units of h
    rel = s + emu * np.abs(h).mean(axis=1) + emu ** 2 + 8 * U24
    rstd = rel * ref["rstd"]
    eh = emu[:, None] + (rel[:, None] + 4 * U24) * np.abs(h)
    y = eh * w + 4 * U24 * (np.abs(h) * w + np.abs(b))
    c1 = s * np.abs(t).mean(axis=1) + 4 * U24 * np.abs(t).mean(axis=1)
    c2 = (s + 4 * U24) * np.abs(t * h).mean(axis=1) + (np.abs(t) * eh).mean(axis=1)
    a2 = np.abs((t * h).mean(axis=1))
    dx = ref["rstd"][:, None] * ((rel[:, None] + 8 * U24) * (np.abs(t) + np.abs(t).mean(axis=1, keepdims=True) + np.abs(h) * a2[:, None])
                                 + c1[:, None] + np.abs(h) * c2[:, None] + eh * a2[:, None])
    sm = 8 * np.sqrt(float(m)) * U24
    dw = (dy * eh).sum(axis=0) + sm * (dy * np.abs(h)).sum(axis=0)
    db = sm * dy.sum(axis=0)
    half = tc.HALF[dt]
    return {"mean": mean, "rstd": rstd, "y": y + half * (np.abs(ref["y"]) + y), "dx": dx + half * (np.abs(ref["dx"]) + dx),
            "dw": dw + U24 * np.abs(ref["dw"]), "db": db + U24 * np.abs(ref["db"])}


class Job:
    def __init__(self, rh, x, w, b, dy, eps, dt, shift=0):
        self.L, self.rh, self.dt, self.eps = rh._lib.lib(), rh, dt, eps
        self.m, self.d = x.shape
        self.shift = shift
        pad = (lambda v: np.concatenate([np.zeros(shift, v.dtype), v.ravel()])) if shift else (lambda v: v)
        self.x, self.w, self.b, self.dy = (tc.up(pad(v)) for v in (x, w, b, dy))
        self.size = 4 if dt == F32 else 2
        self.ws = tc.Out((self.L.ppocr_layernorm_workspace_bytes(self.m, self.d),), np.uint8)
        self.t = np.float32 if dt == F32 else np.uint16

    def outputs(self):
        return {"y": tc.Out((self.m, self.d), self.t), "mean": tc.Out((self.m,), np.float32),
                "rstd": tc.Out((self.m,), np.float32), "dx": tc.Out((self.m, self.d), self.t),
                "dw": tc.Out((self.d,), np.float32), "db": tc.Out((self.d,), np.float32)}

    def at(self, d, size):
        return ctypes.c_void_p(d.p.value + self.shift * size)

    def forward(self, o, st=None):
        self.rh._check(self.L.ppocr_layernorm_forward_dev(self.at(self.x, self.size), self.at(self.w, 4), self.at(self.b, 4), self.m,
                                                          self.d, self.eps, self.dt, o["y"].p, tc.ptr(o.get("mean")),
                                                          tc.ptr(o.get("rstd")), st))

    def backward(self, o, st=None, ws=True):
        self.rh._check(self.L.ppocr_layernorm_backward_dev(
            self.at(self.dy, self.size), self.at(self.x, self.size), self.at(self.w, 4), o["mean"].p, o["rstd"].p, self.m, self.d, self.dt,
            tc.ptr(o.get("dx")), tc.ptr(o.get("dw")), tc.ptr(o.get("db")), self.ws.p if ws else None,
            self.ws.n if ws else 0, st))

    def step(self):
        from ppocr_rechead.hip import synchronize
        o = self.outputs()
        self.forward(o)
        self.backward(o)
        synchronize()
        self.ws.get()
        return {k: v.get() for k, v in o.items()}


def inputs(rng, m, d, dt):
    x = (rng.standard_normal((m, d)) * (0.5 + 2 * rng.random((m, 1))) + 0.3).astype(np.float32)
    dy = (rng.standard_normal((m, d)) * 0.1).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    b = (0.3 * rng.standard_normal(d)).astype(np.float32)
    return tc.typed(x, dt), tc.typed(dy, dt), w, b


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,d", SHAPES)
def test_layer_norm(rh, m, d, dt):
    rng = np.random.default_rng(m + d)
    (x, xv), (dy, dyv), w, b = inputs(rng, m, d, dt)
    print(f"layernorm m={m} d={d} dt={dt}", flush=True)
    ref, h, t = norm64(xv, w, b, 1e-5, dyv)
    tol = tolerances(xv, w, b, dyv, ref, h, t, dt)
    for shift in (0, 1):  # rows that start on a vector boundary, and not
        got = Job(rh, x, w, b, dy, 1e-5, dt, shift).step()
        for key in ("mean", "rstd", "y", "dx", "dw", "db"):
            tc.close(got[key], ref[key], tol[key], f"{key} shift {shift}")


def test_constant_rows_and_offsets(rh):
    """Rows of one value (variance 0), and rows whose mean is large against their spread."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 120)).astype(np.float32)
    x[::4] = 3.0
    x[1::4] += 1000.0
    dy = rng.standard_normal((40, 120)).astype(np.float32)
    w, b = np.ones(120, np.float32), np.zeros(120, np.float32)
    ref, h, t = norm64(x, w, b, 1e-5, dy)
    tol = tolerances(x, w, b, dy, ref, h, t, F32)
    got = Job(rh, x, w, b, dy, 1e-5, F32).step()
    for key in ("mean", "rstd", "y", "dx", "dw", "db"):
        tc.close(got[key], ref[key], tol[key], key)


def test_differences(rh):
    rng = np.random.default_rng(2)
    m, d = 12, 40
    (x, _), (dy, _), w, b = inputs(rng, m, d, F32)
    got = Job(rh, x, w, b, dy, 1e-5, F32).step()

    def total(dx=0.0, dw=0.0, db=0.0):
        return float((norm64(x + dx, w + dw, b + db, 1e-5, dy)[0]["y"] * dy).sum())

    h = 1e-4
    for key, shape in (("dx", (m, d)), ("dw", (d,)), ("db", (d,))):
        for _ in range(3):
            v = rng.standard_normal(shape)
            v /= np.linalg.norm(v)
            q = (total(**{key: h * v}) - total(**{key: -h * v})) / (2 * h)
            assert abs(q - float((got[key] * v).sum())) < 1e-5, key


@pytest.mark.parametrize("d", [120, 1000, 4096])
def test_in_place_and_parts(rh, d):
    from ppocr_rechead.hip import synchronize
    rng = np.random.default_rng(d)
    (x, _), (dy, _), w, b = inputs(rng, 70, d, F32)
    job = Job(rh, x, w, b, dy, 1e-5, F32)
    want = job.step()
    for keys in (("dx",), ("dw",), ("db",), ("dx", "db")):
        o = job.outputs()
        job.forward(o)
        part = {k: o[k] for k in keys + ("mean", "rstd")}
        job.backward(part)
        synchronize()
        for k in keys:
            assert np.array_equal(part[k].get(), want[k]), (keys, k)
    for over in ("dy", "x"):
        again = Job(rh, x, w, b, dy, 1e-5, F32)
        o = again.outputs()
        again.forward(o)
        o["dx"] = getattr(again, over)
        again.backward(o)
        synchronize()
        assert np.array_equal(o["dx"].numpy(), want["dx"]), over
    again = Job(rh, x, w, b, dy, 1e-5, F32)
    again.forward({"y": again.x})
    synchronize()
    assert np.array_equal(again.x.numpy(), want["y"])


def test_nan_stays_in_its_row(rh):
    rng = np.random.default_rng(5)
    (x, _), (dy, _), w, b = inputs(rng, 50, 120, F32)
    want = Job(rh, x, w, b, dy, 1e-5, F32).step()
    x[7, 3] = np.nan
    got = Job(rh, x, w, b, dy, 1e-5, F32).step()
    rest = np.arange(50) != 7
    assert np.isnan(got["y"][7]).all() and np.isnan(got["dx"][7]).all()
    assert np.array_equal(got["y"][rest], want["y"][rest]) and np.array_equal(got["dx"][rest], want["dx"][rest])
    assert np.array_equal(got["db"], want["db"])


def test_host_forms_and_replayed_graph(rh):
    from ppocr_rechead.hip import H2D, Stream, check, hip, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(6)
    sets = [inputs(rng, 90, 120, F32) for _ in range(3)]
    (x, _), (dy, _), w, b = sets[0]
    job, eager = Job(rh, x, w, b, dy, 1e-5, F32), Job(rh, x, w, b, dy, 1e-5, F32)
    want = job.step()
    y, mean, rstd = rh.layer_norm(x, w, b, 1e-5)
    dx, dw, db = rh.layer_norm_backward(dy, x, w, mean, rstd)
    for got, key in ((y, "y"), (mean, "mean"), (rstd, "rstd"), (dx, "dx"), (dw, "dw"), (db, "db")):
        assert np.array_equal(got, want[key]), key
    st, o = Stream(), job.outputs()

    def call():
        job.forward(o, st.h)
        job.backward(o, st.h, ws=True)

    g = _Graph(st, call)
    for which in (1, 2, 0, 1):
        (x, _), (dy, _), w, b = sets[which]
        for j in (job, eager):
            for dd, v in ((j.x, x), (j.dy, dy), (j.w, w), (j.b, b)):
                check(hip().hipMemcpy(dd.p, v.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(v.nbytes), H2D), "hipMemcpy")
        g.replay()
        want = eager.step()
        synchronize()
        for key, v in o.items():
            assert np.array_equal(v.get(), want[key]), (which, key)
    g.close()
