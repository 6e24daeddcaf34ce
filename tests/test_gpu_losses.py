"""The losses over the vocabulary, ppocr_xent_* and ppocr_distill_*, against their formulas in 64
bits, and what the calls promise: rows without a target, masked classes, streams, graphs, equal
bits, memory behind the outputs."""
import ctypes

import numpy as np
import pytest

import train_common as tc
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (1, 5, 3), (2, 33, 8), (33, 100, 33), (31, 32, 32), (32, 129, 64), (65, 257, 80), (120, 1000, 97),
          (130, 131, 120), (257, 300, 128), (40, 640, 160), (70, 517, 192), (50, 385, 200), (129, 700, 256),
          (300, 6906, 80), (45, 18710, 120)]


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_cross_entropy(rh, m, n, k, dt):
    rng = np.random.default_rng(m * 7 + n + k)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    other = rng.integers(0, n, m).astype(np.int32)
    target = np.where(rng.random(m) < 0.2, other, to).astype(np.int32)
    if m > 4:
        target[rng.integers(0, m, max(1, m // 10))] = -1
    grad = (rng.standard_normal(m) * np.exp(rng.standard_normal(m))).astype(np.float32)
    tc.check_step(rh, a, w, b, dt, "xent", target=target, grad=grad)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,tn,tau", [(1, 4, 3, 1, 1.0), (33, 100, 33, 2, 2.0), (65, 257, 80, 7, 0.5),
                                          (130, 131, 120, 64, 4.0), (64, 6906, 80, 32, 1.5), (40, 18710, 120, 16, 2.0),
                                          (50, 385, 200, 33, 1.0), (33, 700, 256, 5, 3.0)])
def test_distillation(rh, m, n, k, tn, tau, dt):
    rng = np.random.default_rng(m * 5 + n + tn)
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    idx, z = tc.teacher_inputs(rng, m, n, tn, to)
    idx[rng.random((m, tn)) < 0.1] = -1
    z[rng.random((m, tn)) < 0.05] = -np.inf
    if tn > 2:
        idx[::3, 1] = idx[::3, 0]  # the same class twice
        idx[1::4, tn - 1] = idx[1::4, 1]
    if m > 3:
        idx[2] = -1  # no teacher at all
        z[3] = -np.inf
    grad = (rng.random(m) * tau * tau).astype(np.float32)
    got, ref = tc.check_step(rh, a, w, b, dt, "distill", idx=idx, z=z, tau=tau, grad=grad)
    if m > 3:
        assert (got["loss"][2:4] == 0).all() and (tc.values(got["da"])[2:4] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_no_bias_and_no_grad(rh, dt):
    rng = np.random.default_rng(3)
    a, w, _, to = tc.head_inputs(rng, 70, 333, 120)
    tc.check_step(rh, a, w, None, dt, "no bias, grad 1", target=to)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_rows_without_label_may_hold_anything(rh, dt):
    """NaN and infinities in rows that have no label, or no gradient, reach no gradient."""
    rng = np.random.default_rng(4)
    a, w, b, to = tc.head_inputs(rng, 100, 500, 120)
    target = to.copy()
    target[[3, 40, 41, 99]] = -1
    target[50] = 500  # not a class: no label in the device form
    grad = rng.random(100).astype(np.float32)
    grad[60] = 0.0
    a[3], a[40, 5], a[99, 0], a[60, 7], a[50] = np.nan, np.inf, -np.inf, np.nan, np.nan
    ar, av = tc.typed(a, dt)
    wr, wv = tc.typed(w, dt)
    got = tc.Loss(rh, ar, wr, b, dt, target, grad=grad).step()
    keep = np.ones(100, bool)
    keep[[3, 40, 99, 60, 50]] = False
    clean = np.where(keep[:, None], av, 0.0).astype(np.float32)
    ci, q, logq, some = tc.teacher64(100, 500, target)
    ref, zz, p, dz, s, al = tc.loss64(clean, wv, b, ci, q, logq, some, 1.0, grad)
    tol = tc.loss_tol(clean, wv, b, zz, p, dz, s, al, ref, dt, 1.0, q, logq)
    assert (got["loss"][[3, 40, 99, 50]] == 0).all() and np.isnan(got["loss"][60])
    tc.close(got["loss"][keep], ref["loss"][keep], tol["loss"][keep], "loss")
    tc.close(got["lse"][keep], ref["lse"][keep], tol["lse"][keep], "lse")
    for key in ("da", "dw", "db"):
        tc.close(got[key], ref[key], tol[key], key)
    assert (tc.values(got["da"])[[3, 40, 41, 99, 60, 50]] == 0).all()


def test_no_row_has_a_label(rh):
    rng = np.random.default_rng(5)
    a, w, b, _ = tc.head_inputs(rng, 77, 300, 80)
    got = tc.Loss(rh, a, w, b, F32, np.full(77, -1, np.int32)).step()
    for key in ("loss", "da", "dw", "db"):
        assert (got[key] == 0).all(), key


@pytest.mark.parametrize("low", [-np.inf, -3.4e38, -1e9])
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_masked_classes(rh, low, dt):
    """A vocabulary masked by its bias: those classes have probability 0 and no gradient, among them
    whole records of 32 and all but one class; a masked label's loss is as large as its mask."""
    rng = np.random.default_rng(6)
    a, w, b, to = tc.head_inputs(rng, 90, 400, 120)
    b[40:200] = low
    b[::7] = low
    target = np.where(np.isin(to, np.nonzero(b < -1e8)[0]), 1, to).astype(np.int32)
    tc.check_step(rh, a, w, b, dt, f"masked {low}", target=target)
    b[:] = low
    b[133] = 0.5
    tc.check_step(rh, a, w, b, dt, f"one class left {low}", target=np.full(90, 133, np.int32))
    target = np.full(90, 5, np.int32)
    got = tc.Loss(rh, *(tc.typed(x, dt)[0] for x in (a, w)), b, dt, target).step()
    assert (got["loss"] >= -low * 0.999).all()
    assert np.isfinite(tc.values(got["dw"])).all() and np.isfinite(tc.values(got["da"])).all()
    assert np.abs(got["db"][5] + 90).max() < 1e-3


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_magnitudes(rh, dt):
    """Rows and classes whose magnitudes lie far apart: each group of 32 has its own scale."""
    rng = np.random.default_rng(7)
    a, w, b, to = tc.head_inputs(rng, 160, 320, 96)
    a[:32] *= 1e-6
    a[32:64] *= 1e3
    a[64:96] = 0.0
    w[64:96] *= 1e-5
    w[96:128] *= 30.0
    w[200:240] = 0.0
    grad = np.where(np.arange(160) % 3 == 0, 1e-7, 1.0).astype(np.float32)
    tc.check_step(rh, a, w, b, dt, "magnitudes", target=to, grad=grad)
    tc.check_step(rh, a * np.float32(1e-20), w, b, dt, "tiny activations", target=to, grad=grad)
    tc.check_step(rh, a * np.float32(1e18), w * np.float32(1e-18), b, dt, "large times small", target=to, grad=grad * np.float32(1e10))


@pytest.mark.parametrize("size", [1e30, 1e-28, 1e-31])
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_gradients_of_any_size(rh, dt, size):
    """Loss scales far from 1, next to rows whose gradient is 2^-14 of theirs."""
    rng = np.random.default_rng(17)
    a, w, b, to = tc.head_inputs(rng, 100, 300, 64)
    grad = (rng.standard_normal(100) * size).astype(np.float32)
    grad[::5] *= np.float32(2.0 ** -14)
    tc.check_step(rh, a, w, b, dt, f"grad {size}", target=to, grad=grad)
    a[32:64] *= np.float32(1e-24)
    tc.check_step(rh, a, w, b, dt, f"grad {size}, a group of tiny rows", target=to, grad=grad)


def test_a_head_that_holds_nan(rh):
    """NaN in a class's weights: every logit sum is NaN, but rows without label or gradient keep 0."""
    rng = np.random.default_rng(18)
    a, w, b, to = tc.head_inputs(rng, 64, 200, 32)
    w[17, 3] = np.nan
    target = np.where(np.arange(64) % 3 == 0, -1, to).astype(np.int32)
    got = tc.Loss(rh, a, w, b, F32, target).step()
    assert (got["loss"][::3] == 0).all() and (got["da"][::3] == 0).all()
    assert np.isnan(got["loss"][1::3]).all() and np.isnan(got["da"][1::3]).all()


@pytest.mark.parametrize("logit", [20.0, 9.0])
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_nearly_certain_labels_keep_their_small_gradient(rh, dt, logit):
    """p(label) close to 1: p - 1 must not be the difference of rounded values.  Every row's gradient
    is right to 1%, but for what 32 bits hold of p: z and lse are about `logit`, each off by two half
    steps of that and their difference as much again, so p - 1 by up to 6 2^-24 logit, times the
    class's weights.  At 20 that is as large as the gradient itself (p - 1 is about 4e-7), at 9 (p - 1
    is about 0.02) a 5000th of it."""
    rng = np.random.default_rng(8)
    w = (rng.standard_normal((200, 64)) * 0.3).astype(np.float32)
    to = rng.integers(0, 200, 64).astype(np.int32)
    a = (w[to] / (w[to] ** 2).sum(axis=1, keepdims=True) * logit).astype(np.float32)
    got, ref = tc.check_step(rh, a, w, None, dt, f"certain {logit}", target=to)
    rows = np.linalg.norm(ref["da"], axis=1)
    err = np.linalg.norm(tc.values(got["da"]) - ref["da"], axis=1)
    assert (err <= 0.01 * rows + 6 * tc.U24 * logit * np.linalg.norm(w, axis=1).max()).all()


def test_gradient_against_differences(rh):
    """The gradients against central differences of the loss in 64 bits, along random directions:
    the difference quotient is off by h^2 / 6 of the third derivative, 2e-8 here."""
    rng = np.random.default_rng(9)
    m, n, k = 20, 90, 24
    a, w, b, to = tc.head_inputs(rng, m, n, k)
    grad = rng.standard_normal(m).astype(np.float32)
    idx, z = tc.teacher_inputs(rng, m, n, 5, to)
    for kind in ({"target": to}, {"idx": idx, "z": z, "tau": 2.0}):
        got = tc.Loss(rh, a, w, b, F32, grad=grad, **kind).step()
        ci, q, logq, some = tc.teacher64(m, n, **kind)

        def total(da, dw, db):
            r, *_ = tc.loss64(a + da, w + dw, b + db, ci, q, logq, some, kind.get("tau", 1.0))
            return float((r["loss"] * grad).sum())

        h = 1e-4
        for which, shape in (("da", (m, k)), ("dw", (n, k)), ("db", (n,))):
            for _ in range(3):
                v = rng.standard_normal(shape)
                v /= np.linalg.norm(v)
                d = {"da": 0.0, "dw": 0.0, "db": 0.0}
                plus = total(**{**d, which: h * v})
                minus = total(**{**d, which: -h * v})
                assert abs((plus - minus) / (2 * h) - float((got[which] * v).sum())) < 1e-5, (kind.keys(), which)


def test_outputs_that_are_not_asked_for(rh):
    from ppocr_rechead.hip import synchronize
    rng = np.random.default_rng(10)
    a, w, b, to = tc.head_inputs(rng, 70, 400, 120)
    job = tc.Loss(rh, a, w, b, F32, to)
    want = job.step()
    for keys in (("da",), ("dw",), ("db",), ("da", "db"), ("dw", "db"), ()):
        o = job.outputs()
        job.forward(o)
        part = {k: v for k, v in o.items() if k in keys or k in ("loss", "lse")}
        job.backward(part)
        synchronize()
        for k in keys:
            assert np.array_equal(part[k].get(), want[k]), (keys, k)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_equal_calls_give_equal_bits(rh, dt):
    """On any stream, with a workspace of its own or the call's, whatever the workspace held."""
    from ppocr_rechead.hip import Stream, synchronize
    rng = np.random.default_rng(11)
    a, w, b, to = tc.head_inputs(rng, 300, 2000, 120)
    idx, z = tc.teacher_inputs(rng, 300, 2000, 9, to)
    for kind in ({"target": to}, {"idx": idx, "z": z, "tau": 2.0}):
        job = tc.Loss(rh, tc.typed(a, dt)[0], tc.typed(w, dt)[0], b, dt, **kind)
        want = job.step()
        st = Stream()
        for fill, ws in ((0xFF, True), (0x7B, True), (0, False)):
            o = job.outputs()
            job.ws.d.fill_bytes(fill)
            synchronize()
            job.forward(o, st.h, ws)
            job.backward(o, st.h, ws)
            st.synchronize()
            for k, v in o.items():
                assert np.array_equal(v.get().view(np.uint8), want[k].view(np.uint8)), (k, fill, ws)
            job.ws.d.fill_bytes(0xA5)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_unaligned_tensors(rh, dt):
    """Tensors that start one value past a vector boundary: the same bits."""
    from ppocr_rechead.hip import synchronize
    rng = np.random.default_rng(19)
    a, w, b, to = tc.head_inputs(rng, 90, 300, 120)
    idx, z = tc.teacher_inputs(rng, 90, 300, 5, to)
    size = 4 if dt == F32 else 2
    for kind in ({"target": to}, {"idx": idx, "z": z, "tau": 2.0}):
        job = tc.Loss(rh, tc.typed(a, dt)[0], tc.typed(w, dt)[0], b, dt, **kind)
        want = job.step()
        o = job.outputs()
        held = []

        class At:
            def __init__(self, d):
                self.p = ctypes.c_void_p(d.p.value + size)

        def past(x):
            d = tc.up(np.concatenate([np.zeros(1, x.dtype), x.ravel()]))
            held.append(d)
            return At(d)

        job.a, job.w = past(tc.typed(a, dt)[0]), past(tc.typed(w, dt)[0])
        wide = {k: tc.Out((v.shape[0] * v.shape[1] + 1,), v.dtype) for k, v in o.items() if k in ("da", "dw")}
        job.forward(o)
        job.backward(dict(o, **{k: At(v) for k, v in wide.items()}))
        synchronize()
        for k, v in want.items():
            got = wide[k].get()[1:].reshape(v.shape) if k in wide else o[k].get()
            assert np.array_equal(got.view(np.uint8), v.view(np.uint8)), (kind.keys(), k)


def test_replayed_graph(rh):
    """A captured step on inputs that change between replays, with eager work in between."""
    from ppocr_rechead.hip import H2D, Stream, check, hip, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(12)
    m, n, k = 200, 1500, 120
    sets = [tc.head_inputs(rng, m, n, k) for _ in range(3)]
    job = tc.Loss(rh, sets[0][0], sets[0][1], sets[0][2], F32, sets[0][3])
    eager = tc.Loss(rh, sets[0][0], sets[0][1], sets[0][2], F32, sets[0][3])
    st = Stream()
    o = job.outputs()

    def put(j, s):
        for d, x in ((j.a, s[0]), (j.w, s[1]), (j.bias, s[2]), (j.target, s[3])):
            check(hip().hipMemcpy(d.p, x.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(x.nbytes), H2D), "hipMemcpy")

    def call():
        job.forward(o, st.h)
        job.backward(o, st.h)

    call()
    st.synchronize()
    g = _Graph(st, call)
    for turn, which in enumerate((1, 0, 2, 2, 1)):
        put(job, sets[which])
        put(eager, sets[which])
        g.replay()
        want = eager.step()
        synchronize()
        for key, v in o.items():
            assert np.array_equal(v.get().view(np.uint8), want[key].view(np.uint8)), (turn, key)
    g.close()


def test_two_calls_at_once(rh):
    """Two problems on two streams, each with its own workspace."""
    from ppocr_rechead.hip import Stream
    rng = np.random.default_rng(13)
    jobs = []
    for m, n in ((400, 3000), (150, 5000)):
        a, w, b, to = tc.head_inputs(rng, m, n, 120)
        jobs.append(tc.Loss(rh, a, w, b, F32, to))
    want = [j.step() for j in jobs]
    streams = [Stream() for _ in jobs]
    outs = [j.outputs() for j in jobs]
    for _ in range(3):
        for j, o, st in zip(jobs, outs, streams):
            j.forward(o, st.h)
            j.backward(o, st.h)
    for st in streams:
        st.synchronize()
    for o, w_ in zip(outs, want):
        for key, v in o.items():
            assert np.array_equal(v.get(), w_[key]), key


def test_host_forms_equal_the_device_forms(rh):
    rng = np.random.default_rng(14)
    a, w, b, to = tc.head_inputs(rng, 60, 700, 120)
    to[5] = -1
    grad = rng.random(60).astype(np.float32)
    want = tc.Loss(rh, a, w, b, F32, to, grad=grad).step()
    loss, lse = rh.cross_entropy(a, w, b, to)
    da, dw, db = rh.cross_entropy_backward(a, w, b, to, lse, grad)
    for got, key in ((loss, "loss"), (lse, "lse"), (da, "da"), (dw, "dw"), (db, "db")):
        assert np.array_equal(got, want[key]), key
    idx, z = tc.teacher_inputs(rng, 60, 700, 6, np.maximum(to, 0))
    want = tc.Loss(rh, a, w, b, F32, idx=idx, z=z, tau=2.0).step()
    loss, lse = rh.distill(a, w, b, idx, z, 2.0)
    da, dw, db = rh.distill_backward(a, w, b, idx, z, 2.0, lse)
    for got, key in ((loss, "loss"), (lse, "lse"), (da, "da"), (dw, "dw"), (db, "db")):
        assert np.array_equal(got, want[key]), key


def test_a_workspace_shared_with_the_head(rh):
    """One workspace in turn for a guarded decode of the head and for a loss: the decode's list
    header survives."""
    from ppocr_rechead.hip import DeviceArray, synchronize
    rng = np.random.default_rng(15)
    a, w, b, to = tc.head_inputs(rng, 120, 1000, 120)
    head = rh.RecHead(qw=rh.QuantizedWeight.from_f32_transposed(w), bias=b)
    big = (rng.standard_normal((120, 120)) * 40).astype(np.float32)
    job = tc.Loss(rh, a, w, b, F32, to)
    ws = DeviceArray((max(job.bytes(), head.workspace_bytes(120, 2)) + 256,), np.uint8)
    ws.fill_bytes(0)
    job.ws.d = ws
    want = head.argmax(big, 2)
    dbig, di, dm = tc.up(big), DeviceArray((120,), np.int32), DeviceArray((120,), np.float32)
    o = job.outputs()
    for _ in range(3):
        job.forward(o)
        job.backward(o)
        rh._check(job.L.ppocr_rh_argmax_dev(head.handle, dbig.p, 120, 2, di.p, dm.p, ws.p, ws.nbytes, None))
        synchronize()
        assert np.array_equal(di.numpy(), want[0]) and np.array_equal(dm.numpy(), want[1])
    head.close()


def test_allocation_failure(rh, monkeypatch):
    """Without a workspace and without memory: PPOCR_ERR_NO_MEMORY from every entry point that
    allocates, outputs untouched, and the next call works."""
    from ppocr_rechead.hip import synchronize
    rng = np.random.default_rng(20)
    a, w, b, to = tc.head_inputs(rng, 50, 200, 40)
    idx, z = tc.teacher_inputs(rng, 50, 200, 3, to)
    for kind, op in (({"target": to}, "SoftmaxCrossEntropy"), ({"idx": idx, "z": z}, "Distill")):
        job = tc.Loss(rh, a, w, b, F32, **kind)
        o = job.outputs()
        monkeypatch.setenv("PPOCR_RECHEAD_FAULT", "alloc")
        for call in (job.forward, job.backward):
            with pytest.raises(rh.OcrError) as e:
                call(o, None, False)
            assert e.value.code == rh.PPOCR_ERR_NO_MEMORY and e.value.op == op
        monkeypatch.delenv("PPOCR_RECHEAD_FAULT")
        synchronize()
        for v in o.values():
            assert (v.get().view(np.uint8) == 0xA5).all()
        job.forward(o, None, False)
        job.backward(o, None, False)
        synchronize()
        want = job.step()
        for k, v in o.items():
            assert np.array_equal(v.get(), want[k]), k
