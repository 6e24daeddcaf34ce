"""The training entry points together, as a program uses them on one stream without a wait between them:
a fine-tuning step of the final LayerNorm and the head, and a student head taught by the top
logits of a resident teacher head."""
import ctypes

import numpy as np
import pytest

import train_common as tc
from test_gpu_layernorm import norm64
from train_common import F32

pytestmark = pytest.mark.gpu


def test_fine_tuning_step(rh):
    """LayerNorm -> cross entropy and back: the gradients of the whole chain against the chain in 64
    bits, and two steps of gradient descent that run on the updated weights."""
    from ppocr_rechead.hip import D2H, DeviceArray, Stream, check, hip
    rng = np.random.default_rng(1)
    m, n, d, eps = 200, 900, 120, 1e-5
    x = (rng.standard_normal((m, d)) * 2 + 0.5).astype(np.float32)
    g = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    c = (0.3 * rng.standard_normal(d)).astype(np.float32)
    w = (rng.standard_normal((n, d)) * 0.2).astype(np.float32)
    b = (rng.standard_normal(n) * 0.01).astype(np.float32)
    target = rng.integers(0, n, m).astype(np.int32)
    target[::9] = -1
    grad = np.full(m, 1.0 / (target >= 0).sum(), np.float32)
    L, st = rh._lib.lib(), Stream()
    dev = {k: tc.up(v) for k, v in dict(x=x, g=g, c=c, w=w, b=b, t=target, grad=grad).items()}
    out = {k: DeviceArray(s, np.float32) for k, s in dict(y=(m, d), mean=(m,), rstd=(m,), loss=(m,), lse=(m,), dy=(m, d), dw=(n, d),
                                                          db=(n,), dx=(m, d), dg=(d,), dc=(d,)).items()}
    size = max(L.ppocr_xent_workspace_bytes(m, n, d, 0), L.ppocr_layernorm_workspace_bytes(m, d))
    ws = DeviceArray((size,), np.uint8)  # one for all of them in turn
    p = {k: v.p for k, v in {**dev, **out}.items()}

    def step():
        rh._check(L.ppocr_layernorm_forward_dev(p["x"], p["g"], p["c"], m, d, eps, 0, p["y"], p["mean"], p["rstd"], st.h))
        rh._check(L.ppocr_xent_forward_dev(p["y"], p["w"], p["b"], p["t"], m, n, d, 0, p["loss"], p["lse"], ws.p, size, st.h))
        rh._check(L.ppocr_xent_backward_dev(p["y"], p["w"], p["b"], p["t"], p["lse"], p["grad"], m, n, d, 0, p["dy"], p["dw"],
                                            p["db"], ws.p, size, st.h))
        rh._check(L.ppocr_layernorm_backward_dev(p["dy"], p["x"], p["g"], p["mean"], p["rstd"], m, d, 0, p["dx"], p["dg"],
                                                 p["dc"], ws.p, size, st.h))

    for _ in range(2):
        step()
        st.synchronize()
        got = {k: v.numpy() for k, v in out.items()}
        ref, *_ = norm64(x, g, c, eps, np.zeros((m, d)))
        ci, q, lq, some = tc.teacher64(m, n, target)
        r, *_ = tc.loss64(ref["y"], w, b, ci, q, lq, some, 1.0, grad)
        back, *_ = norm64(x, g, c, eps, r["da"])
        for key, want in (("loss", r["loss"]), ("dw", r["dw"]), ("db", r["db"]), ("dx", back["dx"]), ("dg", back["dw"]),
                          ("dc", back["db"])):
            # every stage's own error is below 4e-6 of its output's norm (their tests); four stages
            err = np.linalg.norm(got[key] - want) / np.linalg.norm(want)
            print(f"  {key}: {err:.1e} of the norm", flush=True)
            assert err < 2e-5, key
        w, b, g, c = (v - 0.5 * got[k] for v, k in ((w, "dw"), (b, "db"), (g, "dg"), (c, "dc")))
        for k, v in (("w", w), ("b", b), ("g", g), ("c", c)):
            check(hip().hipMemcpy(dev[k].p, v.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(v.nbytes), 1), "hipMemcpy")


def test_student_of_a_resident_teacher(rh):
    """The teacher's logits (ppocr_rh_logits_dev), their top 16 (ppocr_topk_rows_dev), the student's loss
    and gradients (ppocr_distill_*), nothing leaving the GPU; a student equal to its teacher that
    sees all of the teacher's classes has loss and gradients of rounding size."""
    from ppocr_rechead.hip import DeviceArray, Stream
    rng = np.random.default_rng(2)
    m, n, k, top, tau = 150, 800, 120, 16, 2.0
    a, wt, bt, _ = tc.head_inputs(rng, m, n, k)
    ws_ = (wt + rng.standard_normal((n, k)) * 0.01).astype(np.float32)
    teacher = rh.RecHead(w_t=wt, bias=bt)
    L, st = rh._lib.lib(), Stream()
    da_, logits = tc.up(a), DeviceArray((m, n), np.float32)
    idx, val = DeviceArray((m, top), np.int32), DeviceArray((m, top), np.float32)
    job = tc.Loss(rh, a, ws_, bt, F32, idx=np.zeros((m, top), np.int32), z=np.zeros((m, top), np.float32), tau=tau)
    job.idx, job.z = idx, val
    o = job.outputs()
    rh._check(L.ppocr_rh_logits_dev(teacher.handle, da_.p, m, rh.MODE_AUTO, logits.p, None, 0, st.h))
    rh._check(L.ppocr_topk_rows_dev(logits.p, m, n, top, idx.p, val.p, st.h))
    job.forward(o, st.h)
    job.backward(o, st.h)
    st.synchronize()
    ti, tz = idx.numpy(), val.numpy()
    assert np.array_equal(ti, np.argsort(-logits.numpy(), axis=1, kind="stable")[:, :top])
    ci, q, lq, some = tc.teacher64(m, n, idx=ti, z=tz, tau=tau)
    ref, z, p, dz, s, al = tc.loss64(a, ws_, bt, ci, q, lq, some, tau)
    tol = tc.loss_tol(a, ws_, bt, z, p, dz, s, al, ref, F32, tau, q, lq)
    for key in ("loss", "lse", "da", "dw", "db"):
        tc.close(o[key].get(), ref[key], tol[key], key)
    teacher.close()
    # the teacher's own head, all classes known (64 of them)
    a, w, b, _ = tc.head_inputs(rng, 40, 64, 80)
    full = (a.astype(np.float64) @ w.T + b).astype(np.float32)
    every = np.broadcast_to(np.arange(64, dtype=np.int32), (40, 64)).copy()
    got = tc.Loss(rh, a, w, b, F32, idx=every, z=full, tau=1.5).step()
    assert np.abs(got["loss"]).max() < 1e-5
    for key in ("da", "dw", "db"):
        assert np.abs(got[key]).max() < 1e-4, key
