"""Helpers of the losses' tests at magnitudes that lie far apart: the 64-bit formulas with tolerances that
are measured against each output row's own largest contribution."""
import numpy as np

import train_common as tc
from train_common import F32


def targets(kind, rng, m, n, to):
    """Labels, or a teacher's entries, as the arguments of the helpers."""
    if kind == "xent":
        return {"target": to.copy()}
    idx, z = tc.teacher_inputs(rng, m, n, 5, to)
    return {"idx": idx, "z": z, "tau": 2.0}


def without_target(kind, rows):
    key = "target" if "target" in kind else "idx"
    kind[key][rows] = -1


def reference(av, wv, b, kind, grad):
    ci, q, logq, some = tc.teacher64(av.shape[0], wv.shape[0], **kind)
    ref, z, p, dz, s, al = tc.loss64(av, wv, b, ci, q, logq, some, kind.get("tau", 1.0), grad)
    return ref, z, p, dz, s, al, q, logq


def owner_tol(a, w, z, p, dz, s, al, ref, dt, tau):
    """What the gradients may be off by where magnitudes lie far apart.  As tc.loss_tol says, but what
    the fp16 halves of P cannot hold is measured against the largest contribution to the same row
    of da or dw, not against the largest operand of the whole call: P is held to 2^-25 where the
    largest contribution is 2^4 or more, and times operands of at most 2^15 where that contribution's
    own is 2^14 or more, but for the 2^4 that entries of one group may share a scale over: 2^-24 of the
    largest contribution for each entry."""
    k, n, m = a.shape[1], w.shape[0], a.shape[0]
    aw, aa = np.abs(w.astype(np.float64)), np.abs(al)
    size = np.abs(np.where(p > 0, z, 0.0)) + np.abs(ref["lse"])[:, None]
    ez = (aa @ aw.T) / tau * (3 * 2.0 ** -22 + 8 * np.sqrt(3.0 * k) * tc.U24) + 8 * tc.U24 * (size + 1.0)
    lse = np.where(p > 0, ez, 0.0).max(axis=1) + 8 * np.sqrt(n) * tc.U24 + 8 * tc.U24 * (1 + np.abs(ref["lse"]))
    one = 2.0 ** -22 if dt == F32 else 2.0 ** -11
    rel = ez + lse[:, None] + 8 * tc.U24
    e = np.where(p > 0, p * (rel + one), 0.0) * np.abs(s)[:, None] + (one + 8 * tc.U24) * np.abs(dz)
    adz = np.abs(dz) + e
    share = 2.0 ** -24

    def prod(x, ex, y, terms, most):
        return ex @ y + (x @ y) * (3 * 2.0 ** -22 + 8 * np.sqrt(3.0 * terms) * tc.U24) + terms * share * most[:, None]

    da = prod(adz, e, aw, n, (adz * aw.max(axis=1)[None]).max(axis=1))
    dw = prod(adz.T, e.T, aa, m, (adz * aa.max(axis=1)[:, None]).max(axis=0))
    db = (np.where(p > 0, p * rel, 0.0) * np.abs(s)[:, None] + 8 * tc.U24 * np.abs(dz)).sum(axis=0) \
        + adz.sum(axis=0) * 8 * np.sqrt(float(m)) * tc.U24 + 2.0 ** -120
    return {"da": da + tc.HALF[dt] * (np.abs(ref["da"]) + da) + tc.LEAST[dt],
            "dw": dw + tc.HALF[dt] * (np.abs(ref["dw"]) + dw) + tc.LEAST[dt], "db": db}


def run(rh, a, w, b, dt, kind, grad=None):
    ar, av = tc.typed(a, dt)
    wr, wv = tc.typed(w, dt)
    got = tc.Loss(rh, ar, wr, b, dt, kind.get("target"), kind.get("idx"), kind.get("z"), kind.get("tau", 1.0), grad).step()
    return {k: tc.values(v) for k, v in got.items()}, av, wv


def compare(rh, a, w, b, dt, kind, grad, rows, classes, label):
    """A step against the formulas at the given rows (loss, lse, da) and classes (dw, db)."""
    print(f"{label}: m={a.shape[0]} n={w.shape[0]} k={a.shape[1]} {'f32' if dt == F32 else 'bf16'}", flush=True)
    got, av, wv = run(rh, a, w, b, dt, kind, grad)
    tau = kind.get("tau", 1.0)
    ref, z, p, dz, s, al, q, logq = reference(av, wv, b, kind, grad)
    tol = tc.loss_tol(av, wv, b, z, p, dz, s, al, ref, dt, tau, q, logq)
    tol.update(owner_tol(av, wv, z, p, dz, s, al, ref, dt, tau))
    for key, at in (("loss", rows), ("lse", rows), ("da", rows), ("dw", classes), ("db", classes)):
        tc.close(got[key][at], ref[key][at], tol[key][at], f"{label} {key}")
    for key in ("da", "dw", "db"):
        assert np.isfinite(got[key]).all(), key
    return got, ref
