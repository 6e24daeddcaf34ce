"""Shared helpers of the tests of adapted heads and of the losses over lines: inputs, the formulas in 64
bits and the tolerances that follow from the arithmetic."""
import ctypes

import numpy as np

import train_common as tc
from train_common import F32, HALF, LEAST, U24


def ctypes_ptr(a):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


# ---------------------------------------------------------------- adapters beside the head
class Head:
    """A head, its weights in 64 bits and `slots` adapters beside it."""

    def __init__(self, rh, rng, n, k, quant, slots, max_rank, ranks=None, dt=F32, up_scale=0.05):
        self.rh, self.n, self.k, self.slots = rh, n, k, slots
        w = (rng.standard_normal((n, k)) * 0.05).astype(np.float32)
        self.bias = (rng.standard_normal(n) * 0.01).astype(np.float32)
        if quant:
            qw = rh.QuantizedWeight.from_f32_transposed(w)
            self.base = rh.RecHead(qw=qw, bias=self.bias)
            self.w = qw.data.astype(np.float64) * qw.scales.astype(np.float64)[:, None]
        else:
            self.base = rh.RecHead(w_t=w, bias=self.bias)
            self.w = w.astype(np.float64)
        self.quant = quant
        self.head = rh.AdaptedHead(self.base, slots, max_rank)
        self.max_rank = max_rank
        self.adapters = [None] * slots
        ranks = [max_rank] * slots if ranks is None else ranks
        for s, r in enumerate(ranks):
            if r:
                self.set(s, (rng.standard_normal((r, k)) / np.sqrt(k)).astype(np.float32),
                         (rng.standard_normal((n, r)) * up_scale).astype(np.float32), float(0.5 + rng.random()), dt)

    def set(self, slot, down, up, scale, dt=F32):
        from ppocr_rechead.hip import synchronize
        scale = float(np.float32(scale))
        if dt == F32:
            self.head.set_adapter(slot, down, up, scale)
        else:
            (dr, down), (ur, up) = tc.typed(down, dt), tc.typed(up, dt)
            dd, du = tc.up(dr), tc.up(ur)
            self.rh._check(self.rh._lib.lib().ppocr_ra_set_dev(self.head.handle, slot, dd.p, du.p, down.shape[0], scale, dt, None))
            synchronize()
        self.adapters[slot] = (down.astype(np.float64), up.astype(np.float64), scale)

    def rows_of(self, m, off, slot):
        """The slot of each row (-1: none)."""
        out = np.full(m, -1)
        for i in range(len(off) - 1):
            s = int(slot[i])
            out[off[i]:off[i + 1]] = s if 0 <= s < self.slots and self.adapters[s] is not None else -1
        return out

    def exact(self, a, rows):
        """Logits in 64 bits and how far 32-bit ones may be off.

        Each row is held in two fp16 halves of 11 bits: at most 2^-22 of each value is lost (halves below
        the normal numbers lose 2^-25 of a row scaled to 2^14, which is less); fp16 halves of a weight that is
        not int8 lose 2^-22 as well, and the product of the low halves, 2^-22, is left out.  The terms of all
        products are added in fp32, at most as many roundings as there are terms (2 k or 3 k of the head's, 3
        rank of the adapter's), each of at most 2^-24 of the terms' magnitude.  u = down a: halves of both, 3 k
        terms, its own halves and power of two.  up over its class's scale, times scale: two roundings; its halves.
        The row's power of two is exact; scale and bias two roundings more."""
        a64 = a.astype(np.float64)
        z = a64 @ self.w.T + self.bias.astype(np.float64)
        mag = np.abs(a64) @ np.abs(self.w).T
        extra = np.zeros_like(z)
        inner = np.zeros_like(z)
        for s in set(rows.tolist()) - {-1}:
            at = rows == s
            down, up, scale = self.adapters[s]
            u = a64[at] @ down.T
            z[at] += scale * (u @ up.T)
            extra[at] = abs(scale) * (np.abs(u) @ np.abs(up).T)
            inner[at] = abs(scale) * ((np.abs(a64[at]) @ np.abs(down).T) @ np.abs(up).T)
        # ranks are padded to 16, 32 or 64; terms of zeros round nothing
        terms = (2 if self.quant else 3) * self.k + 3 * self.max_rank
        e = mag * (terms * U24 + (1 if self.quant else 3) * 2.0 ** -22)
        e += extra * (terms * U24 + 3 * 2.0 ** -22 + 4 * U24) + inner * (3 * self.k * U24 + 3 * 2.0 ** -22 + 4 * U24)
        return z, e + 4 * U24 * (np.abs(z) + np.abs(self.bias) + mag)


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


class Call:
    """The device form of a call on an adapted head, its outputs guarded."""

    def __init__(self, h, a, off, slot, m=None):
        self.h, self.L = h, h.rh._lib.lib()
        self.m, self.lines = a.shape[0] if m is None else m, len(off) - 1
        self.a, self.off, self.slot = tc.up(a), tc.up(np.asarray(off, np.int64)), tc.up(np.asarray(slot, np.int32))
        self.bytes = self.L.ppocr_ra_workspace_bytes(h.head.handle, self.m)
        self.ws = tc.Out((max(self.bytes, 16),), np.uint8)

    def logits(self, stream=None, ws=True, out=None):
        out = tc.Out((self.m, self.h.n), np.float32) if out is None else out
        self.h.rh._check(self.L.ppocr_ra_logits_dev(self.h.head.handle, self.a.p, self.m, self.off.p, self.lines, self.slot.p,
                                                    out.p, self.ws.p if ws else None, self.bytes if ws else 0, stream))
        return out

    def outputs(self):
        return {"idx": tc.Out((self.m,), np.int32), "maxprob": tc.Out((self.m,), np.float32), "seq": tc.Out((self.m,), np.int32),
                "len": tc.Out((self.lines,), np.int64), "score": tc.Out((self.lines,), np.float32)}

    def decode(self, stream=None, ws=True, o=None):
        o = self.outputs() if o is None else o
        self.h.rh._check(self.L.ppocr_ra_decode_dev(self.h.head.handle, self.a.p, self.m, self.off.p, self.lines, self.slot.p,
                                                    o["idx"].p, o["maxprob"].p, o["seq"].p, o["len"].p, o["score"].p,
                                                    self.ws.p if ws else None, self.bytes if ws else 0, stream))
        return o


def collapse(idx, maxprob, off):
    """Greedy collapse of each line (blank 0)."""
    seqs, scores = [], []
    for i in range(len(off) - 1):
        last, out, total = 0, [], []
        for r in range(off[i], off[i + 1]):
            if idx[r] != 0 and idx[r] != last:
                out.append(int(idx[r]))
                total.append(float(maxprob[r]))
            last = idx[r]
        seqs.append(out)
        scores.append(sum(total) / len(total) if total else 0.0)
    return seqs, scores


# ---------------------------------------------------------------- losses over lines
def line_of(off, m):
    """The line of each of m steps, -1 for none."""
    out = np.full(m, -1)
    for i in range(len(off) - 1):
        out[off[i]:off[i + 1]] = i
    return out


def policy64(loss, old, ref, target, adv, per_row, off, low, high, beta, grad=None):
    """The policy loss and its gradients in 64 bits, and how far 32-bit ones may be off.

    rho: the difference of the logarithms is rounded (2^-24 of it, a relative error of rho), the exponential is
    within 2 half steps, the product with A 1.  The divergence of t: t is rounded as well; below 1 its series has
    13 roundings of falling weight (within 8 half steps of the result), above it is a difference of terms each
    within 3.  Means: sums of 64 bits, one rounding."""
    m, lines = loss.shape[0], len(off) - 1
    line = line_of(off, m)
    on = (line >= 0) & ((target >= 0) if target is not None else True)
    x, o = (np.where(on, v, 0.0).astype(np.float64) for v in (loss, old))
    adv64 = adv.astype(np.float64)
    a = adv64 if per_row else np.where(line >= 0, adv64[np.maximum(line, 0)] if lines else 0.0, 0.0)
    a = np.where(on, a, 0.0)
    low, high, beta = (float(np.float32(v)) for v in (low, high, beta))
    far = o - x
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        rho = np.exp(far)
        cut = ((a > 0) & (far > np.log1p(high))) | ((a < 0) & (far < np.log1p(-low)))
        held = np.where(cut, np.where(a > 0, 1 + high, 1 - low), rho)
        value = np.where(a == 0, 0.0, -held * a)
        slope = np.where(cut | (a == 0), 0.0, rho * a)
        erho = (np.abs(far) + 4) * U24
        ev, es = np.where(a == 0, 0.0, np.abs(value) * np.where(cut, 3 * U24, erho)), np.abs(slope) * erho
        kl, ekl = np.zeros(m), np.zeros(m)
        if ref is not None:
            t = x - np.where(on, ref, 0.0).astype(np.float64)
            em1 = np.expm1(t)
            # the series of e^t - t - 1, 64-bit differences being of no use near 0
            kl = np.where(np.abs(t) < 1e-3, t * t * (0.5 + t / 6 + t * t / 24), em1 - t)
            et = np.abs(t) * U24
            ekl = np.abs(em1) * et + np.where(np.abs(t) < 1, 8 * U24 * kl, 3 * U24 * (np.abs(em1) + np.abs(t)))
            ev = ev + abs(beta) * (ekl + 2 * U24 * kl) + U24 * np.abs(value)
            es = es + abs(beta) * (np.exp(t) * et + 4 * U24 * np.abs(em1)) + U24 * np.abs(slope)
            value, slope = value + beta * kl, slope + beta * em1
    out = {k: np.zeros(lines) for k in ("loss", "kl", "clipped")}
    tol = {k: np.zeros(lines) for k in ("loss", "kl", "clipped")}
    row, erow = np.zeros(m), np.zeros(m)
    for i in range(lines):
        at = (line == i) & on
        c = max(int(at.sum()), 1)
        g = 1.0 if grad is None else float(grad[i])
        for key, v, e in (("loss", value, ev), ("kl", kl, ekl), ("clipped", cut.astype(float), np.zeros(m))):
            out[key][i] = v[at].sum() / c
            tol[key][i] = e[at].sum() / c + 2 * U24 * abs(out[key][i])
        if g != 0.0:
            row[at] = g / c * slope[at]
            erow[at] = abs(g) / c * es[at] + 3 * U24 * np.abs(row[at])
    out["row_grad"], tol["row_grad"] = row, erow
    return out, {k: v + LEAST[F32] for k, v in tol.items()}


def preference64(loss, ref, target, off, beta, smoothing, average, grad=None):
    """The preference loss and its gradients in 64 bits, and how far 32-bit ones may be off: sums and the
    difference of the rewards in 64 bits; the logistic function and its logarithm from an exponential within 4
    half steps, some half steps each; products."""
    m, lines = loss.shape[0], len(off) - 1
    line = line_of(off, m)
    on = (line >= 0) & ((target >= 0) if target is not None else True)
    beta, eps = float(np.float32(beta)), float(np.float32(smoothing))
    gain = (0.0 if ref is None else np.where(on, ref, 0.0).astype(np.float64)) - np.where(on, loss, 0.0).astype(np.float64)
    reward, w = np.zeros(lines), np.zeros(lines)
    for i in range(lines):
        at = (line == i) & on
        w[i] = beta / max(int(at.sum()), 1) if average else beta
        reward[i] = w[i] * gain[at].sum()
    h = reward[0::2] - reward[1::2]
    up, down = np.logaddexp(0.0, -h), np.logaddexp(0.0, h)  # -log s(h), -log s(-h)
    out = {"loss": (1 - eps) * up + eps * down, "reward": reward}
    s, s_ = np.exp(-up), np.exp(-down)  # s(h), s(-h)
    g = np.ones(lines // 2) if grad is None else grad.astype(np.float64)
    slope = eps * s - (1 - eps) * s_
    eslope = 12 * U24 * (eps * s + (1 - eps) * s_)
    row, erow = np.zeros(m), np.zeros(m)
    for i in range(lines):
        at, p = (line == i) & on, i // 2
        sign = -1.0 if i % 2 == 0 else 1.0
        if g[p] != 0.0:
            row[at] = sign * g[p] * slope[p] * w[i]
            erow[at] = abs(g[p] * w[i]) * eslope[p] + 4 * U24 * np.abs(row[at])
    out["row_grad"] = row
    size = np.repeat(np.abs(reward[0::2]) + np.abs(reward[1::2]), 2) if lines else reward
    tol = {"loss": 12 * U24 * ((1 - eps) * up + eps * down), "reward": U24 * (np.abs(reward) + 2.0 ** -20 * size), "row_grad": erow}
    return out, {k: v + LEAST[F32] for k, v in tol.items()}


# ---------------------------------------------------------------- merged adapters
def merge64(w, dw, down, up, scale, dt):
    """The merged weight and the adapter's gradients in 64 bits; products summed in fp32, at most one rounding a
    term of the terms' magnitude, then the rounding of the stored value."""
    scale = float(np.float32(scale))
    w, dw, down, up = (v.astype(np.float64) for v in (w, dw, down, up))
    n, k, rank = w.shape[0], w.shape[1], down.shape[0]
    out = {"w": w + scale * (up @ down), "ddown": scale * (up.T @ dw), "dup": scale * (dw @ down.T)}
    mag = {"w": np.abs(up) @ np.abs(down), "ddown": np.abs(up).T @ np.abs(dw), "dup": np.abs(dw) @ np.abs(down).T}
    terms = {"w": rank + 2, "ddown": n + 2, "dup": k + 2}
    tol = {}
    for key in out:
        e = abs(scale) * mag[key] * terms[key] * U24 + 2 * U24 * np.abs(out[key])
        tol[key] = e + HALF[dt] * (np.abs(out[key]) + e) + LEAST[dt]
    return out, tol
