"""Shared helpers of the training operators' tests: bf16 arrays, device calls through the C ABI
with guarded outputs, the 64-bit formulas and the tolerances that follow from the arithmetic."""
import ctypes

import numpy as np

F32, BF16 = 0, 1
U24 = 2.0 ** -24  # half a step of fp32, relative
HALF = {F32: U24, BF16: 2.0 ** -8}  # largest rounding of a stored value, relative
LEAST = {F32: 2.0 ** -150, BF16: 2.0 ** -134}  # and absolute: below 2^-126 the steps are 2^-149 and 2^-133


def to_bf16(x):
    """Bits of x rounded to bf16 (nearest even)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + (0x7FFF + ((u >> 16) & 1))) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def typed(x, dt):
    """x as the array a call takes for type dt, and the values it holds."""
    if dt == F32:
        x = np.ascontiguousarray(x, np.float32)
        return x, x
    u = to_bf16(np.asarray(x, np.float32))
    return u, from_bf16(u)


def values(x):
    return from_bf16(x) if x.dtype == np.uint16 else x


class Out:
    """A device output followed by memory that a call must leave as it was."""
    TAIL = 256

    def __init__(self, shape, dtype):
        from ppocr_rechead.hip import DeviceArray
        self.shape, self.dtype = shape, np.dtype(dtype)
        self.n = int(np.prod(shape, dtype=np.int64)) * self.dtype.itemsize
        self.d = DeviceArray((self.n + self.TAIL,), np.uint8)
        self.d.fill_bytes(0xA5)

    @property
    def p(self):
        return self.d.p

    def get(self):
        b = self.d.numpy()
        assert (b[self.n:] == 0xA5).all(), "memory behind an output was written"
        return b[:self.n].view(self.dtype).reshape(self.shape)


def up(x):
    from ppocr_rechead.hip import DeviceArray
    return None if x is None else DeviceArray.from_numpy(x)


def ptr(d):
    return None if d is None else d.p


class Loss:
    """A head, its rows and their targets on the device; calls of the losses on them."""

    def __init__(self, rh, a, w, bias, dt, target=None, idx=None, z=None, tau=1.0, grad=None):
        self.rh, self.L, self.dt, self.tau = rh, rh._lib.lib(), dt, float(tau)
        self.m, self.k = a.shape
        self.n = w.shape[0]
        self.xent = target is not None
        self.tn = 1 if self.xent else idx.shape[1]
        self.a, self.w, self.bias = up(a), up(w), up(bias)
        self.target, self.idx, self.z, self.grad = up(target), up(idx), up(z), up(grad)
        self.tdt = np.float32 if dt == F32 else np.uint16
        self.ws = Out((self.bytes(),), np.uint8)

    def bytes(self):
        if self.xent:
            return self.L.ppocr_xent_workspace_bytes(self.m, self.n, self.k, self.dt)
        return self.L.ppocr_distill_workspace_bytes(self.m, self.n, self.k, self.tn, self.dt)

    def outputs(self):
        return {"loss": Out((self.m,), np.float32), "lse": Out((self.m,), np.float32),
                "da": Out((self.m, self.k), self.tdt), "dw": Out((self.n, self.k), self.tdt),
                "db": Out((self.n,), np.float32)}

    def _teacher(self):
        if self.xent:
            return (self.target.p,)
        return (self.idx.p, self.z.p, self.tn, self.tau)

    def forward(self, o, stream=None, ws=True):
        f = self.L.ppocr_xent_forward_dev if self.xent else self.L.ppocr_distill_forward_dev
        self.rh._check(f(self.a.p, self.w.p, ptr(self.bias), *self._teacher(), self.m, self.n, self.k, self.dt,
                         o["loss"].p, o["lse"].p, self.ws.p if ws else None, self.ws.n if ws else 0, stream))

    def backward(self, o, stream=None, ws=True):
        f = self.L.ppocr_xent_backward_dev if self.xent else self.L.ppocr_distill_backward_dev
        self.rh._check(f(self.a.p, self.w.p, ptr(self.bias), *self._teacher(), o["lse"].p, ptr(self.grad), self.m,
                         self.n, self.k, self.dt, ptr(o.get("da")), ptr(o.get("dw")), ptr(o.get("db")),
                         self.ws.p if ws else None, self.ws.n if ws else 0, stream))

    def step(self):
        from ppocr_rechead.hip import synchronize
        o = self.outputs()
        self.forward(o)
        self.backward(o)
        synchronize()
        self.ws.get()
        return {k: v.get() for k, v in o.items()}


# ---------------------------------------------------------------- the formulas in 64 bits
def teacher64(m, n, target=None, idx=None, z=None, tau=1.0):
    """Target distributions: class, weight and log weight per entry (weight 0: absent), and which
    rows have one."""
    if target is not None:
        there = ((target >= 0) & (target < n))[:, None]
        return np.where(there, target[:, None], 0), there.astype(np.float64), np.zeros((m, 1)), there[:, 0]
    t = np.where((idx >= 0) & (idx < n), z.astype(np.float64) / tau, -np.inf)
    top = t.max(axis=1, keepdims=True)
    some = top[:, 0] > -np.inf
    e = np.exp(t - np.where(some[:, None], top, 0.0))
    q = np.where(some[:, None], e / np.where(some, e.sum(axis=1), 1.0)[:, None], 0.0)
    with np.errstate(divide="ignore"):
        return np.where(q > 0, idx, 0), q, np.where(q > 0, np.log(np.where(q > 0, q, 1.0)), 0.0), some


def loss64(a, w, bias, idx, q, logq, some, tau=1.0, grad=None):
    """loss, lse and the gradients; rows without a target or gradient add nothing."""
    a64, w64 = a.astype(np.float64), w.astype(np.float64)
    m, n = a.shape[0], w.shape[0]
    with np.errstate(invalid="ignore", over="ignore"):
        z = (a64 @ w64.T + (0.0 if bias is None else bias.astype(np.float64))) / tau
        top = z.max(axis=1, keepdims=True)
        lse = top[:, 0] + np.log(np.exp(z - top).sum(axis=1))
        zt = np.take_along_axis(z, idx, axis=1)
        terms = np.where(q > 0, q * (logq - np.where(q > 0, zt, 0.0) + lse[:, None]), 0.0)
        p = np.exp(z - lse[:, None])
    loss = np.where(some, terms.sum(axis=1), 0.0)
    s = np.where(some, 1.0 if grad is None else grad.astype(np.float64), 0.0) / tau
    live = s != 0
    dz = np.where(live[:, None], p, 0.0)
    y = np.zeros_like(dz)
    np.add.at(y, (np.arange(m)[:, None], idx), q)
    dz = (dz - np.where(live[:, None], y, 0.0)) * s[:, None]
    al = np.where(live[:, None], a64, 0.0)
    return {"loss": loss, "lse": lse, "da": dz @ w64, "dw": dz.T @ al, "db": dz.sum(axis=0)}, z, p, dz, s, al


def loss_tol(a, w, bias, z, p, dz, s, al, ref, dt, tau, q, logq):
    """How far the outputs may be off.  Logits: operands held to 22 bits (fp32; bf16 exact), the
    product of the low halves left out (2^-22 each) and 3 k sums in fp32 (8 sqrt(3 k) half steps of
    the terms' magnitude), the bias, the scale and the difference to lse some half steps of their
    own.  p then is off by as much, relatively, and by the roundings of exp and of its fp16 halves
    (2^-22; one half with bf16 tensors, 2^-11: fp16 holds 11 bits, steps of
    2^-10 above a power of two, a rounding takes half of one), which also p - q takes.  Products and sums as for
    the logits, then the rounding of the stored value."""
    k, n, m = a.shape[1], w.shape[0], a.shape[0]
    mag = (np.abs(np.where(np.isfinite(a), a, 0.0)).astype(np.float64) @ np.abs(w.astype(np.float64)).T) / tau
    size = np.abs(np.where(p > 0, z, 0.0)) + np.abs(np.where(np.isfinite(ref["lse"]), ref["lse"], 0.0))[:, None]
    ez = mag * (3 * 2.0 ** -22 + 8 * np.sqrt(3.0 * k) * U24) + 8 * U24 * (size + 1.0)
    worst = np.where(p > 0, ez, 0.0).max(axis=1)
    lse = worst + 8 * np.sqrt(n) * U24 + 8 * U24 * (1 + np.abs(np.where(np.isfinite(ref["lse"]), ref["lse"], 0)))
    tn = q.shape[1]
    loss = lse + worst + (8 + tn) * U24 * (np.abs(ref["loss"]) + np.abs(q * logq).sum(axis=1) + size.max(axis=1))
    one = 2.0 ** -22 if dt == F32 else 2.0 ** -11
    rel = ez + lse[:, None] + 8 * U24
    e = np.where(p > 0, p * (rel + one), 0.0) * np.abs(s)[:, None] + (one + 8 * U24) * np.abs(dz)
    adz = np.abs(dz) + e
    aw, aa = np.abs(w.astype(np.float64)), np.abs(al)
    tiny = 2.0 ** -37  # values of P below the last place of an fp16 subnormal, against the largest operand
    smax = np.abs(s).max(initial=0.0)
    def prod(x, ex, y, terms, floor):
        return ex @ y + (x @ y) * (3 * 2.0 ** -22 + 8 * np.sqrt(3.0 * terms) * U24) + floor
    da = prod(adz, e, aw, n, n * aw.max(initial=0.0) * tiny * np.abs(s)[:, None])
    dw = prod(adz.T, e.T, aa, m, m * aa.max(initial=0.0) * tiny * smax)
    db = (np.where(p > 0, p * rel, 0.0) * np.abs(s)[:, None] + 8 * U24 * np.abs(dz)).sum(axis=0) \
        + adz.sum(axis=0) * 8 * np.sqrt(float(m)) * U24 + m * tiny * smax
    return {"loss": loss, "lse": lse, "da": da + HALF[dt] * (np.abs(ref["da"]) + da) + LEAST[dt],
            "dw": dw + HALF[dt] * (np.abs(ref["dw"]) + dw) + LEAST[dt], "db": db + LEAST[F32]}


def close(got, want, tol, label):
    got = values(got).astype(np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - want))
    bad = ~(off <= tol)
    worst = float(np.max(np.where(same, 0.0, off / np.maximum(tol, 1e-300)), initial=0.0))
    print(f"  [{label}] worst error / tolerance {worst:.3f}", flush=True)
    assert not bad.any(), f"{label}: {int(bad.sum())} of {bad.size} beyond the tolerance, worst {worst:.2f} x, " \
                          f"first at {np.argwhere(bad)[0]}: {got[tuple(np.argwhere(bad)[0])]} for " \
                          f"{np.broadcast_to(want, got.shape)[tuple(np.argwhere(bad)[0])]}"


def check_step(rh, a, w, bias, dt, label, target=None, idx=None, z=None, tau=1.0, grad=None):
    """One forward and backward pass against the formulas."""
    ar, av = typed(a, dt)
    wr, wv = typed(w, dt)
    print(f"{label}: m={a.shape[0]} n={w.shape[0]} k={a.shape[1]} {'f32' if dt == F32 else 'bf16'}", flush=True)
    got = Loss(rh, ar, wr, bias, dt, target, idx, z, tau, grad).step()
    ci, q, logq, some = teacher64(a.shape[0], w.shape[0], target, idx, z, tau)
    ref, zz, p, dz, s, al = loss64(av, wv, bias, ci, q, logq, some, tau, grad)
    tol = loss_tol(av, wv, bias, zz, p, dz, s, al, ref, dt, tau, q, logq)
    for key in ("loss", "lse", "da", "dw", "db"):
        close(got[key], ref[key], tol[key], f"{label} {key}")
    return got, ref


def head_inputs(rng, m, n, k, scale=1.0):
    """Rows that lean towards a class each, weights and biases as the head's workloads have them."""
    w = (rng.standard_normal((n, k)) * 0.05).astype(np.float32)
    b = (rng.standard_normal(n) * 0.01).astype(np.float32)
    to = rng.integers(0, n, m)
    d = w[to] / np.maximum(np.linalg.norm(w[to], axis=1, keepdims=True), 1e-2)
    lean = np.log(n + 1.0) * (0.4 + 0.9 * rng.random((m, 1))) / np.maximum(np.linalg.norm(w[to], axis=1, keepdims=True), 1e-2)
    a = (rng.standard_normal((m, k)) * 0.5 + lean * d) * scale
    return a.astype(np.float32), w, b, to.astype(np.int32)


def teacher_inputs(rng, m, n, tn, to):
    idx = rng.integers(0, n, (m, tn)).astype(np.int32)
    idx[:, 0] = to
    z = (rng.standard_normal((m, tn)) * 1.5 + 2.0).astype(np.float32)
    return idx, z
