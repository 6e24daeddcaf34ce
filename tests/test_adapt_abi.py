"""What the entry points that adapt a head refuse, and what they take without work, before any HIP call: no
device is needed.  Every refusal names its operator."""
import ctypes

import numpy as np
import pytest

P = ctypes.c_void_p(1 << 20)  # never read: each call is refused, or has nothing to do
MIS = ctypes.c_void_p((1 << 20) + 4)
NAN, INF = float("nan"), float("inf")


def refused(rh, rc, op):
    assert rc == rh.PPOCR_ERR_INVALID_ARG
    assert rh._lib.last_error().startswith(op + ": "), rh._lib.last_error()


def test_adapted_heads_refuse_null_handles(rh):
    L = rh._lib.lib()
    out = ctypes.c_void_p(5)
    refused(rh, L.ppocr_ra_create(None, 1, 1, ctypes.byref(out)), "LowRankAdapter")
    assert out.value is None
    refused(rh, L.ppocr_ra_create(P, 1, 1, None), "LowRankAdapter")
    refused(rh, L.ppocr_ra_shape(None, None, None), "LowRankAdapter")
    refused(rh, L.ppocr_ra_set(None, 0, P, P, 1, 1.0), "LowRankAdapter")
    refused(rh, L.ppocr_ra_set_dev(None, 0, P, P, 1, 1.0, 0, None), "LowRankAdapter")
    refused(rh, L.ppocr_ra_logits(None, P, P, 1, P, P), "LowRankAdapter")
    refused(rh, L.ppocr_ra_logits_dev(None, P, 1, P, 1, P, P, P, 1 << 30, None), "LowRankAdapter")
    refused(rh, L.ppocr_ra_decode(None, P, P, 1, P, P, P, P, P, P), "LowRankAdapter")
    refused(rh, L.ppocr_ra_decode_dev(None, P, 1, P, 1, P, P, P, P, P, P, P, 1 << 30, None), "LowRankAdapter")
    assert L.ppocr_ra_workspace_bytes(None, 5) == 0
    L.ppocr_ra_destroy(None)


def test_merge_refuses(rh):
    L = rh._lib.lib()

    def forward(w=P, down=P, up=P, n=5, k=8, r=2, s=1.0, dt=0, out=P):
        return L.ppocr_ra_merge_dev(w, down, up, n, k, r, s, dt, out, None)

    def backward(w=P, down=P, up=P, n=5, k=8, r=2, s=1.0, dt=0, out=P, ws=P, size=1 << 30):
        return L.ppocr_ra_merge_backward_dev(w, down, up, n, k, r, s, dt, out, P, ws, size, None)

    for kw in (dict(n=0), dict(n=-1), dict(k=0), dict(k=-1), dict(k=257), dict(n=(1 << 24) + 1), dict(r=0), dict(r=65), dict(r=-1),
               dict(s=NAN), dict(s=INF), dict(dt=2), dict(w=None), dict(down=None), dict(up=None)):
        refused(rh, forward(**kw), "LowRankAdapter")
        refused(rh, backward(**kw), "LowRankAdapter")
    refused(rh, forward(out=None), "LowRankAdapter")
    refused(rh, backward(ws=MIS), "LowRankAdapter")
    refused(rh, backward(size=16), "LowRankAdapter")
    assert L.ppocr_ra_merge_backward_dev(None, None, None, 5, 8, 2, 1.0, 0, None, None, None, 0, None) == rh.PPOCR_OK
    assert L.ppocr_ra_merge_workspace_bytes(0, 8, 2) == 0 and L.ppocr_ra_merge_workspace_bytes(5, 8, 65) == 0
    assert L.ppocr_ra_merge_workspace_bytes(18710, 120, 16) > 0
    a = np.ones((5, 8), np.float32)
    for call in (lambda: rh.merge_adapter(a, np.ones((2, 7)), np.ones((5, 2))), lambda: rh.merge_adapter(a, np.ones((2, 8)), np.ones((4, 2))),
                 lambda: rh.merge_adapter(a[0], np.ones((2, 8)), np.ones((5, 2))), lambda: rh.merge_adapter(a, np.ones((0, 8)), np.ones((5, 0))),
                 lambda: rh.merge_adapter_backward(a, np.ones((2, 8)), np.ones((5, 3))),
                 lambda: rh.merge_adapter(a, np.ones((2, 8)), np.ones((5, 2)), INF)):
        with pytest.raises(rh.OcrError):
            call()


def test_policy_refuses(rh):
    L = rh._lib.lib()

    def call(loss=P, old=P, adv=P, off=P, lines=2, m=4, low=0.2, high=0.2, beta=0.1):
        return L.ppocr_policy_loss_dev(loss, old, None, None, adv, 0, off, lines, m, low, high, beta, None, P, P, P, P, None)

    for kw in (dict(lines=-1), dict(m=-1), dict(lines=(1 << 30) + 1), dict(m=(1 << 30) + 1), dict(low=-0.1), dict(low=1.1), dict(low=NAN),
               dict(high=-0.1), dict(high=NAN), dict(beta=NAN), dict(beta=INF), dict(loss=None), dict(old=None), dict(adv=None), dict(off=None)):
        refused(rh, call(**kw), "PolicyLoss")
    x = np.ones(4, np.float32)
    for f in (lambda: rh.policy_loss(x, x[:3], x[:2], [0, 2, 4]), lambda: rh.policy_loss(x, x, x[:3], [0, 2, 4]),
              lambda: rh.policy_loss(x, x, x[:2], [0, 2, 5]), lambda: rh.policy_loss(x, x, x[:2], [1, 2, 4]),
              lambda: rh.policy_loss(x, x, x[:2], [0, 3, 2]), lambda: rh.policy_loss(x, x, x[:2], [0, 2, 4], np.zeros(3)),
              lambda: rh.policy_loss(x, x, x[:2], [0, 2, 4], None, x[:1]), lambda: rh.policy_loss(x, x, x[:2], [0, 2, 4], clip_low=2.0),
              lambda: rh.policy_loss(x[None], x, x[:2], [0, 2, 4]), lambda: rh.policy_loss(x, x, x[:2], [0, 2, 4], grad=x[:3])):
        with pytest.raises(rh.OcrError):
            f()


def test_preference_refuses(rh):
    L = rh._lib.lib()

    def call(loss=P, off=P, pairs=2, m=4, beta=0.1, smoothing=0.0):
        return L.ppocr_preference_loss_dev(loss, None, None, off, pairs, m, beta, smoothing, 0, None, P, P, P, None)

    for kw in (dict(pairs=-1), dict(pairs=1 << 62), dict(m=-1), dict(pairs=(1 << 29) + 1), dict(m=(1 << 30) + 1), dict(beta=NAN), dict(beta=INF), dict(smoothing=-0.1),
               dict(smoothing=1.1), dict(smoothing=NAN), dict(loss=None), dict(off=None)):
        refused(rh, call(**kw), "PreferenceLoss")
    x = np.ones(4, np.float32)
    for f in (lambda: rh.preference_loss(x, x, [0, 2]), lambda: rh.preference_loss(x, x[:3], [0, 2, 4]),
              lambda: rh.preference_loss(x, x, [0, 2, 5]), lambda: rh.preference_loss(x, x, [0, 3, 2]),
              lambda: rh.preference_loss(x, x, [0, 2, 4], smoothing=-1.0), lambda: rh.preference_loss(x, x, [0, 2, 4], grad=x)):
        with pytest.raises(rh.OcrError):
            f()


def test_clip_refuses(rh):
    L = rh._lib.lib()

    def call(g=(1 << 20, 1 << 21), o=None, n=(10, 10), dt=(0, 0), count=2, most=1.0, ws=P, size=1 << 30):
        V, I, T = ctypes.c_void_p * 2, ctypes.c_int64 * 2, ctypes.c_int32 * 2
        return L.ppocr_grad_clip_dev(None if g is None else V(*g), None if o is None else V(*o), None if n is None else I(*n),
                                     None if dt is None else T(*dt), count, most, P, ws, size, None)

    a, b = 1 << 20, 1 << 21
    for kw in (dict(count=-1), dict(count=65537), dict(most=0.0), dict(most=-1.0), dict(most=NAN), dict(g=None), dict(n=None), dict(dt=None),
               dict(dt=(0, 2)), dict(n=(10, -1)), dict(n=(10, (1 << 40) + 1)), dict(g=(a, None)), dict(o=(a, None)), dict(ws=MIS), dict(size=8),
               dict(g=(a, b + 2)), dict(g=(a, b + 1), dt=(0, 1)),      # not aligned to the type
               dict(g=(a, a)), dict(g=(a, a + 36)),                    # in place over each other
               dict(o=(b, b + 400)), dict(o=(a, b), g=(a, b + 4)),     # over another gradient, beside its own
               dict(o=(a + 4, b)), dict(o=(1 << 22, (1 << 22) + 36)),  # beside its own, over each other
               dict(o=(b, a))):                                        # each other's
        refused(rh, call(**kw), "GradClip")
    assert L.ppocr_grad_clip_workspace_bytes(None, 1) == 0
    assert L.ppocr_grad_clip_workspace_bytes((ctypes.c_int64 * 1)(-1), 1) == 0
    assert L.ppocr_grad_clip_workspace_bytes((ctypes.c_int64 * 1)(10), 65537) == 0
    assert L.ppocr_grad_clip_workspace_bytes(None, 0) > 0
    with pytest.raises(rh.OcrError):
        rh.clip_gradients([np.ones(3)], 0.0)
