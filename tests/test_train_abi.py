"""What the training entry points refuse, and what they take without work, before any HIP call: no
device is needed.  Every refusal names its operator and leaves the outputs alone."""
import ctypes

import numpy as np
import pytest

P = ctypes.c_void_p(1 << 20)  # never read: each call is refused, or has nothing to do
MIS = ctypes.c_void_p((1 << 20) + 4)


def xent(L, which, **kw):
    a = dict(a=P, w=P, bias=P, target=P, m=4, n=10, k=8, dt=0, loss=P, lse=P, grad=P, da=P, dw=P, db=P, ws=P, bytes=1 << 40)
    a.update(kw)
    head = (a["a"], a["w"], a["bias"], a["target"])
    shape = (a["m"], a["n"], a["k"])
    if which == "forward":
        return L.ppocr_xent_forward_dev(*head, *shape, a["dt"], a["loss"], a["lse"], a["ws"], a["bytes"], None)
    return L.ppocr_xent_backward_dev(*head, a["lse"], a["grad"], *shape, a["dt"], a["da"], a["dw"], a["db"], a["ws"],
                                     a["bytes"], None)


def distill(L, which, **kw):
    a = dict(a=P, w=P, bias=P, idx=P, z=P, t=4, tau=1.0, m=4, n=10, k=8, dt=0, loss=P, lse=P, grad=P, da=P, dw=P, db=P, ws=P,
             bytes=1 << 40)
    a.update(kw)
    head = (a["a"], a["w"], a["bias"], a["idx"], a["z"], a["t"], a["tau"])
    shape = (a["m"], a["n"], a["k"])
    if which == "forward":
        return L.ppocr_distill_forward_dev(*head, *shape, a["dt"], a["loss"], a["lse"], a["ws"], a["bytes"], None)
    return L.ppocr_distill_backward_dev(*head, a["lse"], a["grad"], *shape, a["dt"], a["da"], a["dw"], a["db"], a["ws"],
                                        a["bytes"], None)


@pytest.mark.parametrize("which", ["forward", "backward"])
@pytest.mark.parametrize("call,op", [(xent, "SoftmaxCrossEntropy"), (distill, "Distill")])
def test_losses_refuse(rh, call, op, which):
    L = rh._lib.lib()
    bad = [dict(m=-1), dict(n=-1), dict(k=-1), dict(n=0), dict(k=0), dict(k=257), dict(m=(1 << 24) + 1),
           dict(n=(1 << 24) + 1), dict(dt=2), dict(dt=-1), dict(a=None), dict(w=None), dict(lse=None), dict(ws=MIS),
           dict(bytes=100)]
    if which == "forward":
        bad.append(dict(loss=None))
    if call is distill:
        bad += [dict(t=0), dict(t=65), dict(t=-1), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")),
                dict(tau=float("inf")), dict(tau=1e-9), dict(idx=None), dict(z=None)]
    else:
        bad.append(dict(target=None))
    for kw in bad:
        assert call(L, which, **kw) == rh.PPOCR_ERR_INVALID_ARG, kw
        assert rh._lib.last_error().startswith(op + ": "), (kw, rh._lib.last_error())
    if which == "forward":
        assert call(L, which, m=0, a=None, loss=None, lse=None) == rh.PPOCR_OK
    else:
        assert call(L, which, da=None, dw=None, db=None) == rh.PPOCR_OK
        assert call(L, which, m=0, dw=None, db=None) == rh.PPOCR_OK  # da of no rows


def test_workspace_sizes(rh):
    L = rh._lib.lib()
    for bad in ((0, 10, 8, 0), (-1, 10, 8, 0), (4, 0, 8, 0), (4, 10, 0, 0), (4, 10, 300, 0), (4, 10, 8, 7)):
        assert L.ppocr_xent_workspace_bytes(*bad) == 0
    assert L.ppocr_distill_workspace_bytes(4, 10, 8, 65, 0) == 0
    assert L.ppocr_layernorm_workspace_bytes(0, 8) == 0 and L.ppocr_layernorm_workspace_bytes(4, 16385) == 0
    for dt in (0, 1):
        # far below the logits' 4 m n bytes
        assert 0 < L.ppocr_xent_workspace_bytes(30720, 18710, 120, dt) < 30720 * 18710 * 4 // 8
        assert L.ppocr_xent_workspace_bytes(1 << 24, 1 << 24, 256, dt) > 0
    assert L.ppocr_distill_workspace_bytes(100, 1000, 80, 64, 0) > L.ppocr_distill_workspace_bytes(100, 1000, 80, 1, 0)


def test_topk_refuses(rh):
    L = rh._lib.lib()
    for rows, cols, t, x, i, v in ((-1, 5, 1, P, P, P), (5, -1, 1, P, P, P), (5, 5, 0, P, P, P), (5, 5, 65, P, P, P),
                                   (5, 1 << 31, 1, P, P, P), (5, 5, 1, None, P, P), (5, 5, 1, P, None, P), (5, 5, 1, P, P, None)):
        assert L.ppocr_topk_rows_dev(x, rows, cols, t, i, v, None) == rh.PPOCR_ERR_INVALID_ARG
        assert rh._lib.last_error().startswith("TopK: ")
        assert L.ppocr_topk_rows(x, rows, cols, t, i, v) == rh.PPOCR_ERR_INVALID_ARG
    assert L.ppocr_topk_rows_dev(None, 0, 5, 1, None, None, None) == rh.PPOCR_OK


def test_layer_norm_refuses(rh):
    L = rh._lib.lib()

    def forward(x=P, w=P, b=P, m=4, d=8, eps=1e-5, dt=0, y=P):
        return L.ppocr_layernorm_forward_dev(x, w, b, m, d, eps, dt, y, P, P, None)

    def backward(dy=P, x=P, w=P, mean=P, rstd=P, m=4, d=8, dt=0, dx=P, dw=P, db=P, ws=P, size=1 << 30):
        return L.ppocr_layernorm_backward_dev(dy, x, w, mean, rstd, m, d, dt, dx, dw, db, ws, size, None)

    for f, bad in ((forward, [dict(m=-1), dict(d=-1), dict(d=0), dict(d=16385), dict(m=(1 << 31) + 1), dict(dt=3),
                              dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(w=None),
                              dict(b=None), dict(y=None)]),
                   (backward, [dict(m=-1), dict(d=0), dict(d=16385), dict(dt=3), dict(dy=None), dict(x=None), dict(w=None),
                               dict(mean=None), dict(rstd=None), dict(ws=MIS), dict(size=16)])):
        for kw in bad:
            assert f(**kw) == rh.PPOCR_ERR_INVALID_ARG, kw
            assert rh._lib.last_error().startswith("LayerNorm: "), kw
    assert forward(m=0, x=None) == rh.PPOCR_OK
    assert backward(dx=None, dw=None, db=None) == rh.PPOCR_OK


def test_host_forms_of_no_rows(rh):
    """No rows: empty losses, zero gradients, without a device."""
    w = np.ones((5, 3), np.float32)
    loss, lse = rh.cross_entropy(np.zeros((0, 3)), w, None, np.zeros(0))
    assert loss.shape == lse.shape == (0,)
    da, dw, db = rh.cross_entropy_backward(np.zeros((0, 3)), w, None, np.zeros(0), lse)
    assert da.shape == (0, 3) and (dw == 0).all() and dw.shape == (5, 3) and (db == 0).all()
    da, dw, db = rh.distill_backward(np.zeros((0, 3)), w, None, np.zeros((0, 2)), np.zeros((0, 2)), 1.0, lse)
    assert (dw == 0).all() and (db == 0).all()
    y, mean, rstd = rh.layer_norm(np.zeros((0, 3)), np.ones(3), np.ones(3), 1e-5)
    dx, dw, db = rh.layer_norm_backward(y, y, np.ones(3), mean, rstd)
    assert dx.shape == (0, 3) and (dw == 0).all() and (db == 0).all()


def test_mirror_refuses(rh):
    a, w = np.ones((4, 3), np.float32), np.ones((5, 3), np.float32)
    for call in (lambda: rh.cross_entropy(a, np.ones((5, 4)), None, np.zeros(4)),
                 lambda: rh.cross_entropy(a, w, np.ones(4), np.zeros(4)),
                 lambda: rh.cross_entropy(a, w, None, np.zeros(3)),
                 lambda: rh.cross_entropy(a, w, None, np.full(4, 5)),  # not a class
                 lambda: rh.cross_entropy(a[0], w, None, np.zeros(4)),
                 lambda: rh.cross_entropy_backward(a, w, None, np.zeros(4), np.zeros(3)),
                 lambda: rh.cross_entropy_backward(a, w, None, np.zeros(4), np.zeros(4), np.zeros(5)),
                 lambda: rh.cross_entropy_backward(a, w, None, np.full(4, 9), np.zeros(4)),
                 lambda: rh.distill(a, w, None, np.zeros((3, 2)), np.zeros((3, 2))),
                 lambda: rh.distill(a, w, None, np.zeros((4, 2)), np.zeros((4, 3))),
                 lambda: rh.distill(a, w, None, np.full((4, 2), 5), np.zeros((4, 2))),
                 lambda: rh.distill(a, w, None, np.zeros((4, 2)), np.zeros((4, 2)), 0.0),
                 lambda: rh.distill(a, w, None, np.zeros((4, 65)), np.zeros((4, 65))),
                 lambda: rh.topk(a, 0), lambda: rh.topk(a, 65), lambda: rh.topk(a[0], 1),
                 lambda: rh.layer_norm(a, np.ones(4), np.ones(3), 1e-5),
                 lambda: rh.layer_norm(a, np.ones(3), np.ones(3), -1.0),
                 lambda: rh.layer_norm_backward(a, a, np.ones(3), np.ones(3), np.ones(4))):
        with pytest.raises(rh.OcrError):
            call()
