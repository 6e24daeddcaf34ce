"""Adapted calls beside the ordinary ones: ranks above 32 with many rows and slots in any order, FP32 heads of the model's
size, tensors at any address, a captured single line, host calls of several threads."""
import ctypes

import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from test_gpu_adapt import check_decode, check_logits, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False], ids=["q", "w"])
@pytest.mark.parametrize("lengths", ["mixed", "short", "long"])
def test_high_ranks_of_many_rows(rh, quant, lengths):
    """More than 2048 rows under ranks up to 64, several slots: lines of any length, of a few rows, and one beside empty
    ones."""
    rng = np.random.default_rng(1)
    h = ac.Head(rh, rng, 700, 120, quant, 7, 64, ranks=[64, 33, 48, 0, 64, 5, 64])
    each = {"mixed": rng.integers(0, 130, 40), "short": rng.integers(0, 9, 700), "long": np.array([0, 2300, 0, 65, 1])}[lengths]
    off = ac.offsets(each)
    assert off[-1] > 2048
    slot = rng.integers(-1, 9, each.size).astype(np.int32)  # 7 and above: none, in the device form
    if lengths == "long":
        slot[1] = 4
    a = rows(rng, h, int(off[-1]))
    call = ac.Call(h, a, off, slot)
    o = {k: v.get() for k, v in call.decode().items()}
    call.ws.get()
    check_decode(h, a, off, slot, o, lengths)
    check_logits(h, a, off, slot, call.logits().get(), lengths)
    for k, v in call.decode(ws=False).items():
        assert np.array_equal(v.get(), o[k]), k


@pytest.mark.parametrize("rank", [16, 64])
def test_fp32_heads_of_the_models_size(rh, rank):
    rng = np.random.default_rng(2)
    h = ac.Head(rh, rng, 18710, 120, False, 4, rank)
    off = ac.offsets([120, 43, 0, 150, 31])
    slot = np.array([2, -1, 0, 3, 1], np.int32)
    a = rows(rng, h, int(off[-1]))
    check_decode(h, a, off, slot, {k: v.get() for k, v in ac.Call(h, a, off, slot).decode().items()}, f"rank {rank}")


def test_rows_and_outputs_at_any_address(rh):
    """Rows, logits and an adapter's tensors aligned to their type only: the same bits."""
    rng = np.random.default_rng(3)
    h = ac.Head(rh, rng, 333, 120, True, 2, 16)
    off, slot = ac.offsets([40, 1, 59]), [1, -1, 0]
    a = rows(rng, h, 100)
    want = ac.Call(h, a, off, slot)
    z, o = want.logits().get(), want.decode()
    job = ac.Call(h, a, off, slot)
    moved = tc.up(np.concatenate([np.zeros(1, np.float32), a.ravel()]))
    out = tc.Out((1 + 100 * 333,), np.float32)
    w, p = job.ws.p, ctypes.c_void_p
    job.h.rh._check(job.L.ppocr_ra_logits_dev(h.head.handle, p(moved.p.value + 4), 100, job.off.p, 3, job.slot.p, p(out.p.value + 4), w,
                                              job.bytes, None))
    assert np.array_equal(out.get()[1:].reshape(100, 333), z)
    job.a = type("at", (), {"p": p(moved.p.value + 4)})
    for k, v in job.decode().items():
        assert np.array_equal(v.get(), o[k].get()), k
    down, up, scale = (v for v in h.adapters[0])
    for dt, width in ((tc.F32, 4), (tc.BF16, 2)):
        at = []
        for x in (down, up):
            raw, _ = tc.typed(x.astype(np.float32), dt)
            at.append((raw, tc.up(raw), tc.up(np.concatenate([np.zeros(1, raw.dtype), raw.ravel()]))))
        got = []
        for shift in (0, 1):
            d, u = (p(v[1 + shift].p.value + shift * width) for v in at)
            job.h.rh._check(job.L.ppocr_ra_set_dev(h.head.handle, 0, d, u, 16, scale, dt, None))
            got.append(ac.Call(h, a, off, slot).logits().get())
        assert np.array_equal(got[0], got[1])


def test_captured_single_line(rh):
    """A line by itself, which needs no plan: replayed on other offsets and slots."""
    from ppocr_rechead.hip import H2D, Stream, check, hip, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(4)
    h = ac.Head(rh, rng, 700, 120, False, 3, 16)
    m = 150
    a = rows(rng, h, m)
    call = ac.Call(h, a, [0, m], [0])
    st = Stream()
    out, o = tc.Out((m, h.n), np.float32), call.outputs()
    synchronize()
    graph = _Graph(st, lambda: (call.logits(st.h, out=out), call.decode(st.h, o=o)))
    for off, s in (([0, 150], 2), ([0, 40], 0), ([30, 150], -1), ([0, 150], 1)):
        for d, v in ((call.off, np.array(off, np.int64)), (call.slot, np.array([s], np.int32))):
            check(hip().hipMemcpy(d.p, ac.ctypes_ptr(v), ctypes.c_size_t(v.nbytes), H2D), "hipMemcpy")
        synchronize()
        graph.replay()
        check_logits(h, a, off, [s], out.get(), f"replay {off} {s}")
        eager = ac.Call(h, a, off, [s])
        assert np.array_equal(eager.logits().get(), out.get())
        for k, v in eager.decode().items():
            # (rows of no line are left as they were)
            at = slice(*off) if k in ("idx", "maxprob") else slice(None)
            if k != "seq":
                assert np.array_equal(v.get()[at], o[k].get()[at]), (off, s, k)
    graph.close()


def test_host_calls_of_several_threads(rh):
    """Host forms on one handle at once, while another of its slots is set."""
    import threading
    rng = np.random.default_rng(5)
    h = ac.Head(rh, rng, 900, 120, True, 4, 32)
    off = ac.offsets([50, 30, 70])
    a = rows(rng, h, 150)
    slots = [np.array(s, np.int32) for s in ([0, 1, -1], [2, 2, 0], [1, -1, 2])]
    want = [h.head.logits_lines(a, off, s) for s in slots]
    new = ((rng.standard_normal((32, 120)) / 11).astype(np.float32), (rng.standard_normal((900, 32)) * 0.05).astype(np.float32))
    bad = []

    def work(i):
        try:
            for _ in range(8):
                if i < 3:
                    bad.append(not np.array_equal(h.head.logits_lines(a, off, slots[i]), want[i]))
                    h.head.decode_lines(a, off, slots[i])
                else:
                    h.head.set_adapter(3, *new)
        except Exception as e:  # a thread's exception would pass unseen
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not any(bad), bad
    h.adapters[3] = tuple(v.astype(np.float64) for v in new) + (1.0,)
    s = np.array([3, 0, 3], np.int32)
    check_logits(h, a, off, s, h.head.logits_lines(a, off, s), "the slot that was set")
