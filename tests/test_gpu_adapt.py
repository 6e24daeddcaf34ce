"""Low-rank adapters of many text lines beside the shared projection: logits and decoded lines against the
formula in 64 bits, over heads, ranks, types, line lengths and slots, with rows of extreme sizes, replaced
adapters, captured calls, streams and refusals."""
import ctypes

import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from train_common import BF16, F32

pytestmark = pytest.mark.gpu


def rows(rng, h, m, sure=6.0):
    """Rows that lean towards a class each, every third towards the blank."""
    to = rng.integers(min(1, h.n - 1), h.n, m)
    to[::3] = 0
    d = h.w[to]
    size = np.maximum(np.linalg.norm(d, axis=1, keepdims=True), 1e-2)
    return (rng.standard_normal((m, h.k)) * 0.3 + (np.log(h.n) + sure * rng.random((m, 1))) / size * d / size).astype(np.float32)


def check_logits(h, a, off, slot, got, label):
    z, e = h.exact(a, h.rows_of(a.shape[0], off, slot))
    tc.close(got, z, e, label)


def check_decode(h, a, off, slot, o, label):
    z, e = h.exact(a, h.rows_of(a.shape[0], off, slot))
    top = z.max(axis=1)
    best = z.argmax(axis=1)
    err = e.max(axis=1)
    idx = o["idx"]
    # another class only where the errors reach the gap to it
    at = np.arange(len(idx))
    assert (z[at, idx] >= top - 2 * err).all(), label
    assert (idx != best).mean() < 0.01, label
    p = 1.0 / np.exp(z - top[:, None]).sum(axis=1)
    # exponents are off by the logits' errors, the sum adds a tile's 16 values, its tiles, its chunks
    tol = p * (2 * err + (16 + h.n / 32 + 160) * tc.U24)
    tc.close(o["maxprob"], p, tol, label + " maxprob")
    seqs, scores = ac.collapse(idx, o["maxprob"], off)
    for i, want in enumerate(seqs):
        n = int(o["len"][i])
        assert o["seq"][off[i]:off[i] + n].tolist() == want, (label, i)
        assert abs(o["score"][i] - scores[i]) <= (len(want) + 2) * tc.U24 * max(scores[i], 1e-6), (label, i)
        # what lies behind a line's text stays as it was
        assert (o["seq"][off[i] + n:off[i + 1]] == np.int32(-1515870811)).all(), (label, i)


SHAPES = [
    # n, k, INT8, slots, max rank, ranks, type, line lengths
    (700, 120, True, 3, 16, None, F32, [40, 1, 33, 64]),
    (701, 113, True, 2, 16, [16, 7], BF16, [5, 31, 32, 33]),
    (333, 80, True, 5, 32, [1, 17, 32, 0, 9], F32, [50, 20, 0, 90, 13, 7, 64]),
    (1000, 73, False, 4, 64, [64, 33, 48, 5], F32, [100, 3, 77, 1, 1, 40]),
    (515, 117, False, 1, 1, None, BF16, [1]),
    (96, 118, False, 2, 24, None, F32, [200, 130, 64, 1]),
    (31, 120, True, 2, 8, None, F32, [3, 3]),
    (1, 80, False, 1, 4, None, F32, [4]),
    (18710, 120, True, 6, 16, None, F32, [120, 43, 150]),
    (6906, 80, True, 3, 64, None, BF16, [1] * 70),
]


@pytest.mark.parametrize("case", SHAPES, ids=[f"n{c[0]}-k{c[1]}-{'q' if c[2] else 'w'}-r{c[4]}" for c in SHAPES])
def test_logits_and_decode(rh, case):
    n, k, quant, slots, rank, ranks, dt, lengths = case
    print(case, flush=True)
    rng = np.random.default_rng(n + k)
    h = ac.Head(rh, rng, n, k, quant, slots, rank, ranks, dt)
    off = ac.offsets(lengths)
    m = int(off[-1])
    slot = rng.integers(-1, slots, len(lengths)).astype(np.int32)
    if len(lengths) > 1:
        slot[0], slot[-1] = slots - 1, -1
    else:
        slot[0] = 0
    a = rows(rng, h, m)
    call = ac.Call(h, a, off, slot)
    z = call.logits().get()
    check_logits(h, a, off, slot, z, "logits")
    o = {k_: v.get() for k_, v in call.decode().items()}
    call.ws.get()
    check_decode(h, a, off, slot, o, "decode")
    # the call's own workspace, and the host forms: the same bits
    assert np.array_equal(call.logits(ws=False).get(), z)
    assert np.array_equal(h.head.logits_lines(a, off, slot), z)
    d = h.head.decode_lines(a, off, slot)
    assert np.array_equal(d["idx"], o["idx"]) and np.array_equal(d["maxprob"], o["maxprob"])
    assert np.array_equal(d["score"], o["score"]) and np.array_equal(d["seq_len"], o["len"])


def test_many_rows_many_slots(rh):
    """More units than a workgroup's waves, lines of slots in any order, over several row blocks and chunks."""
    rng = np.random.default_rng(5)
    h = ac.Head(rh, rng, 2000, 120, True, 40, 16)
    off = ac.offsets(rng.integers(0, 90, 150))
    slot = rng.integers(-1, 44, 150).astype(np.int32)  # 40 and above: none, in the device form
    a = rows(rng, h, int(off[-1]))
    call = ac.Call(h, a, off, slot)
    check_logits(h, a, off, slot, call.logits().get(), "logits")
    check_decode(h, a, off, slot, {k: v.get() for k, v in call.decode().items()}, "decode")


def test_a_rows_bits_do_not_depend_on_its_company(rh):
    """A line alone, beside others, and as the lines of another order: the same logits, bit for bit."""
    rng = np.random.default_rng(6)
    h = ac.Head(rh, rng, 900, 120, True, 3, 16)
    lengths = [37, 64, 5, 90]
    off = ac.offsets(lengths)
    slot = np.array([0, 1, -1, 2], np.int32)
    a = rows(rng, h, int(off[-1]))
    whole = ac.Call(h, a, off, slot).logits().get()
    for i in range(4):
        part = a[off[i]:off[i + 1]]
        alone = ac.Call(h, part, ac.offsets([lengths[i]]), slot[i:i + 1]).logits().get()
        assert np.array_equal(alone, whole[off[i]:off[i + 1]]), i


@pytest.mark.parametrize("quant", [True, False])
def test_a_rows_bits_do_not_depend_on_its_neighbours(rh, quant):
    """Ordinary rows beside rows of any size, of zeros and of infinities, under one slot: the same bits as beside
    ordinary ones, and in each of several calls."""
    rng = np.random.default_rng(19)
    h = ac.Head(rh, rng, 900, 120, quant, 3, 16)
    lengths = rng.integers(1, 9, 80)
    off = ac.offsets(lengths)
    m = int(off[-1])
    slot = rng.integers(-1, 3, 80).astype(np.int32)
    a = rows(rng, h, m)
    a *= (rng.random((m, 120)) * 2.0 ** rng.integers(-12, 1, (m, 120))).astype(np.float32)  # low halves far below the top
    b = a.copy()
    at = rng.random(m) < 0.3
    b[at] *= (2.0 ** rng.integers(-60, 20, at.sum()))[:, None].astype(np.float32)
    b[np.flatnonzero(at)[::7]] = 0.0
    b[np.flatnonzero(at)[::9], 5] = np.inf
    first, second = ac.Call(h, a, off, slot), ac.Call(h, b, off, slot)
    za, oa = first.logits().get(), {k: v.get() for k, v in first.decode().items()}
    for _ in range(4):
        zb, ob = second.logits().get(), {k: v.get() for k, v in second.decode().items()}
        assert np.array_equal(za[~at], zb[~at])
        for k in ("idx", "maxprob"):
            assert np.array_equal(oa[k][~at], ob[k][~at]), k
        for x, y in ((first.logits().get(), za), (second.logits().get(), zb)):
            assert np.array_equal(x, y, equal_nan=True)


def test_classes_of_tiny_weights(rh):
    """An INT8 head with classes of weights that all but vanish, down to the least scale that packing gives and to
    zeros, beside an ordinary adapter: every class keeps its bits, the head's own calls on the handle theirs."""
    rng = np.random.default_rng(20)
    n, k = 300, 120
    for tiny in (1e-4, 1e-6, 5e-9, 1e-9):
        w = (rng.standard_normal((n, k)) * 0.05).astype(np.float32)
        w[::7] *= np.float32(tiny / 0.05)
        qw = rh.QuantizedWeight.from_f32_transposed(w)
        h = ac.Head(rh, rng, n, k, True, 1, 16)
        h.base = rh.RecHead(qw=qw, bias=h.bias)
        h.w = qw.data.astype(np.float64) * qw.scales.astype(np.float64)[:, None]
        h.head = rh.AdaptedHead(h.base, 1, 16)
        down = (rng.standard_normal((16, k)) / np.sqrt(k)).astype(np.float32)
        up = (rng.standard_normal((n, 16)) * 0.05).astype(np.float32)
        h.set(0, down, up, 1.0)
        a = rows(rng, h, 70)
        call = ac.Call(h, a, [0, 70], [0])
        check_logits(h, a, [0, 70], [0], call.logits().get(), f"weights of {tiny}")
        check_decode(h, a, np.array([0, 70]), [0], {x: v.get() for x, v in call.decode().items()}, f"weights of {tiny}")
        none = ac.Call(h, a, [0, 70], [-1]).logits().get()
        tc.close(none, *h.exact(a, np.full(70, -1)), "no adapter")
        assert np.array_equal(h.head.logits(a), h.base.logits(a))


def test_fp32_heads_of_any_size(rh):
    """FP32 heads whose weights are all small, all large, or far apart from class to class: 22 bits of each class's
    weights, and of classes 2^-8 of the largest and below the same of that."""
    rng = np.random.default_rng(21)
    n, k = 300, 120
    for size in (2.0 ** -30, 1e-6, 1e-3, 1.0, 3000.0, None):
        w = (rng.standard_normal((n, k)) * 0.2).astype(np.float32)
        w *= (10.0 ** rng.uniform(-9, 0, (n, 1))).astype(np.float32) if size is None else np.float32(size)
        w[5] = 0.0
        h = ac.Head(rh, rng, n, k, False, 2, 16, ranks=[0, 0])
        h.base = rh.RecHead(w_t=w, bias=h.bias)
        h.w = w.astype(np.float64)
        h.head = rh.AdaptedHead(h.base, 2, 16)
        most = np.abs(w).max()
        down = (rng.standard_normal((16, k)) / np.sqrt(k)).astype(np.float32)
        for slot, up in enumerate((1e-3, 1.0)):
            h.set(slot, down, (rng.standard_normal((n, 16)) * up * most).astype(np.float32), 1.0)
        a = (rng.standard_normal((90, k)) * 4).astype(np.float32)
        off, slot = ac.offsets([30, 30, 30]), [0, 1, -1]
        z, e = h.exact(a, h.rows_of(90, off, slot))
        # two halves of values below 2 p, p the power of two above 2^-8 of the largest weight or the class's: 2^-25 of a
        # unit of p each, of the weights against the rows and of up (its powers of two undone) against u
        unit = np.maximum(np.maximum(np.abs(w).max(axis=1), 2.0 ** -8 * most), 2.0 ** -35) * 2
        rough = np.abs(a).max(axis=1, keepdims=True) * unit * 2.0 ** -25
        e = e + rough * (k + 16)
        tc.close(ac.Call(h, a, off, slot).logits().get(), z, e, f"weights of {size}")


def test_rows_of_any_size(rh):
    """Rows scaled by powers of two far apart, of zeros, and rows with infinities and NaN beside them: each keeps
    its own bits."""
    rng = np.random.default_rng(7)
    for quant in (True, False):
        h = ac.Head(rh, rng, 400, 120, quant, 2, 16)
        m = 96
        a = rows(rng, h, m)
        plain = a.copy()
        power = rng.integers(-40, 40, m)
        a = (a * (2.0 ** power)[:, None]).astype(np.float32)
        a[5] = 0.0
        a[11, 3] = np.inf
        a[40, 7] = np.nan
        a[41] = -np.inf
        odd = np.zeros(m, bool)
        odd[[11, 40, 41]] = True
        off, slot = ac.offsets([48, 48]), np.array([0, 1], np.int32)
        call = ac.Call(h, a, off, slot)
        z = call.logits().get()
        assert np.isnan(z[odd]).all()
        a0 = np.where(odd[:, None], 0.0, a).astype(np.float32)
        want, e = h.exact(a0, h.rows_of(m, off, slot))
        tc.close(z[~odd], want[~odd], e[~odd], f"sizes, INT8 {quant}")
        o = {k: v.get() for k, v in call.decode().items()}
        assert (o["idx"][odd] == 0).all()
        assert (o["idx"] >= 0).all() and (o["idx"] < h.n).all()
        ok = ~odd & (np.abs(power) < 3)
        assert np.array_equal(o["idx"][ok], want[ok].argmax(axis=1))
        del plain


def test_large_and_small_adapters(rh):
    """Adapters far larger and smaller than the head's weights, with rows of down and columns of up far
    apart from each other."""
    rng = np.random.default_rng(8)
    for quant in (True, False):
        h = ac.Head(rh, rng, 300, 120, quant, 4, 16, ranks=[0, 0, 0, 0])
        for s, (dscale, uscale) in enumerate(((1.0, 1e4), (1e-6, 1e-3), (1e5, 1e-7), (1e8, 1e6))):
            down = (rng.standard_normal((12, 120)) * dscale).astype(np.float32)
            up = (rng.standard_normal((300, 12)) * uscale).astype(np.float32)
            h.set(s, down, up, 1.0)
        a = rows(rng, h, 128)
        off, slot = ac.offsets([32] * 4), np.arange(4, dtype=np.int32)
        check_logits(h, a, off, slot, ac.Call(h, a, off, slot).logits().get(), f"adapters, INT8 {quant}")
        # components of one adapter that cancel each other's size
        down = (rng.standard_normal((16, 120)) * 10.0 ** rng.integers(-8, 8, (16, 1))).astype(np.float32)
        up = (rng.standard_normal((300, 16)) / np.abs(down).sum(axis=1)).astype(np.float32)
        h.set(0, down, up, 2.0)
        check_logits(h, a, off, slot, ac.Call(h, a, off, slot).logits().get(), f"components, INT8 {quant}")


def test_replaced_and_emptied_slots(rh):
    rng = np.random.default_rng(9)
    h = ac.Head(rh, rng, 500, 80, True, 3, 32)
    a = rows(rng, h, 60)
    off, slot = ac.offsets([20, 20, 20]), np.array([0, 1, 2], np.int32)
    call = ac.Call(h, a, off, slot)
    check_logits(h, a, off, slot, call.logits().get(), "first")
    # a smaller rank over a larger one, another slot emptied
    h.set(0, rng.standard_normal((3, 80)).astype(np.float32), (rng.standard_normal((500, 3)) * 0.1).astype(np.float32), -1.5)
    h.head.clear_adapter(1)
    h.adapters[1] = None
    z = call.logits().get()
    check_logits(h, a, off, slot, z, "second")
    # an emptied slot, no slot, and the head without adapters: equal bits of the first two
    none = ac.Call(h, a, off, np.array([-1, -1, 1], np.int32)).logits().get()
    assert np.array_equal(none[20:40], z[20:40])
    base = h.head.logits(a)
    assert np.abs(base - none).max() < 1e-4
    assert np.array_equal(base, h.base.logits(a))


def test_rows_of_no_line_and_offsets_that_go_backwards(rh):
    """Rows that no line covers have the head's own logits; offsets that go backwards give each row the
    adapter of one of the lines, or none."""
    rng = np.random.default_rng(10)
    h = ac.Head(rh, rng, 300, 120, True, 3, 8)
    m = 100
    a = rows(rng, h, m)
    call = ac.Call(h, a, [10, 30, 70], [0, 2])
    want, e = h.exact(a, np.concatenate([np.full(10, -1), np.full(20, 0), np.full(40, 2), np.full(30, -1)]))
    tc.close(call.logits().get(), want, e, "gaps")
    each = [h.exact(a, np.full(m, s)) for s in (-1, 0, 1, 2)]
    for off in ([50, 20, 90, 10], [-5, 40, 200, 60], [1 << 40, 5, 3, -(1 << 40)]):
        z = ac.Call(h, a, off, [0, 1, 2]).logits().get()
        fits = np.stack([(np.abs(z - w) <= t).all(axis=1) for w, t in each])
        assert fits.any(axis=0).all(), off
    # no lines at all
    none = ac.Call(h, a, [0], np.zeros(1, np.int32))
    tc.close(none.logits().get(), *each[0], "no lines")


def test_single_lines(rh):
    """One line, wherever it begins and ends and whatever slot it names; rows before and behind it are the head's."""
    rng = np.random.default_rng(17)
    h = ac.Head(rh, rng, 333, 120, True, 2, 16)
    big = ac.Head(rh, rng, 333, 120, False, 2, 64)
    for m in (1, 31, 32, 33, 100, 2100):
        for head in (h, big):
            a = rows(rng, head, m)
            each = [head.exact(a, np.full(m, s)) for s in (-1, 0, 1)]
            for off, slot in (([0, m], 1), ([0, m], -1), ([0, m], 2), ([m // 3, m], 0), ([0, m - m // 3], 1), ([m // 3, m // 2], 0),
                              ([-9, 1 << 40], 1), ([m, 0], 1), ([m, m], 0)):
                lo, hi = (min(max(x, 0), m) for x in off)
                used = slot if 0 <= slot < 2 else -1
                at = np.zeros((m, 1), bool)
                at[lo:hi] = True
                z, e = (np.where(at, each[used + 1][x], each[0][x]) for x in (0, 1))
                call = ac.Call(head, a, off, [slot])
                tc.close(call.logits().get(), z, e, f"{m} {off} {slot}")
                o = {k: v.get() for k, v in call.decode().items()}
                if off == [0, m]:
                    check_decode(head, a, np.array(off), [slot], o, f"{m} {slot}")


def test_no_lines(rh):
    """Without lines every row is the head's, and no table is read."""
    rng = np.random.default_rng(18)
    h = ac.Head(rh, rng, 100, 80, True, 2, 4)
    a = rows(rng, h, 50)
    d, out = tc.up(a), tc.Out((50, 100), np.float32)
    h.rh._check(h.rh._lib.lib().ppocr_ra_logits_dev(h.head.handle, d.p, 50, None, 0, None, out.p, None, 0, None))
    tc.close(out.get(), *h.exact(a, np.full(50, -1)), "no lines")


def test_slots_beyond_the_first_thousand(rh):
    rng = np.random.default_rng(11)
    h = ac.Head(rh, rng, 64, 80, True, 4096, 1, ranks=[0] * 4096)
    used = [0, 1000, 4095]
    for s in used:
        h.set(s, rng.standard_normal((1, 80)).astype(np.float32), rng.standard_normal((64, 1)).astype(np.float32), 0.3)
    a = rows(rng, h, 400)
    off = ac.offsets([1] * 400)
    slot = rng.choice(used + [77, -1], 400).astype(np.int32)
    check_logits(h, a, off, slot, ac.Call(h, a, off, slot).logits().get(), "4096 slots")


def test_captured_calls(rh):
    """Calls recorded into graphs with workspaces of their own, replayed on other rows, lines and slots."""
    from ppocr_rechead.hip import H2D, Stream, check, hip, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(12)
    h = ac.Head(rh, rng, 1200, 120, True, 4, 16)
    m, lines = 300, 6
    a = rows(rng, h, m)
    call = ac.Call(h, a, ac.offsets([50] * lines), np.zeros(lines, np.int32))
    st = Stream()
    out, o = tc.Out((m, h.n), np.float32), call.outputs()
    synchronize()
    graph = _Graph(st, lambda: (call.logits(st.h, out=out), call.decode(st.h, o=o)))
    for turn in range(4):
        cut = np.sort(rng.integers(0, m, lines - 1))
        off = np.concatenate([[0], cut, [m]]).astype(np.int64)
        slot = rng.integers(-1, 4, lines).astype(np.int32)
        a = rows(rng, h, m)
        for d, v in ((call.a, a), (call.off, off), (call.slot, slot)):
            check(hip().hipMemcpy(d.p, ac.ctypes_ptr(v), ctypes.c_size_t(v.nbytes), H2D), "hipMemcpy")
        o["seq"].d.fill_bytes(0xA5)
        synchronize()
        graph.replay()
        check_logits(h, a, off, slot, out.get(), f"replay {turn}")
        got = {k: v.get() for k, v in o.items()}
        check_decode(h, a, off, slot, got, f"replay {turn}")
        eager = {k: v.get() for k, v in ac.Call(h, a, off, slot).decode().items()}
        for k in got:
            assert np.array_equal(got[k], eager[k]), (turn, k)
    graph.close()


def test_two_streams_at_once(rh):
    from ppocr_rechead.hip import Stream
    rng = np.random.default_rng(13)
    h = ac.Head(rh, rng, 3000, 120, False, 3, 32)
    jobs = []
    for i in range(2):
        off = ac.offsets(rng.integers(20, 200, 12))
        slot = rng.integers(-1, 3, 12).astype(np.int32)
        a = rows(rng, h, int(off[-1]))
        jobs.append((ac.Call(h, a, off, slot), Stream(), a, off, slot))
    for _ in range(3):
        got = [(c.decode(s.h), c.logits(s.h)) for c, s, *_ in jobs]
        for (c, s, a, off, slot), (o, z) in zip(jobs, got):
            s.synchronize()
            check_logits(h, a, off, slot, z.get(), "streams")
            check_decode(h, a, off, slot, {k: v.get() for k, v in o.items()}, "streams")


def test_handles_in_any_order(rh):
    """The head may be destroyed before the handles made from it, and an adapted head may be made from another."""
    rng = np.random.default_rng(14)
    h = ac.Head(rh, rng, 200, 120, True, 2, 8)
    other = rh.AdaptedHead(h.head, 1, 4)
    a = rows(rng, h, 10)
    h.base.close()
    off, slot = ac.offsets([10]), np.zeros(1, np.int32)
    check_logits(h, a, off, slot, h.head.logits_lines(a, off, slot), "after the head")
    want, e = h.exact(a, np.full(10, -1))
    tc.close(other.logits_lines(a, off, slot), want, e, "a second handle")
    h.head.close()
    tc.close(other.logits_lines(a, off, slot), want, e, "after the first")
    assert other.device_bytes() > 0
    other.close()


def test_refusals(rh):
    rng = np.random.default_rng(15)
    h = ac.Head(rh, rng, 50, 80, True, 2, 4)
    L, P = h.rh._lib.lib(), ctypes.c_void_p(1 << 20)
    out = ctypes.c_void_p()
    for slots, rank in ((0, 4), (4097, 4), (2, 0), (2, 65), (-1, 4)):
        assert L.ppocr_ra_create(h.base.handle, slots, rank, ctypes.byref(out)) == rh.PPOCR_ERR_INVALID_ARG and not out.value
    # a head that no matrix kernel takes
    odd = rh.RecHead(w_t=np.ones((5, 64), np.float32))
    assert L.ppocr_ra_create(odd.handle, 1, 1, ctypes.byref(out)) == rh.PPOCR_ERR_INVALID_ARG
    big = rh.RecHead(w_t=np.full((5, 80), 40000.0, np.float32))
    assert L.ppocr_ra_create(big.handle, 1, 1, ctypes.byref(out)) == rh.PPOCR_ERR_INVALID_ARG
    # INT8 scales that leave an adapter no unit
    for bad in (0.0, 1e-12, float("inf"), float("nan")):
        qw = rh.QuantizedWeight.from_f32_transposed(np.ones((5, 80), np.float32))
        qw.scales[3] = bad
        assert L.ppocr_ra_create(rh.RecHead(qw=qw).handle, 1, 1, ctypes.byref(out)) == rh.PPOCR_ERR_INVALID_ARG, bad
        assert "scale of class 3" in rh._lib.last_error()
    qw = rh.QuantizedWeight.from_f32_transposed(np.ones((5, 80), np.float32))
    qw.scales[:] = [1.0, 2.0 ** -20, 2.0 ** 20, 1.0, 2.0 ** -21]
    assert L.ppocr_ra_create(rh.RecHead(qw=qw).handle, 1, 1, ctypes.byref(out)) == rh.PPOCR_ERR_INVALID_ARG and not out.value
    assert "further apart" in rh._lib.last_error()
    # a head without adapters
    assert L.ppocr_ra_set_dev(h.base.handle, 0, P, P, 1, 1.0, 0, None) == rh.PPOCR_ERR_INVALID_ARG
    assert L.ppocr_ra_workspace_bytes(h.base.handle, 5) == 0
    assert L.ppocr_ra_shape(h.base.handle, None, None) == rh.PPOCR_ERR_INVALID_ARG
    a = h.head.handle
    for kw in (dict(slot=2), dict(slot=-1), dict(rank=5), dict(rank=-1), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(down=None), dict(up=None), dict(dt=2)):
        v = dict(slot=0, down=P, up=P, rank=2, scale=1.0, dt=0)
        v.update(kw)
        assert L.ppocr_ra_set_dev(a, v["slot"], v["down"], v["up"], v["rank"], v["scale"], v["dt"], None) == rh.PPOCR_ERR_INVALID_ARG, kw
        assert rh._lib.last_error().startswith("LowRankAdapter: ")
    size = L.ppocr_ra_workspace_bytes(a, 8)
    for kw in (dict(m=-1), dict(lines=-1), dict(m=(1 << 30) + 1), dict(a=None), dict(off=None), dict(slot=None), dict(ws=ctypes.c_void_p((1 << 20) + 4)),
               dict(size=size - 1)):
        v = dict(a=P, m=8, off=P, lines=1, slot=P, ws=P, size=size)
        v.update(kw)
        head = (a, v["a"], v["m"], v["off"], v["lines"], v["slot"])
        assert L.ppocr_ra_logits_dev(*head, P, v["ws"], v["size"], None) == rh.PPOCR_ERR_INVALID_ARG, kw
        assert L.ppocr_ra_decode_dev(*head, P, P, P, P, P, v["ws"], v["size"], None) == rh.PPOCR_ERR_INVALID_ARG, kw
    assert L.ppocr_ra_logits_dev(a, P, 8, P, 1, P, None, P, size, None) == rh.PPOCR_ERR_INVALID_ARG
    assert L.ppocr_ra_decode_dev(a, P, 8, P, 1, P, P, P, None, P, P, P, size, None) == rh.PPOCR_ERR_INVALID_ARG
    assert L.ppocr_ra_decode_dev(a, None, 0, None, 0, None, None, None, None, None, None, None, 0, None) == rh.PPOCR_OK
    x = np.ones((8, 80), np.float32)
    for call in (lambda: h.head.logits_lines(x, [0, 8], [2]), lambda: h.head.logits_lines(x, [0, 9], [0]),
                 lambda: h.head.logits_lines(x, [0, 8], [0, 1]), lambda: h.head.logits_lines(x[:, :79], [0, 8], [0]),
                 lambda: h.head.logits_lines(x, [0, 9, 8], [0, 0]), lambda: h.head.set_adapter(0, x[:2], np.ones((49, 2))),
                 lambda: h.head.set_adapter(0, np.ones((5, 80)), np.ones((50, 5))), lambda: h.head.set_adapter(2, x[:2], np.ones((50, 2)))):
        with pytest.raises(rh.OcrError):
            call()
    empty = h.head.decode_lines(np.zeros((0, 80)), [0, 0, 0], [0, -1])
    assert (empty["seq_len"] == 0).all() and (empty["score"] == 0).all()
    assert h.head.logits_lines(np.zeros((0, 80)), [0], []).shape == (0, 50)


def test_allocation_failures(rh, monkeypatch):
    """No device memory: a status, no handle, and the head as it was."""
    rng = np.random.default_rng(16)
    h = ac.Head(rh, rng, 100, 80, True, 1, 4)
    a = rows(rng, h, 4)
    call = ac.Call(h, a, ac.offsets([4]), [0])
    out = ctypes.c_void_p()
    monkeypatch.setenv("PPOCR_RECHEAD_FAULT", "alloc")
    assert call.L.ppocr_ra_create(h.base.handle, 1, 4, ctypes.byref(out)) == rh.PPOCR_ERR_NO_MEMORY and not out.value
    with pytest.raises(rh.OcrError) as e:
        call.logits(ws=False)
    assert e.value.code == rh.PPOCR_ERR_NO_MEMORY
    monkeypatch.delenv("PPOCR_RECHEAD_FAULT")
    check_logits(h, a, ac.offsets([4]), [0], call.logits().get(), "after the failure")
