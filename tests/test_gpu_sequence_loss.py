"""The policy and preference losses over lines of steps against the formulas in 64 bits."""
import numpy as np
import pytest

import adapt_common as ac
import train_common as tc

pytestmark = pytest.mark.gpu


def steps(rng, m, masked=0.1):
    loss = np.exp(rng.standard_normal(m) * 2 - 2).astype(np.float32)
    target = np.where(rng.random(m) < masked, -1, 3).astype(np.int32)
    old = np.maximum(loss + rng.standard_normal(m) * 0.2, 0).astype(np.float32)
    ref = np.maximum(loss + rng.standard_normal(m) * 0.4, 0).astype(np.float32)
    return loss, old, ref, target


class Policy:
    def __init__(self, rh, loss, old, ref, target, adv, off, low=0.2, high=0.28, beta=0.05, grad=None):
        self.rh, self.L = rh, rh._lib.lib()
        self.m, self.lines = loss.shape[0], len(off) - 1
        self.per_row = adv.shape[0] == self.m and self.m != self.lines
        self.v = (loss, old, ref, target, adv, off, low, high, beta, grad)
        self.dev = [tc.up(x) for x in (loss, old, ref, target, adv, np.asarray(off, np.int64), grad)]
        self.par = (low, high, beta)

    def outputs(self):
        return {"loss": tc.Out((self.lines,), np.float32), "kl": tc.Out((self.lines,), np.float32),
                "clipped": tc.Out((self.lines,), np.float32), "row_grad": tc.Out((self.m,), np.float32)}

    def run(self, o, stream=None):
        loss, old, ref, target, adv, off, grad = (tc.ptr(d) for d in self.dev)
        self.rh._check(self.L.ppocr_policy_loss_dev(loss, old, ref, target, adv, int(self.per_row), off, self.lines, self.m,
                                                    *self.par, grad, *(tc.ptr(o.get(k)) for k in ("loss", "kl", "clipped", "row_grad")),
                                                    stream))
        return o

    def check(self, got, label):
        loss, old, ref, target, adv, off, low, high, beta, grad = self.v
        ref64, tol = ac.policy64(loss, old, ref, target, adv, self.per_row, off, low, high, beta, grad)
        for k in got:
            tc.close(got[k], ref64[k], tol[k], f"{label} {k}")


class Preference:
    def __init__(self, rh, loss, ref, target, off, beta=0.1, smoothing=0.0, average=False, grad=None):
        self.rh, self.L = rh, rh._lib.lib()
        self.m, self.pairs = loss.shape[0], (len(off) - 1) // 2
        self.v = (loss, ref, target, off, beta, smoothing, average, grad)
        self.dev = [tc.up(x) for x in (loss, ref, target, np.asarray(off, np.int64), grad)]

    def outputs(self):
        return {"loss": tc.Out((self.pairs,), np.float32), "reward": tc.Out((2 * self.pairs,), np.float32),
                "row_grad": tc.Out((self.m,), np.float32)}

    def run(self, o, stream=None):
        loss, ref, target, off, grad = (tc.ptr(d) for d in self.dev)
        beta, smoothing, average = self.v[4:7]
        self.rh._check(self.L.ppocr_preference_loss_dev(loss, ref, target, off, self.pairs, self.m, beta, smoothing, int(average),
                                                        grad, *(tc.ptr(o.get(k)) for k in ("loss", "reward", "row_grad")), stream))
        return o

    def check(self, got, label):
        want, tol = ac.preference64(*self.v)
        for k in got:
            tc.close(got[k], want[k], tol[k], f"{label} {k}")


LENGTHS = [[1], [7, 0, 1, 64, 65], [120] * 29, [257, 255, 256, 3], [1000, 4097, 2], [1] * 500, [0, 0, 5], [20000], [0],
           [600] * 5, [5000, 9000], [16384], [30000, 3, 0, 70001, 65, 20000], [2] * 3 + [300000], [33000, 32999]]
IDS = [f"{len(x)}x{max(x)}" for x in LENGTHS]


@pytest.mark.parametrize("lengths", LENGTHS, ids=IDS)
@pytest.mark.parametrize("per_row,with_ref", [(False, True), (True, False), (True, True)])
def test_policy(rh, lengths, per_row, with_ref):
    print(lengths[:6], flush=True)
    rng = np.random.default_rng(len(lengths) + max(lengths))
    off = ac.offsets(lengths)
    m, lines = int(off[-1]) + 3, len(lengths)  # steps behind the last line
    loss, old, ref, target = steps(rng, m)
    adv = rng.standard_normal(m if per_row else lines).astype(np.float32)
    grad = rng.standard_normal(lines).astype(np.float32)
    job = Policy(rh, loss, old, ref if with_ref else None, target, adv, off, grad=grad)
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    job.check(got, "policy")
    assert (got["row_grad"][off[-1]:] == 0).all()
    for key in got:  # each output alone, the same bits
        assert np.array_equal(job.run({key: job.outputs()[key]})[key].get(), got[key]), key
    if off[-1] == m - 3:
        host = rh.policy_loss(loss, old, adv, off, target, ref if with_ref else None, 0.2, 0.28, 0.05, grad)
        for a, b in zip(host, (got["loss"], got["kl"], got["clipped"], got["row_grad"])):
            assert np.array_equal(a, b)


def test_policy_next_to_the_border(rh):
    """Steps on either side of the clipping's border by a unit of the last place: the side is that of 64 bits."""
    for low, high in ((0.2, 0.28), (0.0, 0.0), (1.0, 0.5), (0.25, np.float32(3e38))):
        for sign in (1.0, -1.0):
            edge = np.log1p(float(np.float32(high))) if sign > 0 else np.log1p(-float(np.float32(low))) if low < 1 else -30.0
            x = np.float32(2.5)
            near = [np.float32(x + np.float32(edge))]
            for _ in range(6):
                near.append(np.nextafter(near[-1], np.float32(100)))
            for _ in range(6):
                near.insert(0, np.nextafter(near[0], np.float32(-100)))
            old = np.array(near, np.float32)
            loss = np.full(old.size, x, np.float32)
            job = Policy(rh, loss, old, None, None, np.full(old.size, sign, np.float32), ac.offsets([1] * old.size), low, high, 0.0)
            job.per_row = False
            got = {k: v.get() for k, v in job.run(job.outputs()).items()}
            job.check(got, f"border {low} {high} {sign}")


def test_policy_extremes(rh):
    """Steps that do not count hold anything; an advantage of 0 takes nothing from an infinite ratio; ratios and
    divergences beyond 32 bits; equal policies; a line whose grad is 0."""
    nan, inf = np.nan, np.inf
    loss = np.array([1, nan, 0, 300, 2, 0.5, inf, 1e-30, 3, 0.25], np.float32)
    old = np.array([1, inf, 200, 0, 2, 0.5, nan, 0, nan, 0.25], np.float32)
    ref = np.array([1, nan, 0, 300, 2 + 2.0 ** -20, 0.5, 1, 0, 3, 80], np.float32)
    target = np.array([0, -1, 0, 0, 0, 0, -1, 0, 0, 0], np.int32)
    adv = np.array([1, nan, 0, 1, -2, 0.5, 1, 1, 1, -1], np.float32)
    off = ac.offsets([2, 2, 2, 2, 1, 1])
    grad = np.array([1, 1, 1, 1, 0, 1], np.float32)
    job = Policy(rh, loss, old, ref, target, adv, off, 0.2, 0.2, 0.1, grad)
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    want, tol = ac.policy64(loss, old, ref, target, adv, True, off, 0.2, 0.2, 0.1, grad)
    keep = np.array([0, 1, 2, 3, 5])
    for k in ("loss", "kl", "clipped"):
        tc.close(got[k][keep], want[k][keep], tol[k][keep], k)
    assert np.isnan(got["loss"][4]) and got["row_grad"][8] == 0  # a NaN that counts shows, its grad being 0 in no gradient
    tc.close(np.delete(got["row_grad"], 8), np.delete(want["row_grad"], 8), np.delete(tol["row_grad"], 8), "row_grad")
    # a ratio that 32 bits do not hold
    job = Policy(rh, np.array([0, 0], np.float32), np.array([200, 200], np.float32), None, None, np.array([-1, 1], np.float32),
                 ac.offsets([1, 1]), 0.2, 0.2, 0.0)
    job.per_row = False
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    assert got["loss"][0] == inf and got["row_grad"][0] == -inf
    assert abs(got["loss"][1] + 1.2) < 1e-6 and got["row_grad"][1] == 0
    # all steps masked, no lines, no steps
    z = np.zeros(5, np.float32)
    job = Policy(rh, z + nan, z, z, np.full(5, -1, np.int32), np.ones(1, np.float32), ac.offsets([5]))
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    assert all((v == 0).all() for v in got.values())
    job = Policy(rh, z, z, z, None, np.zeros(0, np.float32), np.zeros(1, np.int64))
    assert (job.run({"row_grad": job.outputs()["row_grad"]})["row_grad"].get() == 0).all()
    job = Policy(rh, z[:0], z[:0], None, None, np.ones(2, np.float32), np.zeros(3, np.int64))
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    assert (got["loss"] == 0).all() and (got["clipped"] == 0).all()


def test_small_divergences(rh):
    """e^t - t - 1 of tiny t, which a difference would lose."""
    t = np.concatenate([10.0 ** np.arange(-12.0, 1.5, 0.25), -(10.0 ** np.arange(-12.0, 1.5, 0.25)), [0.0, 1.0, -1.0, 60.0, -60.0]])
    loss = np.maximum(t, 0).astype(np.float32)
    ref = np.maximum(-t, 0).astype(np.float32)
    job = Policy(rh, loss, loss, ref, None, np.zeros(t.size, np.float32), ac.offsets([1] * t.size), beta=1.0)
    job.per_row = False
    job.check({k: v.get() for k, v in job.run(job.outputs()).items()}, "divergence")


def test_clamped_offsets(rh):
    """Offsets outside [0, m], and steps before the first line and behind the last: gradient 0 there."""
    rng = np.random.default_rng(3)
    m = 100
    loss, old, ref, target = steps(rng, m)
    adv = rng.standard_normal(3).astype(np.float32)
    for off in ([5, 20, 60, 90], [-7, 20, 60, 1 << 40], [30, 30, 30, 100]):
        inside = np.clip(off, 0, m)
        job = Policy(rh, loss, old, ref, target, adv, off)
        job.v = job.v[:5] + (inside,) + job.v[6:]
        job.check({k: v.get() for k, v in job.run(job.outputs()).items()}, str(off))
    pair = Preference(rh, loss, ref, target, [5, 40, 90])
    pair.check({k: v.get() for k, v in pair.run(pair.outputs()).items()}, "preference")
    # offsets that go backwards: every output is written with some number, and nothing behind it
    for off in ([90, 10, 50, 20], [1 << 50, -3, 200, 0]):
        job = Policy(rh, loss, old, ref, target, adv, off)
        job.run(job.outputs())["loss"].get()
        pair = Preference(rh, loss, ref, target, off[:3])
        for v in pair.run(pair.outputs()).values():
            v.get()


@pytest.mark.parametrize("lengths", [x for x in LENGTHS if len(x) > 1], ids=[i for i in IDS if not i.startswith("1x")])
@pytest.mark.parametrize("average,smoothing,with_ref", [(False, 0.0, True), (True, 0.1, True), (False, 0.5, False), (True, 1.0, True)])
def test_preference(rh, lengths, average, smoothing, with_ref):
    lengths = lengths[:len(lengths) // 2 * 2]
    rng = np.random.default_rng(len(lengths) + max(lengths) + 1)
    off = ac.offsets(lengths)
    m = int(off[-1]) + 5
    loss, _, ref, target = steps(rng, m)
    loss[target < 0] = np.nan
    grad = rng.standard_normal(len(lengths) // 2).astype(np.float32)
    job = Preference(rh, loss, ref if with_ref else None, target, off, 0.3, smoothing, average, grad)
    got = {k: v.get() for k, v in job.run(job.outputs()).items()}
    job.check(got, "preference")
    for key in got:
        assert np.array_equal(job.run({key: job.outputs()[key]})[key].get(), got[key]), key
    host = rh.preference_loss(loss, ref if with_ref else None, off, target, 0.3, smoothing, average, grad)
    for a, b in zip(host, (got["loss"], got["reward"].reshape(-1, 2), got["row_grad"])):
        assert np.array_equal(a, b)


def test_preference_extremes(rh):
    """Rewards far apart in both directions, equal lines, empty lines, and a pair whose grad is 0 and holds NaN."""
    loss = np.array([0, 500, 500, 0, 1, 1, 2, np.nan, 1, 0, 90, 0], np.float32)
    ref = np.zeros(12, np.float32)
    off = ac.offsets([1, 1, 1, 1, 1, 1, 1, 0, 1, 1, 1, 1])
    off[7:] = [7, 7, 8, 10, 11, 12]  # pair 3: one line empty, the other too; pair 4 holds the NaN
    grad = np.array([1, 1, 1, 1, 0, 1], np.float32)
    for smoothing in (0.0, 0.2):
        job = Preference(rh, loss, ref, None, off, 1.0, smoothing, False, grad)
        got = {k: v.get() for k, v in job.run(job.outputs()).items()}
        want, tol = ac.preference64(np.nan_to_num(loss, nan=0.0), ref, None, off, 1.0, smoothing, False, grad)
        odd = np.arange(6) == 4
        assert (got["row_grad"][off[8]:off[10]] == 0).all()
        for k in ("loss", "reward"):
            skip = odd if k == "loss" else np.repeat(odd, 2)
            tc.close(got[k][~skip], want[k][~skip], tol[k][~skip], k)
        rows = np.ones(12, bool)
        rows[off[8]:off[10]] = False
        tc.close(got["row_grad"][rows], want["row_grad"][rows], tol["row_grad"][rows], "row_grad")


def test_gradients_by_differences(rh):
    """Both losses' row gradients against differences of the formulas in 64 bits."""
    rng = np.random.default_rng(8)
    off = ac.offsets([9, 4, 6, 11])
    m = 30
    loss, old, ref, target = steps(rng, m)
    adv, grad = rng.standard_normal(4).astype(np.float32), rng.standard_normal(4).astype(np.float32)
    row = rh.policy_loss(loss, old, adv, off, target, ref, 0.2, 0.28, 0.5, grad)[3]
    pg = rng.standard_normal(2).astype(np.float32)
    prow = rh.preference_loss(loss, ref, off, target, 0.3, 0.1, True, pg)[2]

    def policy(x):
        return float((ac.policy64(x, old, ref, target, adv, False, off, 0.2, 0.28, 0.5)[0]["loss"] * grad).sum())

    def preference(x):
        return float((ac.preference64(x, ref, target, off, 0.3, 0.1, True)[0]["loss"] * pg).sum())

    for r in range(0, m, 3):
        x = loss.astype(np.float64)
        h = 1e-6
        lo, hi = x.copy(), x.copy()
        lo[r] -= h
        hi[r] += h
        assert abs((policy(hi) - policy(lo)) / (2 * h) - row[r]) < 1e-4 * (1 + abs(row[r]))
        assert abs((preference(hi) - preference(lo)) / (2 * h) - prow[r]) < 1e-5


def test_captured_and_on_two_streams(rh):
    from ppocr_rechead.hip import Stream, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(9)
    off = ac.offsets([50] * 40)
    loss, old, ref, target = steps(rng, 2000)
    a = Policy(rh, loss, old, ref, target, rng.standard_normal(40).astype(np.float32), off)
    b = Preference(rh, loss, ref, target, off)
    st, other = Stream(), Stream()
    oa, ob = a.outputs(), b.outputs()
    graph = _Graph(st, lambda: (a.run(oa, st.h), b.run(ob, st.h)))
    for _ in range(3):
        for v in (*oa.values(), *ob.values()):
            v.d.fill_bytes(0xA5)
        synchronize()
        oc = b.run(b.outputs(), other.h)
        graph.replay()
        other.synchronize()
        a.check({k: v.get() for k, v in oa.items()}, "replay")
        b.check({k: v.get() for k, v in ob.items()}, "replay")
        b.check({k: v.get() for k, v in oc.items()}, "beside it")
    graph.close()


def test_few_long_lines(rh):
    """Lines that several workgroups share: captured beside a call on another stream, in-bounds for any offsets, steps
    of no line cleared, a NaN kept to its line, and lines whose grad is 0."""
    from ppocr_rechead.hip import Stream, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(10)
    off = np.array([1000, 41000, 41003, 41003, 150000], np.int64)
    m = 150500
    loss, old, ref, target = steps(rng, m)
    adv, grad = rng.standard_normal(4).astype(np.float32), np.array([1, 2, 3, -0.5], np.float32)
    a = Policy(rh, loss, old, ref, target, adv, off, grad=grad)
    b = Preference(rh, loss, ref, target, off, 0.01, 0.1, True)
    st, other = Stream(), Stream()
    oa, ob = a.outputs(), b.outputs()
    graph = _Graph(st, lambda: (a.run(oa, st.h), b.run(ob, st.h)))
    for _ in range(3):
        for v in (*oa.values(), *ob.values()):
            v.d.fill_bytes(0xA5)
        synchronize()
        oc, od = b.run(b.outputs(), other.h), a.run(a.outputs(), other.h)
        graph.replay()
        other.synchronize()
        for job, o in ((a, oa), (b, ob), (b, oc), (a, od)):
            job.check({k: v.get() for k, v in o.items()}, "long lines")
    graph.close()
    for back in ([140000, 10, 90000, 20, 60000], [1 << 50, -3, 200, 0, 1 << 40]):
        a, b = Policy(rh, loss, old, ref, target, adv, back), Preference(rh, loss, ref, target, back)
        for o in (a.run(a.outputs()), b.run(b.outputs())):
            for v in o.values():
                v.get()
    bad, none = loss.copy(), np.array([1, 1, 1, 0], np.float32)
    bad[100000] = np.nan
    target[100000] = 3
    got = {k: v.get() for k, v in (lambda j: j.run(j.outputs()))(Policy(rh, bad, old, ref, target, adv, off, grad=none)).items()}
    want, tol = ac.policy64(loss, old, ref, target, adv, False, off, 0.2, 0.28, 0.05, none)
    assert np.isnan(got["loss"][3]) and (got["row_grad"][41003:] == 0).all()
    tc.close(got["loss"][:3], want["loss"][:3], tol["loss"][:3], "lines beside a NaN")
    tc.close(got["row_grad"][:41003], want["row_grad"][:41003], tol["row_grad"][:41003], "gradients beside a NaN")
