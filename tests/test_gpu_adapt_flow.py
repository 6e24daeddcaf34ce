"""The entry points that adapt a head together, as a program uses them on one stream without a wait between
them: an adapter trained on sampled readings and on preferences under its merged weight, its gradients
clipped, then served beside the shared head."""
import ctypes

import numpy as np
import pytest

import adapt_common as ac
import train_common as tc
from train_common import F32

pytestmark = pytest.mark.gpu


class Step:
    """One training step of an adapter: merge, cross entropy, a loss over lines, and back to the clipped
    gradients of the adapter and of the bias."""

    def __init__(self, rh, rng, preference, n=900, k=120, rank=16, lines=6):
        self.rh, self.L, self.preference = rh, rh._lib.lib(), preference
        self.shape = (n, k, rank)
        self.scale, self.most = 1.5, 0.05
        lengths = rng.integers(5, 60, lines)
        self.off = ac.offsets(lengths)
        m = self.m = int(self.off[-1])
        a, w, b, to = tc.head_inputs(rng, m, n, k)
        self.v = {"a": a, "w": w, "b": b, "down": (rng.standard_normal((rank, k)) / np.sqrt(k)).astype(np.float32),
                  "up": (rng.standard_normal((n, rank)) * 0.05).astype(np.float32),
                  "target": np.where(rng.random(m) < 0.1, -1, to).astype(np.int32), "off": self.off,
                  "old": (rng.random(m) * 3).astype(np.float32), "ref": (rng.random(m) * 3).astype(np.float32),
                  "adv": rng.standard_normal(lines).astype(np.float32)}
        self.units = lines // 2 if preference else lines
        self.v["grad"] = np.full(self.units, 1.0 / self.units, np.float32)
        self.d = {key: tc.up(x) for key, x in self.v.items()}
        shapes = {"merged": (n, k), "loss": (m,), "lse": (m,), "lines": (self.units,), "rows": (m,), "da": (m, k), "dw": (n, k),
                  "db": (n,), "ddown": (rank, k), "dup": (n, rank), "norm": (1,)}
        self.o = {key: tc.Out(s, np.float32) for key, s in shapes.items()}
        self.grads = ["ddown", "dup", "db"]
        P, I, T = ctypes.c_void_p * 3, ctypes.c_int64 * 3, ctypes.c_int32 * 3
        self.tables = (P(*[self.o[g].p.value for g in self.grads]), None, I(rank * k, n * rank, n), T(0, 0, 0))
        self.bytes = max(self.L.ppocr_xent_workspace_bytes(m, n, k, 0), self.L.ppocr_ra_merge_workspace_bytes(n, k, rank),
                         self.L.ppocr_grad_clip_workspace_bytes(self.tables[2], 3))
        self.ws = tc.Out((self.bytes,), np.uint8)  # one for all of them in turn

    def run(self, st):
        L, d, o, check = self.L, {k: v.p for k, v in self.d.items()}, {k: v.p for k, v in self.o.items()}, self.rh._check
        n, k, rank = self.shape
        m, ws = self.m, (self.ws.p, self.bytes, st)
        low_rank = (n, k, rank, self.scale, F32)
        check(L.ppocr_ra_merge_dev(d["w"], d["down"], d["up"], *low_rank, o["merged"], st))
        check(L.ppocr_xent_forward_dev(d["a"], o["merged"], d["b"], d["target"], m, n, k, F32, o["loss"], o["lse"], *ws))
        if self.preference:
            check(L.ppocr_preference_loss_dev(o["loss"], d["ref"], d["target"], d["off"], self.units, m, 0.2, 0.1, 1, d["grad"],
                                              o["lines"], None, o["rows"], st))
        else:
            check(L.ppocr_policy_loss_dev(o["loss"], d["old"], d["ref"], d["target"], d["adv"], 0, d["off"], self.units, m, 0.2,
                                          0.28, 0.1, d["grad"], o["lines"], None, None, o["rows"], st))
        check(L.ppocr_xent_backward_dev(d["a"], o["merged"], d["b"], d["target"], o["lse"], o["rows"], m, n, k, F32, o["da"],
                                        o["dw"], o["db"], *ws))
        check(L.ppocr_ra_merge_backward_dev(o["dw"], d["down"], d["up"], *low_rank, o["ddown"], o["dup"], *ws))
        check(L.ppocr_grad_clip_dev(*self.tables, 3, self.most, o["norm"], *ws))

    def expect(self, down=None, up=None, b=None):
        """(the mean loss, the clipped gradients, their norm before) in 64 bits."""
        v = self.v
        down, up, b = (v[k].astype(np.float64) if x is None else x for k, x in (("down", down), ("up", up), ("b", b)))
        w = v["w"].astype(np.float64) + self.scale * (up @ down)
        ci, q, lq, some = tc.teacher64(self.m, self.shape[0], v["target"])
        r, *_ = tc.loss64(v["a"], w, b, ci, q, lq, some)
        if self.preference:
            out, _ = ac.preference64(r["loss"], v["ref"], v["target"], self.off, 0.2, 0.1, True, v["grad"])
        else:
            out, _ = ac.policy64(r["loss"], v["old"], v["ref"], v["target"], v["adv"], False, self.off, 0.2, 0.28, 0.1, v["grad"])
        g, *_ = tc.loss64(v["a"], w, b, ci, q, lq, some, grad=out["row_grad"])
        raw = {"ddown": self.scale * (up.T @ g["dw"]), "dup": self.scale * (g["dw"] @ down.T), "db": g["db"]}
        norm = np.sqrt(sum((x ** 2).sum() for x in raw.values()))
        return float((out["loss"] * v["grad"]).sum()), {k: x * min(1.0, self.most / norm) for k, x in raw.items()}, norm, raw


@pytest.mark.parametrize("preference", [False, True], ids=["policy", "preference"])
def test_training_step(rh, preference):
    """The whole chain against 64 bits, as single calls and as a graph replayed between other work; its
    gradients also against differences of the loss."""
    from ppocr_rechead.hip import Stream, synchronize
    from test_gpu_graph_replay import _Graph
    rng = np.random.default_rng(20 + preference)
    job, other = Step(rh, rng, preference), Step(rh, rng, not preference, lines=4)
    st = Stream()
    synchronize()

    def check():
        loss, want, norm, _ = job.expect()
        got = {k: v.get() for k, v in job.o.items()}
        job.ws.get()
        assert abs(float((got["lines"].astype(np.float64) * job.v["grad"]).sum()) - loss) < 2e-5 * (1 + abs(loss))
        assert abs(got["norm"][0] - norm) < 2e-5 * norm
        for key in job.grads:
            # every stage's own error is below 4e-6 of its output's norm (their tests); five stages
            err = np.linalg.norm(got[key] - want[key]) / np.linalg.norm(want[key])
            print(f"  {key}: {err:.1e} of the norm", flush=True)
            assert err < 2.5e-5, key
        return got

    job.run(st.h)
    st.synchronize()
    first = check()
    graph = _Graph(st, lambda: job.run(st.h))
    for _ in range(3):
        for v in job.o.values():
            v.d.fill_bytes(0xA5)
        other.run(None)
        synchronize()
        graph.replay()
        again = check()
        for key in first:
            assert np.array_equal(first[key], again[key]), key
    graph.close()
    # differences of the loss in 64 bits by single values of the adapter and of the bias
    *_, raw = job.expect()
    for key, name in (("ddown", "down"), ("dup", "up"), ("db", "b")):
        x = job.v[name].astype(np.float64)
        for at in rng.permutation(np.argwhere(np.abs(raw[key]) > 0.1 * np.abs(raw[key]).max()))[:3]:
            at, h = tuple(at), 1e-5
            lo, hi = x.copy(), x.copy()
            lo[at] -= h
            hi[at] += h
            diff = (job.expect(**{name: hi})[0] - job.expect(**{name: lo})[0]) / (2 * h)
            assert abs(diff - raw[key][at]) < 1e-3 * np.abs(raw[key]).max(), (key, at)


def test_a_trained_adapter_is_served(rh):
    """The adapter beside the shared head gives the logits of its merged weight, from the same tensors, and of two
    lines of one page only the one that names it."""
    from ppocr_rechead.hip import DeviceArray, Stream
    rng = np.random.default_rng(30)
    job = Step(rh, rng, False)
    n, k, rank = job.shape
    head = rh.RecHead(w_t=job.v["w"], bias=job.v["b"])
    served = rh.AdaptedHead(head, 3, 16)
    st = Stream()
    L = rh._lib.lib()
    job.run(st.h)
    # the slot is set on the stream that the training ran on, and read behind it
    rh._check(L.ppocr_ra_set_dev(served.handle, 2, job.d["down"].p, job.d["up"].p, rank, job.scale, F32, st.h))
    off = np.array([0, 40, job.m], np.int64)
    slot = np.array([2, -1], np.int32)
    doff, dslot, z = tc.up(off), tc.up(slot), DeviceArray((job.m, n), np.float32)
    rh._check(L.ppocr_ra_logits_dev(served.handle, job.d["a"].p, job.m, doff.p, 2, dslot.p, z.p, None, 0, st.h))
    st.synchronize()
    z = z.numpy()
    merged = rh.RecHead(w_t=job.o["merged"].get(), bias=job.v["b"])
    assert np.abs(z[:40] - merged.logits(job.v["a"][:40])).max() < 1e-4
    assert np.abs(z[40:] - head.logits(job.v["a"][40:])).max() < 1e-4
    assert np.abs(z[:40] - head.logits(job.v["a"][:40])).max() > 1e-2
    text = served.decode_lines(job.v["a"], off, slot)
    assert np.array_equal(text["idx"], z.argmax(axis=1))
