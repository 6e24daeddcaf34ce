"""LayerNorm over more rows than its grids hold at once, so that every workgroup takes several, reading
ahead and keeping its weights: one shape and more for each number of lanes a row is given."""
import numpy as np
import pytest

import train_common as tc
from test_gpu_layernorm import Job, inputs, norm64, tolerances
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

DT = pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
# rows that a grid takes at once, forward: 32768 up to 128 columns, 8192 up to 512, 5120 up to 1024,
# 2048, 1280, 512, 256 up to 2048, 4096, 8192, 16384; backward fewer
SHAPES = [(70001, 120), (33000, 77), (17003, 260), (11001, 1000), (4500, 2048), (2701, 4096), (1100, 8192), (530, 8193),
          (601, 16384)]


@pytest.mark.parametrize("m,d", [(33000, 77), (11001, 1000), (2701, 4096), (1100, 8192), (601, 16384)])
@DT
def test_in_place_where_workgroups_take_several_rows(rh, m, d, dt):
    """y over x, dx over dy and dx over x: the bits of outputs of their own."""
    from ppocr_rechead.hip import synchronize
    rng = np.random.default_rng(m)
    (x, _), (dy, _), w, b = inputs(rng, m, d, dt)
    want = Job(rh, x, w, b, dy, 1e-5, dt).step()
    for over in ("dy", "x"):
        job = Job(rh, x, w, b, dy, 1e-5, dt)
        o = job.outputs()
        job.forward(o)
        o["dx"] = getattr(job, over)
        job.backward(o)
        synchronize()
        assert np.array_equal(o["dx"].numpy(), want["dx"]), over
        assert np.array_equal(o["dw"].get(), want["dw"]) and np.array_equal(o["db"].get(), want["db"]), over
    job = Job(rh, x, w, b, dy, 1e-5, dt)
    job.forward({"y": job.x})
    synchronize()
    assert np.array_equal(job.x.numpy(), want["y"])


@pytest.mark.parametrize("m,d", SHAPES)
@DT
def test_several_rows_a_workgroup(rh, m, d, dt):
    rng = np.random.default_rng(m + d)
    (x, xv), (dy, dyv), w, b = inputs(rng, m, d, dt)
    print(f"layernorm m={m} d={d} dt={dt}", flush=True)
    ref, h, t = norm64(xv, w, b, 1e-5, dyv)
    tol = tolerances(xv, w, b, dyv, ref, h, t, dt)
    for shift in (0, 1):  # rows that start on a vector boundary, and not
        got = Job(rh, x, w, b, dy, 1e-5, dt, shift).step()
        for key in ("mean", "rstd", "y", "dx", "dw", "db"):
            tc.close(got[key], ref[key], tol[key], f"{key} shift {shift}")
