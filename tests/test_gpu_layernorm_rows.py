"""LayerNorm over more rows than its grids hold at once, so that every workgroup takes several, reading
ahead and keeping its weights."""
import numpy as np
import pytest

import train_common as tc
from test_gpu_layernorm import Job, inputs
from train_common import BF16, F32

pytestmark = pytest.mark.gpu

DT = pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])


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
