"""Decoding under adapters where the rows of a wave, the plan of the lines and the head's type are other ones than in the
small cases: ranks above 32 with many rows, slots in any order, and FP32 heads of the model's size."""
import numpy as np
import pytest

import adapt_common as ac
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
