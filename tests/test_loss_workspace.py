"""Sizes of the losses' workspaces where one side is far longer than the other; no device is needed."""
import pytest


@pytest.mark.parametrize("m,n,k", [(2000, 600_000, 120), (8192, 1 << 21, 256), (1 << 21, 2000, 120), (1, 1 << 20, 64),
                                   (1 << 22, 32, 256)])
@pytest.mark.parametrize("dt", [0, 1], ids=["f32", "bf16"])
def test_long_and_short_sides(rh, m, n, k, dt):
    """No more than the records and a few sums of each output, however many chunks the other side's
    stream could be cut into: per row and class, records of at most 2 x 2 x 2 bytes a value (k to a
    multiple of 64) and 14 more, sums of 4 bytes a value each, here up to 8 of them on average, and
    1 GB for the chunks of whichever side is short."""
    pieces = (k + 63) // 64 * 64
    most = (m + n) * (8 * pieces + 14 + 8 * 4 * pieces) + (1 << 30)
    lists = (m + 31) // 32 * (32 * 8 + 2 * ((n + 127) // 128 + 1))
    assert rh._lib.lib().ppocr_xent_workspace_bytes(m, n, k, dt) < most + lists
