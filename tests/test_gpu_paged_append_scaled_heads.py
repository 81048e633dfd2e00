"""Appends to 8-bit caches with short heads, of which a wavefront has many side by side, and with blocks far longer than a wavefront holds: codes, scales
and queries bit for bit by the rules."""
import numpy as np
import pytest

from frankentorch_amd.device import DeviceBuffer
from scaled_case import Scaled
from test_gpu_paged_append_scaled import Call, ragged, same

pytestmark = pytest.mark.gpu


def by_the_rules(hip, p, counts, starts, hq, rotary, inter):
    device = p.upload()
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    call = Call(p, 103, ragged(counts, starts), hq, rotary, inter, 3000 if rotary else 0)
    got, want = call.run(hip, device, bad), call.expect()
    same(p)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32)) and bad.to_host()[0] == -1


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 104, 248])
@pytest.mark.parametrize("block", [1, 4, 16, 96])
@pytest.mark.parametrize("dtype,inter", [("i8", False), ("e4m3", True)])
def test_short_heads(hip, d, block, dtype, inter):
    counts, starts = [130, 1, 47], [5, 16, 95]
    for rotary in (d, 8):
        p = Scaled(101, 3, 3, d, 96, block, dtype, 2).fill(102, starts)
        by_the_rules(hip, p, counts, starts, 5, rotary, inter)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("counts,starts", [([1, 1], [1999, 2500]), ([700, 3], [1300, 2560]), ([2100], [400])], ids=str)
def test_long_blocks(hip, dtype, counts, starts):
    """One scale for a page of 2560 positions: few tokens behind many, which may have to be brought to a new scale, and runs longer than what is held."""
    p = Scaled(104, len(counts), 2, 64, 2560, 2560, dtype, 2).fill(105, starts)
    by_the_rules(hip, p, counts, starts, 2, 64, False)
