"""Appends to 8-bit caches whose tokens do not ascend by one: what is left out behind the first that does not, in blocks of every kind of length and
over the cuts of a call, on the path of 128-bit accesses and element by element."""
import numpy as np
import pytest

from frankentorch_amd.device import DeviceBuffer
from paged_case import rotated
from scaled_case import Scaled
from test_gpu_paged_append_scaled import Call, same

pytestmark = pytest.mark.gpu

PATHS = pytest.mark.parametrize("lead", [0, 1], ids=["vectors", "elements"])  # of the operands


def by_the_rules(hip, p, places, left_out, lead):
    device = p.upload()
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    call = Call(p, 66, places, 2, 64, max_pos=2000, lead=lead)
    got = call.run(hip, device, bad)
    turned = Call(p, 66, places, 2, 64, max_pos=2000, lead=lead)
    keep = np.ones(len(places), bool)
    keep[left_out] = False
    call.proj, call.seqs, call.positions = call.proj[keep], call.seqs[keep], call.positions[keep]
    call.expect()
    same(p)
    assert bad.to_host()[0] == (min(left_out) if left_out else -1)
    # the queries of every token are rotated
    want = rotated(turned.heads(0, 2), turned.positions, turned.cos, turned.sin, 64, False, np.float32)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@PATHS
@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_behind_a_token_that_is_left_out(hip, lead, dtype):
    """What a call has of a block behind a token that is left out is left out as well, also where it would go on from the tokens before or from the one
    left out; the next block is not touched by that. Blocks of one position know only a place that comes twice."""
    twice = [(0, x) for x in (3, 4, 4, 5, 6, 16, 17)]
    gap = [(1, x) for x in (4, 6, 7, 5, 16)]
    back = [(2, x) for x in (5, 4, 5, 6, 32)]
    places = twice + gap + back
    p = Scaled(67, 3, 2, 64, 16, 16, dtype, 3).fill(68, [3, 4, 5])
    by_the_rules(hip, p, places, [2, 3, 4, 8, 9, 10, 13, 14, 15], lead)
    p = Scaled(67, 3, 2, 64, 16, 1, dtype, 3).fill(68, [3, 4, 5])
    places = twice + [(1, x) for x in (4, 6, 7, 16)] + [(2, x) for x in (5, 6, 6, 6, 7)]
    by_the_rules(hip, p, places, [2, 13, 14], lead)


@PATHS
@pytest.mark.parametrize("before", [0, 300, 1100])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_left_out_over_the_cuts(hip, lead, before, block):
    """The same in calls that are cut into 1, 4 or 32 tokens a wavefront: the rest of the block reaches over one cut or many."""
    p = Scaled(69, 2, 16, 64, 128, block, "i8", 10)
    first = [(0, i) for i in range(before)]
    rest = [(1, i) for i in (0, 1, 2, 4)] + [(1, i) for i in range(5, 2 * block + 3)]
    places = first + rest
    by_the_rules(hip, p, places, list(range(before + 3, before + 4 + block - 5)), lead)
