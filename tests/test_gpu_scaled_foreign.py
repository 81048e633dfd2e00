"""8-bit caches that something else has filled: NaN codes."""
import numpy as np
import pytest

from scaled_case import Scaled
from test_gpu_paged_append_scaled import Call, ragged

pytestmark = pytest.mark.gpu


# ---- appends ----------------------------------------------------------------------------------------------------------------

PATHS = pytest.mark.parametrize("lead", [0, 1], ids=["vectors", "elements"])  # of the operands: by 128 bits, or element by element


@PATHS
def test_nan_codes_stay_when_their_block_grows(hip, lead):
    """Of the NaN codes (whichever sign) before the tokens, each is one afterwards; all else is as by the rules."""
    p = Scaled(61, 1, 2, 64, 16, 8, "e4m3", 2).fill(62, [13])
    for which, pos, h, c, code in ((0, 8, 0, 3, 127), (0, 12, 1, 60, 255), (1, 9, 0, 0, 255), (1, 12, 1, 63, 127)):
        p.codes[which][p.row_at(0, pos, h) + c] = code
    device = p.upload()
    held = [(x & 127) == 127 for x in p.codes]
    call = Call(p, 63, ragged([2], [13]), std=1000.0, lead=lead)  # every scale grows
    had = [p.scales[w][p.scale_at(0, 13, h)] for w in range(2) for h in range(2)]
    call.run(hip, device)
    with np.errstate(invalid="ignore"):
        call.expect()
    assert all(p.scales[w][p.scale_at(0, 13, h)] > x for (w, h), x in zip(((0, 0), (0, 1), (1, 0), (1, 1)), had))
    for w in range(2):
        got = p.buffers[w].to_host()
        rows = [p.row_at(0, pos, h) for pos in range(15) for h in range(2)]
        at = np.concatenate([np.arange(r, r + 64) for r in rows])
        before = np.concatenate([np.arange(p.row_at(0, pos, h), p.row_at(0, pos, h) + 64) for pos in range(13) for h in range(2)])
        nan = np.zeros(got.shape, bool)
        nan[before] = held[w][before]
        assert nan.sum() == 2 and np.all((got[nan] & 127) == 127)
        rest = at[~nan[at]]
        zero = lambda x: np.where(x == 128, 0, x)
        assert np.array_equal(zero(got[rest]), zero(p.codes[w][rest]))
        assert np.array_equal(p.scale_buffers[w].to_host(), p.scales[w], equal_nan=True)
