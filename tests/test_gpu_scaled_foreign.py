"""8-bit caches that something else has filled: NaN codes, scales that are negative, subnormal or infinite."""
import numpy as np
import pytest

from scaled_case import Scaled, codes, values
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


@PATHS
@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("had", [-0.5, -0.013, 1e-40, -1e-44, 0.0, np.inf, -np.inf, np.nan, 0.017, -3e38])
def test_scales_of_any_kind_before_the_tokens(hip, lead, dtype, had):
    """A block whose scale is no power of two, negative, subnormal or not finite gets zeros, small and large elements: what it held keeps its sign
    and its value to half a step of the scale that holds then, and so do the new elements; scales of one size or more stay as they are."""
    top = 127.0 if dtype == "i8" else 448.0
    for size in (0.0, 0.01, 1000.0):
        p = Scaled(64, 1, 1, 64, 16, 16, dtype, 1)
        rng = np.random.RandomState(7)
        for w in range(2):
            for pos in range(5):
                r = p.row_at(0, pos, 0)
                p.codes[w][r:r + 64] = codes(rng.uniform(-top, top, 64), dtype)
            p.scales[w][p.scale_at(0, 0, 0)] = had
        old = [np.stack([values(p.codes[w][p.row_at(0, pos, 0):][:64], dtype) for pos in range(5)]) for w in range(2)]
        device = p.upload()
        call = Call(p, 65, ragged([2], [5]), lead=lead)
        call.proj = (call.proj * np.float32(size)).astype(np.float32)
        call.run(hip, device)
        for w in range(2):
            x = call.proj[:, w * 64:(w + 1) * 64].astype(np.float64)
            now = p.scale_buffers[w].to_host()[p.scale_at(0, 0, 0)]
            got = p.buffers[w].to_host()
            held = np.stack([values(got[p.row_at(0, pos, 0):][:64], dtype) for pos in range(7)])
            if not np.isfinite(had):
                assert not np.isfinite(now)
                continue
            need = np.max(np.abs(x)) / top
            assert np.isfinite(now) and abs(float(now)) >= max(abs(float(np.float32(had))), need * (1 - 2.0 ** -20))
            if abs(float(np.float32(had))) >= 2 * need:
                assert now == np.float32(had)
            want = np.concatenate([old[w] * float(np.float32(had)), x])
            # half a step: of whole numbers 1/2; of e4m3 2^-4 of the number, 2^-10 where it is subnormal; and 2^-22 for quotients by scales that are no powers of two
            step = 0.5 * abs(float(now)) if dtype == "i8" else np.maximum(np.abs(want) * 2.0 ** -4, abs(float(now)) * 2.0 ** -10)
            assert np.all(np.abs(held * float(now) - want) <= step * (1 + 2.0 ** -10) + np.abs(want) * 2.0 ** -22), (size, w)
