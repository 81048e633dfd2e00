"""8-bit caches that something else has filled: NaN codes, scales that are negative, subnormal or infinite, in appends and in attention; scales
of V from one end of float32 to the other in one sequence."""
import math

import numpy as np
import pytest

from scaled_case import Scaled, codes, values
from test_gpu_paged_append_scaled import Call, ragged
from test_gpu_paged_sdpa_scaled import expected, made, queries, run

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


# ---- attention --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (128, 16, 4), (128, 16, 1), (64, 8, 8), (80, 16, 16), (20, 16, 4)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_scale_that_is_not_finite_is_nan(hip, dtype, d, page, block, value):
    """Whoever sees the block gets NaN, whatever the sign of the scores that an infinite scale of K would give and whatever the codes; nobody else does."""
    lens, hkv, new, hq = [100, 100, 100, 40], 2, 3, 4
    p = made(71, lens, hkv, d, page, block, dtype)
    q = np.abs(queries(len(lens), new, hq, d))
    one = 1 if dtype == "i8" else 0x38
    for s, sign in ((0, 0), (1, 1)):  # scores of one sign in the block of K
        start = 20 - 20 % block
        for pos in range(start, start + block):
            r = p.row_at(s, pos, 0)
            p.codes[0][r:r + d] = (256 - one if dtype == "i8" else one | 128) if sign else one
    ref = expected(p, q, 0.2, lens)
    p.scales[0][p.scale_at(0, 20, 0)] = value
    p.scales[0][p.scale_at(1, 20, 0)] = value
    p.scales[1][p.scale_at(2, 20, 1)] = value
    got = run(hip, p, q, 0.2, lens)
    nan = np.zeros(ref.shape, bool)
    nan[0, :, :2] = nan[1, :, :2] = nan[2, :, 2:] = True
    assert np.array_equal(np.isnan(got), nan)
    assert np.max(np.abs(got[~nan] - ref[~nan])) <= 2e-5 * np.max(np.abs(ref[~nan]))


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 4, 1])
@pytest.mark.parametrize("size", [1e-37, 1e-33, 1e30, 1e35])
def test_queries_near_the_ends_of_float32(hip, dtype, block, size):
    """Scales of K bring the scores back: what scores are multiplied by goes through neither end."""
    lens, d = [150, 33], 128
    p = made(74, lens, 2, d, 16, block, dtype)
    for s, n in enumerate(lens):
        for pos in range(0, n, block):
            for h in range(2):
                p.scales[0][p.scale_at(s, pos, h)] /= np.float32(size)
    q = (queries(2, 2, 4, d) * np.float32(size)).astype(np.float32)
    got, ref = run(hip, p, q, 0.1, lens), expected(p, q, 0.1, lens)
    assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(ref))


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("d,block", [(64, 16), (128, 1), (64, 4), (20, 4)])
@pytest.mark.parametrize("large", [1e24, 1e30, 2.0 ** 108])
def test_scales_of_v_far_apart(hip, dtype, d, block, large):
    """One block of V has a scale that takes the products beyond float32's range under the factor that weights otherwise carry, and codes of 0 in half of its columns;
    the others are from 1e-36 to 1. Every output is compared by itself, with the sum of its terms' sizes. Scores are below 8: roundings of them move a
    weight by 3 x 8 log2(e) x 2^-24, the products' and the sums' add as much again, far below 2e-5."""
    n, hkv = 300, 2
    p = made(72, [n], hkv, d, 16, block, dtype)
    q = queries(1, 2, 4, d, std=0.3)
    rng = np.random.RandomState(9)
    for h in range(hkv):
        for pos in range(0, n, block):
            p.scales[0][p.scale_at(0, pos, h)] = 0.01
            p.scales[1][p.scale_at(0, pos, h)] = 10.0 ** rng.uniform(-36, -33) if h else 10.0 ** rng.uniform(-36, 0)
        p.scales[1][p.scale_at(0, 100, h)] = large
        for pos in range(100 - 100 % block, 100 - 100 % block + block):
            r = p.row_at(0, pos, h)
            p.codes[1][r:r + d // 2] = 0
    got, ref = run(hip, p, q, 0.05, [n]), expected(p, q, 0.05, [n])
    p.codes[1] = np.abs(np.clip(p.codes[1].view(np.int8).astype(np.int32), -127, 127)).astype(np.uint8) if dtype == "i8" else p.codes[1] & 127
    p.scales[1] = np.abs(p.scales[1])
    size = expected(p, q, 0.05, [n])
    assert np.all(np.isfinite(got)) and np.all(np.abs(got - ref) <= 2e-5 * size)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [1, 4, 16])
@pytest.mark.parametrize("low,high", [(0.01, 30.0), (1e-30, 1e-28), (1e20, 1e30), (1e-20, 1e20)])
def test_each_output_by_itself(hip, dtype, block, low, high):
    """Scales of any size and sign, each output against the sum of its own terms' sizes (scores stay below 60: 3 roundings of 60 log2(e) units of 2^-24
    and a few more of the products are within 2e-5)."""
    lens, hkv, d = [300, 40], 2, 64
    p = made(73, lens, hkv, d, 16, block, dtype)
    rng = np.random.RandomState(5)
    q = queries(2, 1, 4, d, std=0.5)
    for s, n in enumerate(lens):
        for pos in range(0, n, block):
            for h in range(hkv):
                p.scales[0][p.scale_at(s, pos, h)] = rng.uniform(0.001, 0.004) * rng.choice([-1, 1])
                p.scales[1][p.scale_at(s, pos, h)] = math.exp(rng.uniform(math.log(low), math.log(high))) * rng.choice([-1, 1, 1])
    got, ref = run(hip, p, q, 0.125, lens), expected(p, q, 0.125, lens)
    p.codes[1] = np.abs(np.clip(p.codes[1].view(np.int8).astype(np.int32), -127, 127)).astype(np.uint8) if dtype == "i8" else p.codes[1] & 127
    p.scales[1] = np.abs(p.scales[1])
    assert np.all(np.abs(got - ref) <= 2e-5 * expected(p, q, 0.125, lens))
