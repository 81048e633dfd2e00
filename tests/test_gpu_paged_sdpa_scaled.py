"""Attention over a cache of 8-bit numbers against the definition in 64 bits over the values that the codes and scales stand for."""
import math

import numpy as np
import pytest

from conftest import TOL_GEMM_F32, rel_err
from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer, Stream
from paged_case import attention
from scaled_case import Scaled, values

pytestmark = pytest.mark.gpu


def queries(seqs, new, hq, d, seed=3, std=1.5):
    return synth.normal(seed, "q", (seqs, new, hq, d), 0.0, std)


def run(hip, p, q, scale, lens, max_len=None, bad=None, table=None, stream=None):
    device = p.upload()
    desc = hip.paged_sdpa_desc(p.cache, q.shape[2], q.shape[1], max_len)
    out = DeviceBuffer.from_host(np.full(q.shape, 7.0, np.float32))
    hip.paged_sdpa_scaled(p.cache, p.sc, desc, scale, DeviceBuffer.from_host(q), *device, p.dev_table if table is None else DeviceBuffer.from_host(table),
                          DeviceBuffer.from_host(np.array(lens, np.int32)), out, bad_index=bad, stream=stream)
    hip.synchronize()
    return out.to_host()


def made(seed, lens, hkv, d, page, block, dtype, room=1, **kw):
    return Scaled(seed, len(lens), hkv, d, page, block, dtype, max(-(-max(x, 0) // page) for x in lens) + room, **kw).fill(seed + 1, lens)


def expected(p, q, scale, lens):
    k, v = ([p.rows(w, s, max(n, 0)) for s, n in enumerate(lens)] for w in range(2))
    return attention(q, k, v, scale, lens)


# (lens, hq, hkv, new, d, page, block, dtype)
CASES = [
    ([1], 1, 1, 1, 64, 16, 16, "e4m3"), ([0, 1, 2], 2, 2, 1, 64, 16, 16, "i8"), ([31, 32, 33], 4, 2, 1, 64, 16, 16, "e4m3"), ([15, 16, 17, 0, 5], 8, 1, 1, 128, 16, 16, "i8"),
    ([63, 64, 65, 127, 128, 129], 6, 2, 1, 64, 32, 32, "e4m3"), ([255, 256, 257], 8, 8, 1, 128, 64, 16, "i8"), ([300, 7, 0, 1], 12, 12, 1, 64, 16, 16, "e4m3"),
    ([1000, 3], 8, 2, 1, 128, 128, 64, "i8"), ([2500, 1, 900], 32, 8, 1, 128, 16, 16, "e4m3"), ([4099], 8, 1, 1, 64, 16, 16, "i8"), ([3000, 2999], 4, 4, 1, 128, 48, 48, "e4m3"),
    # several new tokens: the first of them may see nothing
    ([0, 1, 3, 4, 5, 8, 40], 4, 2, 4, 64, 16, 16, "e4m3"), ([7, 8, 9, 600], 8, 2, 8, 128, 16, 16, "i8"), ([2, 33, 700], 5, 1, 7, 64, 16, 16, "e4m3"),
    # more than 16 query rows on a K/V head
    ([200, 17, 1100], 17, 1, 1, 64, 16, 16, "i8"), ([400, 31], 32, 1, 4, 128, 16, 16, "e4m3"), ([77, 900], 24, 2, 3, 64, 16, 16, "i8"),
    # a scale a token, and blocks that are no multiples of 16
    ([200, 33], 4, 2, 1, 128, 16, 1, "e4m3"), ([200, 33], 4, 2, 1, 64, 32, 1, "i8"), ([700, 5], 8, 2, 4, 128, 32, 2, "i8"), ([130, 41], 4, 4, 1, 128, 48, 24, "e4m3"),
    ([90, 300], 2, 1, 1, 256, 16, 4, "i8"), ([90, 300], 4, 2, 2, 64, 64, 8, "e4m3"), ([65, 64], 2, 1, 1, 128, 48, 3, "i8"),
    # head sizes, pages that are no multiple of anything
    ([70, 1, 40], 4, 2, 1, 32, 16, 16, "i8"), ([70, 300], 4, 4, 2, 80, 16, 16, "e4m3"), ([70, 300], 4, 2, 1, 96, 16, 1, "i8"), ([90, 333], 4, 2, 1, 256, 16, 16, "e4m3"),
    ([90, 333, 2], 4, 1, 3, 256, 32, 32, "i8"), ([260], 3, 1, 1, 208, 16, 16, "e4m3"), ([45, 130], 2, 1, 1, 40, 16, 16, "i8"), ([45, 130], 2, 1, 1, 20, 16, 8, "e4m3"),
    ([45, 130], 4, 2, 2, 7, 16, 16, "i8"), ([33], 1, 1, 1, 1, 16, 16, "e4m3"), ([100, 65, 1], 4, 2, 1, 64, 1, 1, "i8"), ([100, 65, 3], 4, 2, 2, 128, 5, 5, "e4m3"),
    ([100, 650], 4, 2, 1, 64, 24, 12, "i8"), ([777, 20], 8, 2, 1, 128, 40, 40, "e4m3"), ([300, 299], 4, 4, 1, 64, 7, 7, "i8"), ([100, 650], 16, 2, 4, 80, 8, 8, "e4m3"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(hip, case):
    lens, hq, hkv, new, d, page, block, dtype = case
    p = made(11, lens, hkv, d, page, block, dtype)
    q, scale = queries(len(lens), new, hq, d), 1.0 / math.sqrt(d)
    got, ref = run(hip, p, q, scale, lens), expected(p, q, scale, lens)
    assert rel_err(got, ref) <= TOL_GEMM_F32
    assert np.all(got[ref == 0] == 0)  # a query that sees nothing gives zeros
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, scale, lens).view(np.uint32))  # and runs repeat


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("pad,lead,heads_inside,scale_pad", [(0, 0, True, 0), (16, 0, False, 3), (16, 32, True, 1), (3, 0, False, 0), (0, 1, False, 0), (8, 8, True, 0), (1, 5, True, 2)])
def test_layouts_and_alignments(hip, dtype, pad, lead, heads_inside, scale_pad):
    lens, hq, hkv, new, d = [130, 0, 33, 700], 8, 2, 2, 64
    p = made(12, lens, hkv, d, 16, 16, dtype, pad=pad, lead=lead, heads_inside=heads_inside, scale_pad=scale_pad)
    q = queries(len(lens), new, hq, d)
    assert rel_err(run(hip, p, q, 0.2, lens), expected(p, q, 0.2, lens)) <= TOL_GEMM_F32


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [1, 16])
def test_scales_of_any_size(hip, dtype, block):
    """Scales that are no powers of two, negative, zero, very small and very large in V, against each output by itself."""
    lens, hkv, d = [300, 40], 2, 64
    p = made(13, lens, hkv, d, 16, block, dtype)
    rng = np.random.RandomState(5)
    q, scale = queries(2, 1, 4, d, std=0.5), 0.125
    for low, high in ((0.01, 30.0), (1e-30, 1e-28), (1e20, 1e30)):
        for s, n in enumerate(lens):
            for pos in range(0, n, block):
                for h in range(hkv):
                    p.scales[0][p.scale_at(s, pos, h)] = rng.uniform(0.005, 0.02) * rng.choice([-1, 1])
                    p.scales[1][p.scale_at(s, pos, h)] = math.exp(rng.uniform(math.log(low), math.log(high))) * rng.choice([-1, 0, 1, 1])
        got, ref = run(hip, p, q, scale, lens), expected(p, q, scale, lens)
        assert rel_err(got, ref) <= TOL_GEMM_F32, (low, high)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128, 20])
def test_a_scale_that_is_not_finite(hip, dtype, d):
    """A NaN scale of K or V makes what sees its block NaN and nothing else, also where only the later of the new tokens see it."""
    lens, hkv, new, hq = [100, 64, 50, 50, 35], 2, 4, 4
    p = made(14, lens, hkv, d, 16, 16 if d != 20 else 4, dtype)
    q = queries(len(lens), new, hq, d)
    ref = expected(p, q, 0.2, lens)
    p.scales[0][p.scale_at(0, 20, 0)] = np.nan   # all queries of heads 0, 1 of sequence 0
    p.scales[1][p.scale_at(1, 40, 1)] = np.inf   # heads 2, 3 of sequence 1
    p.scales[1][p.scale_at(2, 48, 0)] = np.nan   # positions 48, 49: the third and fourth query of heads 0, 1 of sequence 2
    p.scales[0][p.scale_at(3, 48, 1)] = np.nan   # the same of heads 2, 3 of sequence 3
    got = run(hip, p, q, 0.2, lens)
    nan = np.zeros(ref.shape, bool)
    nan[0, :, :2] = nan[2, 2:, :2] = nan[3, 2:, 2:] = True
    # (infinite: the codes' signs make it +-inf or NaN; not finite either way)
    fine = ~nan
    fine[1, :, 2:] = False
    assert np.all(np.isnan(got[nan])) and not np.any(np.isfinite(got[1, :, 2:]))
    assert rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32


def test_nan_codes(hip):
    """A NaN code of e4m3 in V reaches the outputs of its column, in K whatever sees the key; only of queries that see it."""
    lens, hkv, d, new = [40, 40, 90], 1, 64, 3
    p = made(15, lens, hkv, d, 16, 16, "e4m3")
    q = queries(3, new, 2, d)
    ref = expected(p, q, 0.2, lens)
    p.codes[1][p.row_at(0, 39, 0) + 5] = 127   # seen by the last query alone
    p.codes[0][p.row_at(1, 38, 0) + 9] = 255   # by the last two
    p.codes[1][p.row_at(2, 3, 0) + 60] = 255   # by all
    got = run(hip, p, q, 0.2, lens)
    nan = np.zeros(ref.shape, bool)
    nan[0, 2, :, 5] = nan[1, 1:] = nan[2, :, :, 60] = True
    assert np.array_equal(np.isnan(got), nan)
    assert rel_err(got[~nan], ref[~nan]) <= TOL_GEMM_F32


def test_what_is_invalid_is_reported(hip):
    lens, hkv, d = [40, 200, 30, 60, 80], 2, 64
    p = made(16, lens, hkv, d, 16, 16, "i8")
    q = queries(5, 1, 4, d)
    ref = expected(p, q, 0.2, lens)
    table = p.table.copy()
    table[1, 5], table[3, 0] = 9999, -1
    bad = DeviceBuffer.from_host(np.array([0], np.int64))
    got = run(hip, p, q, 0.2, [40, 200, -1, 60, 80], bad=bad, table=table)
    assert bad.to_host()[0] == 1
    assert np.all(np.isnan(got[[1, 2, 3]])) and rel_err(got[[0, 4]], ref[[0, 4]]) <= TOL_GEMM_F32
    got = run(hip, p, q, 0.2, [40, 200, 30, 60, 80], max_len=80, bad=bad)
    assert bad.to_host()[0] == 1 and np.all(np.isnan(got[1])) and rel_err(got[[0, 2, 3, 4]], ref[[0, 2, 3, 4]]) <= TOL_GEMM_F32


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e3, 1e25])
def test_queries_of_any_size(hip, dtype, size):
    """Queries are cut into parts after a power of two: sizes far from one, with scales of K that bring the scores back."""
    lens, d = [150, 33], 128
    p = made(17, lens, 2, d, 16, 16, dtype)
    for s, n in enumerate(lens):
        for pos in range(0, n, 16):
            for h in range(2):
                p.scales[0][p.scale_at(s, pos, h)] /= np.float32(size)
    q = (queries(2, 2, 4, d) * np.float32(size)).astype(np.float32)
    assert rel_err(run(hip, p, q, 0.1, lens), expected(p, q, 0.1, lens)) <= TOL_GEMM_F32


def test_queries_that_are_not_finite(hip):
    lens, d = [150, 33], 64
    p = made(18, lens, 2, d, 16, 16, "e4m3")
    q = queries(2, 2, 4, d)
    ref = expected(p, q, 0.2, lens)
    q[0, 0, 1, 3], q[1, 1, 2, 5] = np.nan, np.inf
    got = run(hip, p, q, 0.2, lens)
    nan = np.zeros(ref.shape, bool)
    nan[0, 0, 1] = nan[1, 1, 2] = True
    assert np.all(np.isnan(got[nan])) and rel_err(got[~nan], ref[~nan]) <= TOL_GEMM_F32


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_small_weights_alone(hip, dtype):
    """Outputs that V leaves to keys far below the heaviest ones, each against the sum of its terms' sizes (a column has about three
    terms, whose signs may nearly cancel). Three roundings of a score of up to 80 / ln 2 = 115 in units of log2 move a weight by up to
    3 * 115 * 2^-24 * ln 2 = 1.4e-5 of itself, exp2 and the products by a few 2^-24 more: 2e-5."""
    n, d = 200, 64
    p = made(19, [n], 1, d, 16, 1, dtype)
    q = np.zeros((1, 1, 1, d), np.float32)
    q[..., 0] = 1.0
    for pos in range(n):  # key `pos` scores -pos / 2.5: down to -80
        r = p.row_at(0, pos, 0)
        p.codes[0][r:r + d] = 0
        p.codes[0][r] = 0xff if dtype == "i8" else 0xb8  # -1
        p.scales[0][p.scale_at(0, pos, 0)] = pos / 2.5
        r = p.row_at(0, pos, 0)
        column = pos * d // n
        keep = p.codes[1][r + column] | 1
        p.codes[1][r:r + d] = 0
        p.codes[1][r + column] = keep if keep & 127 != 127 else 1  # each column of V is held by a few keys
    got, ref = run(hip, p, q, 1.0, [n]), expected(p, q, 1.0, [n])
    p.codes[1] = np.abs(p.codes[1].view(np.int8)).view(np.uint8) if dtype == "i8" else p.codes[1] & 127
    assert np.all(np.abs(got - ref) <= 2e-5 * expected(p, q, 1.0, [n]))


def test_streams_and_graphs(hip):
    """One captured call serves every length up to max_len: replays on another stream, between eager calls, against eager ones."""
    from frankentorch_amd import _lib
    from frankentorch_amd.core import check
    from test_gpu_stream_scratch import Graph

    lens, d = [600, 33, 250, 1], 128
    p = made(20, lens, 2, d, 16, 16, "e4m3")
    device = p.upload()
    q = queries(4, 1, 8, d)
    desc = hip.paged_sdpa_desc(p.cache, 8, 1, 640)
    dq, dl = DeviceBuffer.from_host(q), DeviceBuffer.from_host(np.array(lens, np.int32))
    outs = [DeviceBuffer(q.shape) for _ in range(2)]
    work = [hip.paged_sdpa_scaled_workspace(p.cache, p.sc, desc) for _ in range(2)]
    home, side = Stream(), Stream()

    def call(i, stream):
        hip.paged_sdpa_scaled(p.cache, p.sc, desc, 0.1, dq, *device, p.dev_table, dl, outs[i], workspace=work[i], stream=stream)

    call(0, home.handle)
    home.synchronize()
    graph = Graph(home, lambda stream: call(0, stream))
    for now in ([600, 33, 250, 1], [1, 0, 600, 17], [128, 129, 255, 640 - 16], [600, 600 - 1, 250, 1]):
        now = [min(a, b) for a, b in zip(now, lens)]
        check(_lib.load().fth_memcpy_h2d(dl.ptr, np.array(now, np.int32).ctypes.data, 16))
        graph.replay(side)
        side.synchronize()
        call(1, home.handle)
        home.synchronize()
        got = [o.to_host() for o in outs]
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
        assert rel_err(got[0], expected(p, q, 0.1, now)) <= TOL_GEMM_F32
    graph.free()


def test_large_batches_in_even_shares(hip):
    """A batch that fills the chip: long and short sequences cut end to end."""
    lens = [1 + (i * 7919) % 9000 for i in range(40)]
    hq, hkv, d = 8, 8, 128
    for dtype, block in (("e4m3", 16), ("i8", 1)):
        p = Scaled(21, len(lens), hkv, d, 16, block, dtype, -(-max(lens) // 16))
        rng = np.random.RandomState(3)
        p.codes = [rng.randint(0, 120, c.size).astype(np.uint8) ^ (rng.randint(0, 2, c.size).astype(np.uint8) << 7) for c in p.codes]
        p.scales = [np.exp(rng.normal(-4.0, 0.5, x.size)).astype(np.float32) if dtype == "i8" else np.exp(rng.normal(-4.0, 0.3, x.size)).astype(np.float32) for x in p.scales]
        q = queries(len(lens), 1, hq, d)
        got = run(hip, p, q, 0.02, lens)
        assert np.array_equal(got, run(hip, p, q, 0.02, lens))
        for s in (0, 1, 17, 39):
            for h in (0, 5):
                at = p.lead + p.table[s].astype(np.int64) * p.cache.page_stride
                rows = (at[:, None] + h * p.cache.head_stride + np.arange(16) * p.cache.row_stride).reshape(-1)[:lens[s]]
                sc = (p.table[s].astype(np.int64)[:, None] * p.sc.page_stride + h * p.sc.head_stride + np.arange(16) // block).reshape(-1)[:lens[s]]
                k, v = (values(p.codes[w][rows[:, None] + np.arange(d)].ravel(), dtype).reshape(-1, d) * p.scales[w][sc][:, None].astype(np.float64) for w in range(2))
                x = k @ q[s, 0, h].astype(np.float64) * float(np.float32(0.02))
                w = np.exp(x - x.max())
                assert rel_err(got[s, 0, h], (w[:, None] * v).sum(0) / w.sum()) <= TOL_GEMM_F32


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_one_key_above_tens_of_thousands(hip, dtype):
    """130 heads take one share each: 20000 keys of one weight, 9 to 14 nats below the first, under values of one are one. Sums of weights go over
    8 keys of a tile, 8 tiles, 20 such groups, 16 lanes and 4 wavefronts: at most 7 + 8 + 20 + 5 roundings of 2^-24 of a sum of positive numbers; the
    products' over 3 x 8 steps of the matrix units, counted twice, 20 groups and 4 wavefronts."""
    n, heads, d = 20000, 130, 64
    p = Scaled(22, 1, heads, d, 64, 64, dtype, -(-n // 64))
    one = 1 if dtype == "i8" else 0x38
    p.codes = [np.zeros_like(p.codes[0]), np.full_like(p.codes[1], one)]
    p.scales = [np.ones_like(x) for x in p.scales]
    for h in range(heads):
        at = p.row_at(0, 0, h)
        p.codes[0][at:at + d] = one
    q = np.repeat(np.linspace(9.0, 14.0, heads, dtype=np.float32)[None, None, :, None] / d, d, axis=3)
    got = run(hip, p, q, 1.0, [n])
    assert np.max(np.abs(got.astype(np.float64) - 1)) <= (40 + 48 + 24) * 2.0 ** -24
