"""Attention over a paged cache against the definition in 64 bits: lengths around the tiles, pages and shares, head layouts,
storage types, strides and alignments, what lies past a sequence's end, and what the call reports and refuses."""
import ctypes as C
import math

import numpy as np
import pytest

from conftest import TOL_GEMM_F32, rel_err
from frankentorch_amd import _lib, synth
from frankentorch_amd.device import DeviceBuffer, Stream
from paged_case import Paged, attention, from_storage, to_storage

pytestmark = pytest.mark.gpu


def run(hip, p, q, scale, max_len=None, bad=None, stream=None, lens=None, table=None):
    kc, vc = p.upload()
    desc = hip.paged_sdpa_desc(p.cache, q.shape[2], q.shape[1], max_len)
    out = DeviceBuffer.from_host(np.full(q.shape, 7.0, np.float32))
    dq, dl = DeviceBuffer.from_host(q), DeviceBuffer.from_host(np.array(p.lens if lens is None else lens, np.int32))
    hip.paged_sdpa(p.cache, desc, scale, dq, kc, vc, p.dev_table if table is None else DeviceBuffer.from_host(table), dl, out, bad_index=bad, stream=stream)
    hip.synchronize()
    return out.to_host()


def queries(p, hq, new, seed=3, std=1.5):
    return synth.normal(seed, "q", (len(p.lens), new, hq, p.d), 0.0, std)


# (lens, hq, hkv, new, d, page, dtype)
CASES = [
    ([1], 1, 1, 1, 64, 16, "f32"), ([0, 1, 2], 2, 2, 1, 64, 16, "f32"), ([31, 32, 33], 4, 2, 1, 64, 16, "bf16"), ([15, 16, 17, 0, 5], 8, 1, 1, 128, 16, "f16"),
    ([63, 64, 65, 127, 128, 129], 6, 2, 1, 64, 32, "f32"), ([255, 256, 257], 8, 8, 1, 128, 64, "bf16"), ([300, 7, 0, 1], 12, 12, 1, 64, 16, "f32"),
    ([1000, 3], 8, 2, 1, 128, 128, "f16"), ([2500, 1, 900], 32, 8, 1, 128, 16, "bf16"), ([4099], 8, 1, 1, 64, 16, "f32"), ([5000, 4999], 4, 4, 1, 128, 48, "f16"),
    # several new tokens: the first of them may see nothing
    ([0, 1, 3, 4, 5, 8, 40], 4, 2, 4, 64, 16, "f32"), ([7, 8, 9, 600], 8, 2, 8, 128, 16, "bf16"), ([2, 33, 700], 5, 1, 7, 64, 16, "f16"), ([513], 32, 8, 2, 128, 32, "f32"),
    # more than 16 query rows on a K/V head
    ([200, 17, 1100], 17, 1, 1, 64, 16, "bf16"), ([400, 31], 32, 1, 4, 128, 16, "f16"), ([77, 900], 24, 2, 3, 64, 16, "f32"), ([50], 33, 1, 8, 128, 16, "bf16"),
    # head sizes, pages that are no multiple of anything
    ([70, 1, 40], 4, 2, 1, 32, 16, "f32"), ([70, 300], 4, 4, 2, 80, 16, "bf16"), ([70, 300], 4, 2, 1, 96, 16, "f16"), ([90, 333], 4, 2, 1, 256, 16, "bf16"),
    ([90, 333, 2], 4, 1, 3, 256, 16, "f32"), ([260], 3, 1, 1, 200, 16, "f16"), ([45, 130], 2, 1, 1, 40, 16, "f32"), ([45, 130], 2, 1, 1, 20, 16, "f16"),
    ([45, 130], 4, 2, 2, 7, 16, "bf16"), ([33], 1, 1, 1, 1, 16, "f32"), ([100, 65, 1], 4, 2, 1, 64, 1, "bf16"), ([100, 65, 3], 4, 2, 2, 128, 5, "f32"),
    ([100, 650], 4, 2, 1, 64, 24, "f16"), ([777, 20], 8, 2, 1, 128, 40, "bf16"), ([300, 299], 4, 4, 1, 64, 7, "f16"), ([100, 650], 16, 2, 4, 72, 8, "f32"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(hip, case):
    lens, hq, hkv, new, d, page, dtype = case
    p = Paged(11, lens, hkv, d, page, dtype)
    q, scale = queries(p, hq, new), 1.0 / math.sqrt(d)
    got = run(hip, p, q, scale)
    ref = attention(q, p.k, p.v, scale, lens)
    assert rel_err(got, ref) <= TOL_GEMM_F32
    assert np.all(got[ref == 0] == 0)  # a query that sees nothing gives zeros
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, scale).view(np.uint32))  # and runs repeat


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,lead,heads_inside", [(0, 0, True), (8, 0, False), (8, 16, True), (3, 0, False), (0, 1, False), (1, 5, True)])
def test_layouts_and_alignments(hip, dtype, pad, lead, heads_inside):
    """Rows apart from each other, caches that start anywhere, heads beside each other; queries and outputs with strides."""
    lens, hq, hkv, new, d = [130, 0, 33, 700], 8, 2, 2, 64
    p = Paged(12, lens, hkv, d, 16, dtype, pad, lead, heads_inside)
    q, scale = queries(p, hq, new), 0.2
    kc, vc = p.upload()
    for qpad in (4, 1):
        desc = hip.paged_sdpa_desc(p.cache, hq, new)
        desc.q_head_stride, desc.q_row_stride, desc.q_seq_stride = new * (d + qpad), d + qpad, hq * new * (d + qpad)  # [seq, head, token, d]
        desc.o_row_stride, desc.o_head_stride, desc.o_seq_stride = d + qpad, new * (d + qpad), hq * new * (d + qpad)
        store = np.full((len(lens), hq, new, d + qpad), np.nan, np.float32)
        store[..., :d] = q.transpose(0, 2, 1, 3)
        out = DeviceBuffer.from_host(np.full(store.shape, 7.0, np.float32))
        hip.paged_sdpa(p.cache, desc, scale, DeviceBuffer.from_host(store), kc, vc, p.dev_table, DeviceBuffer.from_host(np.array(lens, np.int32)), out)
        hip.synchronize()
        got = out.to_host()
        assert np.all(got[..., d:] == 7.0)  # nothing between the rows is written
        assert rel_err(got[..., :d].transpose(0, 2, 1, 3), attention(q, p.k, p.v, scale, lens)) <= TOL_GEMM_F32


def test_shared_pages_and_other_orders(hip):
    """Two sequences share a prompt's pages, each goes on in its own; the same pages in another place give the same bits."""
    page, d, hkv = 16, 64, 2
    p = Paged(13, [40, 40, 40], hkv, d, page, "bf16")
    p.table[1, :2] = p.table[0, :2]
    for x in (p.k, p.v):
        x[1][:, :32] = x[0][:, :32]
    q = queries(p, 4, 1)
    got = run(hip, p, q, 0.125)
    assert rel_err(got, attention(q, p.k, p.v, 0.125, p.lens)) <= TOL_GEMM_F32
    other = Paged(13, [40, 40, 40], hkv, d, page, "bf16", spare=9)
    for s in range(3):
        for x, y, store in ((p.k, other.k, other.stores[0]), (p.v, other.v, other.stores[1])):
            store[other.index(s, np.arange(40))] = x[s].transpose(1, 0, 2)
    assert np.array_equal(run(hip, other, q, 0.125).view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 31, 33, 64, 300, 1030])
def test_values_that_are_not_finite(hip, dtype, n):
    """In a visible V row an infinity is infinite in the outputs and a NaN is NaN, in that column; a NaN in a visible K row is
    NaN everywhere; a score of minus infinity weighs nothing. The other sequence and the other K/V head never see them."""
    for what in ("v_inf", "v_nan", "k_nan", "k_inf"):
        for at in {0, n // 2, n - 1}:
            p = Paged(14, [n, n], 2, 64, 16, dtype)
            q = np.abs(queries(p, 4, 1)) + np.float32(0.25)
            if what == "v_inf":
                p.v[0][0, at, 3], p.v[0][0, at, 9] = np.inf, -np.inf
            elif what == "v_nan":
                p.v[0][0, at, 5] = np.nan
            elif what == "k_nan":
                p.k[0][0, at, 7] = np.nan
            else:
                p.k[0][0, at, 7] = -np.inf  # the queries are positive: the score is -inf
            for x, store in ((p.k, p.stores[0]), (p.v, p.stores[1])):
                store[p.index(0, np.arange(n))] = x[0].transpose(1, 0, 2)
            got, ref = run(hip, p, q, 0.125), attention(q, p.k, p.v, 0.125, p.lens)
            fine = np.isfinite(ref)
            assert np.array_equal(got[~fine], ref[~fine], equal_nan=True), (what, at)
            if fine.any():
                assert rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32, (what, at)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_extreme_scores_and_scales(hip, dtype):
    """Scores of thousands (one key takes all the weight), a scale of zero (the mean of V) and a negative one, tiny and huge queries."""
    for std, scale in ((200.0, 1.0), (1.0, 0.0), (1.0, -0.3), (1e-30, 1e29), (1e20, 1e-20), (3e4, 1e-4), (1e-6, 1e5)):
        p = Paged(15, [500, 33, 1], 2, 128, 16, dtype)
        q = queries(p, 8, 1, std=std)
        got, ref = run(hip, p, q, scale), attention(q, p.k, p.v, np.float32(scale), p.lens)
        # scores of thousands are rounded to parts of a thousandth: weights move by as much
        size = float(np.max(np.abs(q))) * 12 * 4 * abs(scale)
        assert rel_err(got, ref) <= max(TOL_GEMM_F32, 4 * size * 2.0 ** -23), (std, scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_invalid_sequences_are_reported(hip, dtype):
    """A length below zero, above max_len or above what the table holds, a page that does not exist in the middle: NaN for that
    sequence, the lowest one in bad_index, the others as ever. Without bad_index the same values."""
    p = Paged(16, [100, 90, 80, 700, 60], 2, 64, 16, dtype, room=0)
    q = queries(p, 4, 2)
    ref = attention(q, p.k, p.v, 0.125, p.lens)
    bad = DeviceBuffer((1,), np.int64)

    def check(hurt, **kw):
        got = run(hip, p, q, 0.125, bad=bad, **kw)
        assert bad.to_host()[0] == (min(hurt) if hurt else -1)
        fine = [s for s in range(5) if s not in hurt]
        assert np.all(np.isnan(got[list(hurt)])) and rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32
        again = run(hip, p, q, 0.125, **kw)
        assert np.array_equal(got.view(np.uint32), again.view(np.uint32))

    check([])
    check([1], lens=[100, -1, 80, 700, 60])
    check([0, 3], lens=[2 ** 31 - 1, 90, 80, 705, 60])
    check([3], max_len=699)
    for at in (0, 3, 43):
        for page in (-1, -2 ** 31, p.cache.num_pages, 2 ** 31 - 1):
            table = p.table.copy()
            table[3, at] = page
            check([3], table=table)


def test_empty_calls(hip):
    p = Paged(17, [], 2, 64, 16, "f32")
    q = np.zeros((0, 1, 4, 64), np.float32)
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    assert run(hip, p, q, 1.0, bad=bad).size == 0 and bad.to_host()[0] == -1
    p = Paged(17, [0, 0], 2, 64, 16, "bf16", spare=0, room=0)  # no pages at all
    q = queries(p, 4, 1)
    assert np.all(run(hip, p, q, 1.0, max_len=0) == 0)


def test_a_long_cache(hip):
    """Offsets past 2^32 bytes: two sequences whose pages lie at both ends of a cache of 5 GiB, lengths over many shares."""
    page, d, hkv, n = 64, 128, 2, 30011
    used = -(-n // page)
    pages = (5 << 30) // (hkv * page * d * 2)
    stores = [DeviceBuffer((pages * hkv * page * d,), np.uint16) for _ in range(2)]
    order = [np.arange(used)[::-1], np.arange(used)]  # the first sequence runs backwards from the front, the other at the very end
    table = np.stack([order[0], pages - used + order[1]]).astype(np.int32)
    q, rows = synth.normal(18, "q", (2, 1, 4, d)), ([], [])
    for s in range(2):
        for which, store, kept in zip("kv", stores, rows):
            x = np.full((hkv, used * page, d), np.nan, np.float32)
            x[:, :n] = from_storage(to_storage(synth.normal(18, "%s%d" % (which, s), (hkv, n, d)), "bf16"), "bf16")
            kept.append(x[:, :n])
            block = np.ascontiguousarray(to_storage(x, "bf16").reshape(hkv, used, page, d).transpose(1, 0, 2, 3)[order[s]])
            at = 0 if s == 0 else (pages - used) * hkv * page * d
            assert _lib.load().fth_memcpy_h2d(store.view(at).ptr, block.ctypes.data, block.nbytes) == 0
    cache = hip.paged_cache(pages, page, hkv, d, 2, used, "bf16")
    desc, out = hip.paged_sdpa_desc(cache, 4, 1), DeviceBuffer((2, 1, 4, d))
    hip.paged_sdpa(cache, desc, 0.125, DeviceBuffer.from_host(q), *stores, DeviceBuffer.from_host(table), DeviceBuffer.from_host(np.array([n, n], np.int32)), out)
    hip.synchronize()
    assert rel_err(out.to_host(), attention(q, *rows, 0.125, [n, n])) <= TOL_GEMM_F32


def test_streams_and_graphs(hip):
    """One captured call serves every length up to max_len: replays on another stream, between eager calls, against eager ones."""
    from test_gpu_stream_scratch import Graph

    p = Paged(19, [900, 400, 3, 77], 2, 128, 16, "bf16")
    q = queries(p, 8, 1)
    kc, vc = p.upload()
    home, side = Stream(), Stream()
    desc, dq = hip.paged_sdpa_desc(p.cache, 8, 1, 900), DeviceBuffer.from_host(q)
    lens, out, eager = DeviceBuffer.from_host(np.array(p.lens, np.int32)), DeviceBuffer(q.shape), DeviceBuffer(q.shape)
    ws = [hip.paged_sdpa_workspace(p.cache, desc) for _ in range(2)]
    call = lambda o, w, stream: hip.paged_sdpa(p.cache, desc, 0.125, dq, kc, vc, p.dev_table, lens, o, workspace=w, stream=stream)
    call(out, ws[0], home.handle)
    home.synchronize()
    graph = Graph(home, lambda stream: call(out, ws[0], stream))
    for step in ([900, 400, 0, 77], [1, 2, 3, 4], [0, 0, 0, 0], [899, 399, 0, 77], [900, 400, 0, 77]):
        _lib.load().fth_memcpy_h2d(lens.ptr, np.array(step, np.int32).ctypes.data, 16)
        graph.replay(side)
        call(eager, ws[1], home.handle)
        hip.synchronize()
        assert np.array_equal(out.to_host().view(np.uint32), eager.to_host().view(np.uint32))
        assert rel_err(out.to_host(), attention(q, p.k, p.v, 0.125, step)) <= TOL_GEMM_F32
    graph.free()


def test_a_workspace_that_is_too_small_is_refused(hip):
    p = Paged(20, [5000], 2, 128, 16, "bf16")
    desc = hip.paged_sdpa_desc(p.cache, 8, 1)
    need = _lib.load().fth_dev_paged_sdpa_workspace_bytes(C.byref(p.cache), C.byref(desc))
    kc, vc = p.upload()
    q, lens = DeviceBuffer.from_host(queries(p, 8, 1)), DeviceBuffer.from_host(np.array([5000], np.int32))
    out = DeviceBuffer.from_host(np.full((1, 1, 8, 128), 7.0, np.float32))
    ws = DeviceBuffer((need // 4 + 4,), np.float32)
    args = lambda w, n: (C.byref(p.cache), C.byref(desc), C.c_float(0.1), q.ptr, kc.ptr, vc.ptr, p.dev_table.ptr, lens.ptr, out.ptr, None, w, n, None)
    fn = _lib.load().fth_dev_paged_sdpa_f32
    if need:
        assert fn(*args(ws.ptr, need - 1)) == 105 and fn(*args(None, need)) == 105
        hip.synchronize()
        assert np.all(out.to_host() == 7.0)
    assert fn(*args(ws.ptr, need)) == 0
    hip.synchronize()
    assert np.all(out.to_host() != 7.0)


@pytest.mark.parametrize("dtype,std", [("f16", 2e-5), ("f16", 6e-7), ("f16", 6e3), ("bf16", 1e-39), ("bf16", 1e30), ("f32", 1e-39), ("f32", 1e15)])
def test_small_and_large_caches(hip, dtype, std):
    """Keys and values among the subnormal numbers of their type, and near its ends: scores of a few units by the scale."""
    for q_std in (1.0, 1e-5, 1e5):
        p = Paged(21, [130, 5], 2, 64, 16, dtype, std=std)
        q, scale = queries(p, 4, 1, std=q_std), np.float32(min(1e37, 0.3 / (std * q_std)))
        got, ref = run(hip, p, q, scale), attention(q, p.k, p.v, scale, p.lens)
        # results below 2^-126 may be rounded to multiples of 2^-149 at each of 130 steps, or flushed
        assert np.max(np.abs(got - ref)) <= TOL_GEMM_F32 * np.max(np.abs(ref)) + 2.0 ** -126, (q_std,)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_that_are_not_finite(hip, dtype):
    """A query row with NaN or an infinity gives NaN, as the formula does; the rows beside it do not see it."""
    p = Paged(22, [200, 3], 2, 64, 16, dtype)
    q = queries(p, 8, 2)
    q[0, 0, 1, 5], q[0, 1, 6, 0], q[1, 1, 3, 63] = np.nan, np.inf, -np.inf
    got, ref = run(hip, p, q, 0.125), attention(q, p.k, p.v, 0.125, p.lens)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.isnan(ref).sum() == 3 * 64
    assert rel_err(got[~np.isnan(ref)], ref[~np.isnan(ref)]) <= TOL_GEMM_F32


@pytest.mark.parametrize("dtype,page,d", [("f32", 16, 64), ("f16", 16, 128), ("bf16", 16, 64), ("bf16", 5, 128), ("f16", 16, 40), ("f32", 16, 7), ("bf16", 16, 256)])
@pytest.mark.parametrize("n", [1, 4, 33, 35, 64, 130, 515])
def test_later_tokens_that_are_not_finite(hip, dtype, page, d, n):
    """Infinities and NaN in K and V of the newest tokens: the queries before them do not see them, those after do, in their column."""
    new, hq, hkv = 6, 4, 2
    for what in ("inf", "nan", "k"):
        for at in {n - 1, max(0, n - 3), max(0, n - new)}:
            p = Paged(23, [n, 40], hkv, d, page, dtype)
            q = np.abs(queries(p, hq, new)) + np.float32(0.25)
            if what == "k":
                p.k[0][0, at, 2 % d] = -np.inf  # weighs nothing where it is seen
            else:
                p.v[0][1, at, 3 % d] = {"inf": np.inf, "nan": np.nan}[what]
                p.v[0][1, at, d - 1] = -np.inf
            for x, store in ((p.k, p.stores[0]), (p.v, p.stores[1])):
                store[p.index(0, np.arange(n))] = x[0].transpose(1, 0, 2)
            got, ref = run(hip, p, q, 0.125), attention(q, p.k, p.v, 0.125, p.lens)
            fine = np.isfinite(ref)
            assert np.array_equal(got[~fine], ref[~fine], equal_nan=True), (what, at)
            assert rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32, (what, at)
