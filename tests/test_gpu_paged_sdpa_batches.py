"""Attention over a paged cache for batches that fill the chip, where the keys of all sequences are shared out end to end if there are
enough of them, and cut by sequence if not: cuts anywhere, sequences of very different lengths among them, against the definition
in 64 bits."""
import numpy as np
import pytest

from conftest import TOL_GEMM_F32, rel_err
from frankentorch_amd import _lib, synth
from frankentorch_amd.device import DeviceBuffer, Stream
from paged_case import Paged, attention
from test_gpu_paged_sdpa import queries, run

pytestmark = pytest.mark.gpu


def lengths(seed, num, longest, new):
    """Mostly short ones, empty ones, the edges of tiles and of steps, a few long ones, in no order."""
    edges = [0, 1, new, new + 1, 31, 32, 33, 127, 128, 129, 135, 255, 256, 257, longest, longest - 1, longest // 2]
    drawn = (synth.uniform(seed, "lens", (num,)) ** 3 * 300).astype(int).tolist()
    x = (edges + drawn)[:num]
    return [x[i] for i in np.argsort(synth.uniform(seed, "order", (num,)))]


# (sequences, hq, hkv, new, d, page, dtype, longest, lead)
CASES = [
    (70, 8, 4, 1, 128, 16, "bf16", 2100, 0), (300, 1, 1, 1, 64, 16, "f32", 2200, 0), (50, 40, 2, 2, 128, 16, "f16", 2300, 0), (130, 4, 2, 8, 72, 8, "f32", 1900, 0),
    (64, 4, 4, 3, 256, 16, "bf16", 1100, 0), (256, 2, 1, 8, 40, 16, "f16", 6600, 0), (65, 16, 4, 4, 128, 5, "f16", 2100, 0), (150, 2, 2, 1, 64, 64, "bf16", 4200, 0),
    (70, 8, 4, 1, 128, 16, "bf16", 2100, 1), (40, 64, 8, 1, 128, 32, "f32", 1030, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(hip, case):
    num, hq, hkv, new, d, page, dtype, longest, lead = case
    p = Paged(31, lengths(31, num, longest, new), hkv, d, page, dtype, lead=lead)
    q = queries(p, hq, new)
    got = run(hip, p, q, 0.11)
    ref = attention(q, p.k, p.v, 0.11, p.lens)
    for s in range(num):  # each by itself: a long sequence must not hide a short one
        assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if ref[s].any() else not got[s].any(), p.lens[s]
    assert np.all(got[ref == 0] == 0)
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, 0.11).view(np.uint32))


@pytest.mark.parametrize("lens", [[0] * 64, [1] * 64, [128] * 64, [600] * 64, [0] * 63 + [2100], [2100] + [0] * 63, [0, 700] * 32, [2100] * 2 + [1] * 62], ids=lambda x: "%d_%d_%d" % (x[0], x[1], x[-1]))
def test_even_and_uneven_batches(hip, lens):
    p = Paged(32, lens, 4, 128, 16, "bf16", room=140)
    q = queries(p, 8, 1)
    got, ref = run(hip, p, q, 0.1, max_len=2200), attention(q, p.k, p.v, 0.1, lens)
    for s in range(64):
        assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if lens[s] else not got[s].any()


# (sequences, hq, hkv, new, d, page, dtype, longest): long enough on average to be shared out end to end
LONG = [(32, 128, 1, 1, 128, 16, "bf16", 3500), (34, 32, 2, 8, 64, 16, "f32", 2700), (16, 256, 1, 1, 256, 16, "bf16", 2000), (32, 120, 1, 1, 72, 8, "f32", 3000),
        (32, 64, 1, 2, 64, 32, "f16", 6500), (100, 36, 1, 1, 128, 16, "f16", 3000), (70, 8, 4, 1, 128, 16, "bf16", 3000)]


def long_lengths(seed, num, longest, new):
    x = [0, new, 128, 129, longest, longest, 127, 1] + (longest * (0.35 + 0.65 * synth.uniform(seed, "lens", (num,)))).astype(int).tolist()
    return [x[i] for i in np.argsort(synth.uniform(seed, "order", (num,)))]


@pytest.mark.parametrize("case", LONG, ids=str)
def test_long_batches(hip, case):
    num, hq, hkv, new, d, page, dtype, longest = case
    p = Paged(36, long_lengths(36, num, longest, new), hkv, d, page, dtype)
    q, bad = queries(p, hq, new), DeviceBuffer((1,), np.int64)
    got = run(hip, p, q, 0.1, bad=bad)
    assert bad.to_host()[0] == -1
    ref = attention(q, p.k, p.v, 0.1, p.lens)
    for s in range(num):
        assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if ref[s].any() else not got[s].any(), p.lens[s]
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, 0.1).view(np.uint32))
    # two sequences that are not there: the others stay as they are, though the cuts move
    told, table = list(p.lens), p.table.copy()
    first, second = p.lens.index(longest), p.lens.index(128)
    told[second], table[first, (longest - 1) // page // 2] = longest + 5000, -3
    got = run(hip, p, q, 0.1, lens=told, table=table, bad=bad)
    assert bad.to_host()[0] == min(first, second) and np.all(np.isnan(got[[first, second]]))
    fine = [s for s in range(num) if s not in (first, second)]
    assert rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32


def test_a_graph_serves_long_and_short_batches(hip):
    from test_gpu_stream_scratch import Graph

    lens = long_lengths(37, 32, 3500, 1)
    p = Paged(37, lens, 1, 128, 16, "bf16")
    q = queries(p, 128, 1)
    kc, vc = p.upload()
    home, side = Stream(), Stream()
    desc, dq = hip.paged_sdpa_desc(p.cache, 128, 1, 3500), DeviceBuffer.from_host(q)
    dl, out = DeviceBuffer.from_host(np.array(lens, np.int32)), DeviceBuffer(q.shape)
    ws = hip.paged_sdpa_workspace(p.cache, desc)
    call = lambda stream: hip.paged_sdpa(p.cache, desc, 0.1, dq, kc, vc, p.dev_table, dl, out, workspace=ws, stream=stream)
    call(home.handle)
    home.synchronize()
    graph = Graph(home, call)
    for step in ([n // 4 for n in lens], lens, [min(n, 3) for n in lens], lens, [0] * 32, [n // 3 for n in lens], lens):
        _lib.load().fth_memcpy_h2d(dl.ptr, np.array(step, np.int32).ctypes.data, 128)
        graph.replay(side)
        hip.synchronize()
        got = out.to_host()
        assert rel_err(got, attention(q, p.k, p.v, 0.1, step)) <= TOL_GEMM_F32
        call(home.handle)
        hip.synchronize()
        assert np.array_equal(got.view(np.uint32), out.to_host().view(np.uint32))
    graph.free()


def test_invalid_sequences_are_reported(hip):
    lens = lengths(33, 70, 2100, 2)
    p = Paged(33, lens, 4, 128, 16, "f16")
    q = queries(p, 8, 2)
    ref, bad = attention(q, p.k, p.v, 0.1, lens), DeviceBuffer((1,), np.int64)
    long = lens.index(2100)
    for first, page_at in ((5, 0), (60, 64), (69, 131), (0, None)):
        told, table, hurt = list(lens), p.table.copy(), {first}
        told[first] = -1 if page_at else 2 ** 31 - 1
        if page_at is not None:
            table[long, page_at] = p.cache.num_pages
            hurt.add(long)
        got = run(hip, p, q, 0.1, lens=told, table=table, bad=bad)
        assert bad.to_host()[0] == min(hurt)
        fine = [s for s in range(70) if s not in hurt]
        assert np.all(np.isnan(got[sorted(hurt)])) and rel_err(got[fine], ref[fine]) <= TOL_GEMM_F32


def test_values_that_are_not_finite_stay_where_they_are_seen(hip):
    """NaN in V of the last of four new tokens reaches the last query alone, wherever the cuts fall."""
    lens = [n for n in range(120, 140)] + [0, 3, 2100] + [250 + n for n in range(41)]
    p = Paged(34, lens, 4, 128, 16, "bf16")
    q = queries(p, 8, 4)
    ref = attention(q, p.k, p.v, 0.1, lens)
    for s, n in enumerate(lens):
        if n:
            p.stores[1][p.index(s, np.array([n - 1]))] = np.nan
    got = run(hip, p, q, 0.1)
    some = [s for s, n in enumerate(lens) if n]
    assert np.all(np.isnan(got[some, 3])) and np.all(got[lens.index(0)] == 0)
    assert rel_err(got[:, :3], ref[:, :3]) <= TOL_GEMM_F32


def test_a_graph_serves_every_batch(hip):
    from test_gpu_stream_scratch import Graph

    lens = lengths(35, 70, 2100, 1)
    p = Paged(35, lens, 4, 128, 16, "bf16")
    q = queries(p, 8, 1)
    kc, vc = p.upload()
    home, side = Stream(), Stream()
    desc, dq = hip.paged_sdpa_desc(p.cache, 8, 1, 2100), DeviceBuffer.from_host(q)
    dl, out, eager = DeviceBuffer.from_host(np.array(lens, np.int32)), DeviceBuffer(q.shape), DeviceBuffer(q.shape)
    ws = [hip.paged_sdpa_workspace(p.cache, desc) for _ in range(2)]
    call = lambda o, w, stream: hip.paged_sdpa(p.cache, desc, 0.1, dq, kc, vc, p.dev_table, dl, o, workspace=w, stream=stream)
    call(out, ws[0], home.handle)
    home.synchronize()
    graph = Graph(home, lambda stream: call(out, ws[0], stream))
    for step in (lens, [min(n, 1) for n in lens], [0] * 70, [n // 2 for n in lens], lens):
        _lib.load().fth_memcpy_h2d(dl.ptr, np.array(step, np.int32).ctypes.data, 280)
        graph.replay(side)
        call(eager, ws[1], home.handle)
        hip.synchronize()
        got = out.to_host()
        assert np.array_equal(got.view(np.uint32), eager.to_host().view(np.uint32))
        assert rel_err(got, attention(q, p.k, p.v, 0.1, step)) <= TOL_GEMM_F32
    graph.free()


@pytest.mark.parametrize("lens", [[5, 300, 0, 131] * 16, [40] * 63 + [3000], [700] * 64], ids=lambda x: str(x[-1]))
def test_a_bound_far_above_the_lengths(hip, lens):
    p = Paged(38, lens, 4, 128, 16, "bf16", room=4096)
    q = queries(p, 8, 1)
    got, ref = run(hip, p, q, 0.1, max_len=65536), attention(q, p.k, p.v, 0.1, lens)
    for s, n in enumerate(lens):
        assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if n else not got[s].any()
