"""New keys and values into a paged cache: bit for bit what stepwise float32 gives (each product and sum rounded), near the
rotation in 64 bits, and nothing written anywhere else."""
import numpy as np
import pytest

from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer
from paged_case import Paged, from_storage, rotated, to_storage

pytestmark = pytest.mark.gpu


def tokens_of(lens, new):
    """(seq_ids, positions) of the last new[s] positions of every sequence, in an order that mixes the sequences."""
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(new)]).astype(np.int32)
    pos = np.concatenate([np.arange(x - n, x) for x, n in zip(lens, new)]).astype(np.int32)
    order = np.argsort(synth.uniform(5, "order", (len(seq),)))
    return seq[order], pos[order]


def expect(p, seq, pos, k, v):
    stores = [from_storage(to_storage(x, p.dtype), p.dtype) for x in p.stores]
    for t in range(len(seq)):
        if seq[t] >= 0 and pos[t] >= 0:
            at = p.index(seq[t], np.array([pos[t]]))[0]
            for store, x in zip(stores, (k, v)):
                store[at] = from_storage(to_storage(x[t], p.dtype), p.dtype)
    return stores


# (lens, new, hq, hkv, d, page, rotary, interleaved, dtype)
CASES = [
    ([1], [1], 1, 1, 64, 16, 64, False, "f32"), ([17, 1, 40], [1, 1, 1], 8, 2, 128, 16, 128, False, "bf16"), ([33, 0, 5], [20, 0, 5], 4, 4, 64, 16, 0, False, "f32"),
    ([100, 31], [100, 2], 8, 2, 128, 48, 64, True, "f16"), ([50, 60], [50, 7], 6, 3, 64, 5, 32, False, "bf16"), ([50, 9], [13, 9], 0, 2, 128, 1, 128, True, "f16"),
    ([40], [40], 5, 1, 80, 16, 80, False, "bf16"), ([40, 3], [40, 3], 5, 1, 80, 16, 20, True, "f32"), ([30], [30], 3, 1, 20, 7, 6, False, "f16"),
    ([30], [30], 3, 1, 7, 7, 6, True, "bf16"), ([30, 2], [30, 1], 2, 2, 33, 16, 2, False, "f32"), ([9], [9], 1, 1, 1, 4, 0, False, "bf16"), ([300], [300], 4, 1, 256, 16, 256, False, "f16"),
    ([64], [64], 4, 2, 72, 16, 24, False, "bf16"), ([64], [64], 4, 2, 72, 16, 24, True, "f16"), ([700, 650], [600, 650], 12, 12, 64, 16, 0, False, "f32"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("layout", ["contiguous", "packed", "odd"])
def test_against_stepwise_float32(hip, case, layout):
    lens, new, hq, hkv, d, page, rotary, inter, dtype = case
    p = Paged(31, lens, hkv, d, page, dtype, pad=3 if layout == "odd" else 0, lead=1 if layout == "odd" else 0, heads_inside=layout == "packed")
    seq, pos = tokens_of(lens, new)
    t = len(seq)
    q, k, v = (synth.normal(31, n, (t, h, d)) for n, h in (("nq", hq), ("nk", hkv), ("nv", hkv)))
    max_pos = max(lens)
    cos, sin = hip.rotary_tables(max_pos, rotary) if rotary else (None, None)
    kc, vc = p.upload()
    desc = hip.paged_append_desc(p.cache, t, hq, rotary, max_pos, inter)
    if layout == "contiguous":
        dq, dk, dv = (DeviceBuffer.from_host(x) if x.size else None for x in (q, k, v))
    else:
        pad = 5 if layout == "odd" else 0
        proj = np.full((t, (hq + 2 * hkv) * d + pad), np.nan, np.float32)
        proj[:, pad:] = np.concatenate([q.reshape(t, -1), k.reshape(t, -1), v.reshape(t, -1)], 1)
        whole = DeviceBuffer.from_host(proj)
        desc.q_row_stride = desc.k_row_stride = desc.v_row_stride = proj.shape[1]
        dq, dk, dv = whole.view(pad), whole.view(pad + hq * d), whole.view(pad + (hq + hkv) * d)
    out = DeviceBuffer.from_host(np.full((t, hq, d), 7.0, np.float32)) if hq else None
    bad = DeviceBuffer((1,), np.int64)
    tables = [DeviceBuffer.from_host(x) if rotary else None for x in (cos, sin)]
    args = (p.dev_table, DeviceBuffer.from_host(seq), DeviceBuffer.from_host(pos))
    hip.paged_append(p.cache, desc, dq if hq else None, dk, dv, *tables, *args, out, kc, vc, bad)
    hip.synchronize()
    assert bad.to_host()[0] == -1
    turn = lambda x, kind: rotated(x, pos, cos, sin, rotary, inter, kind) if rotary else x.astype(kind)
    want = expect(p, seq, pos, turn(k, np.float32), v)
    for got, ref in zip(p.download(), want):
        assert np.array_equal(got, ref, equal_nan=True)
    if hq:
        got = out.to_host()
        assert np.array_equal(got, turn(q, np.float32))
        # three roundings, of numbers no larger than 2 max(|a|, |b|) each
        assert np.all(np.abs(got - turn(q, np.float64)) <= 3 * 2.0 ** -24 * 2 * np.abs(q).max())
        if layout == "contiguous":  # in place
            hip.paged_append(p.cache, desc, dq, dk, dv, *tables, *args, dq, kc, vc)
            hip.synchronize()
            assert np.array_equal(dq.to_host(), got)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1])
def test_skipped_and_invalid_tokens(hip, dtype, pad):
    """Position -1 is skipped without a report; other positions, sequences, pages and rows of the tables that do not exist are
    reported, the lowest first; none of them writes anything, and the tokens beside them are stored."""
    d, hkv, hq = 64, 2, 4
    p = Paged(32, [40, 50], hkv, d, 16, dtype, pad=pad)
    p.table[0, 1] = p.cache.num_pages
    p.table[1, 3] = -1
    seq = np.array([0, 1, 0, 2, -1, 1, 1, 0, 1, 0], np.int32)
    pos = np.array([3, -1, 5, 0, 0, 2 ** 31 - 1, -2, 20, 49, 39], np.int32)
    good = np.array([0, 2, 9])
    t = len(seq)
    q, k, v = (synth.normal(32, n, (t, h, d)) for n, h in (("q", hq), ("k", hkv), ("v", hkv)))
    cos, sin = hip.rotary_tables(40, d)
    bad, bufs = DeviceBuffer((1,), np.int64), [DeviceBuffer.from_host(x) for x in (q, k, v, cos, sin)]

    def call(seq, pos, max_pos):
        kc, vc = p.upload()
        out = DeviceBuffer.from_host(np.full(q.shape, 7.0, np.float32))
        hip.paged_append(p.cache, hip.paged_append_desc(p.cache, t, hq, d, max_pos), *bufs, p.dev_table, DeviceBuffer.from_host(seq), DeviceBuffer.from_host(pos), out, kc, vc, bad)
        hip.synchronize()
        return out.to_host(), p.download(), int(bad.to_host()[0])

    for max_pos, ok in ((40, good), (39, good[:2])):
        out, stores, first = call(seq, pos, max_pos)
        assert first == 3
        rk = rotated(k, np.clip(pos, 0, 39), cos, sin, d, False, np.float32)
        kept = np.where(np.isin(np.arange(t), ok), pos, -1)
        for got, ref in zip(stores, expect(p, seq, kept, rk, v)):
            assert np.array_equal(got, ref, equal_nan=True)
        assert np.array_equal(out[ok], rotated(q, np.clip(pos, 0, 39), cos, sin, d, False, np.float32)[ok])
        assert np.all(np.delete(out, ok, axis=0) == 7.0)
    assert call(np.zeros(t, np.int32), np.array([-1] * 9 + [2], np.int32), 40)[2] == -1
    assert call(np.zeros(t, np.int32), np.array([0] * 9 + [40], np.int32), 40)[2] == 9


def test_values_at_the_ends_of_the_types(hip):
    """NaN stays NaN, infinities stay, what F16 cannot hold becomes infinite, ties go to even, subnormals are kept."""
    x = np.array([np.nan, np.inf, -np.inf, 65504.0, 65519.9, 65520.0, -1e6, 6e-8, 2.9e-8, 1.0009765625 - 2 ** -11, 1.0 + 2 ** -11, 1.0 + 3 * 2 ** -11, 1e-39, -0.0, 3.3895314e38, 1.0039062],
                 np.float32).reshape(1, 1, 16)
    for dtype in ("f32", "f16", "bf16"):
        p = Paged(33, [1], 1, 16, 16, dtype)
        kc, vc = p.upload()
        b = DeviceBuffer.from_host(x)
        hip.paged_append(p.cache, hip.paged_append_desc(p.cache, 1), None, b, b, None, None, p.dev_table, DeviceBuffer.from_host(np.zeros(1, np.int32)),
                         DeviceBuffer.from_host(np.zeros(1, np.int32)), None, kc, vc)
        hip.synchronize()
        ref = from_storage(to_storage(x, dtype), dtype).reshape(-1)
        for got in p.download():
            assert np.array_equal(got[p.index(0, np.array([0]))].reshape(-1), ref, equal_nan=True), dtype


def test_nothing_to_append(hip):
    p = Paged(34, [5], 1, 64, 16, "bf16")
    kc, vc = p.upload()
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    hip.paged_append(p.cache, hip.paged_append_desc(p.cache, 0), None, None, None, None, None, p.dev_table, None, None, None, kc, vc, bad)
    assert bad.to_host()[0] == -1


@pytest.mark.parametrize("d,rotary,interleaved", [(64, 64, False), (64, 32, True), (20, 6, False)])
def test_queries_alone(hip, d, rotary, interleaved):
    """Without keys and values only queries are rotated: no sequence, table or cache is looked at; positions still count."""
    t, hq = 37, 5
    q, pos = synth.normal(35, "q", (t, hq, d)), (np.arange(t) * 3 % 50).astype(np.int32)
    cos, sin = hip.rotary_tables(50, rotary)
    cache, bad = hip.paged_cache(0, 16, 1, d, 0, 0, "bf16"), DeviceBuffer((1,), np.int64)
    bufs = [DeviceBuffer.from_host(x) for x in (cos, sin)]

    def call(pos):
        out = DeviceBuffer.from_host(np.full(q.shape, 7.0, np.float32))
        hip.paged_append(cache, hip.paged_append_desc(cache, t, hq, rotary, 50, interleaved), DeviceBuffer.from_host(q), None, None, *bufs, None, None,
                         DeviceBuffer.from_host(pos), out, None, None, bad)
        hip.synchronize()
        return out.to_host(), int(bad.to_host()[0])

    ref = rotated(q, pos, cos, sin, rotary, interleaved, np.float32)
    out, first = call(pos)
    assert first == -1 and np.array_equal(out, ref)
    pos[[4, 9, 30]] = -1, 50, -2
    out, first = call(pos)
    kept = np.delete(np.arange(t), [4, 9, 30])
    assert first == 9 and np.array_equal(out[kept], ref[kept]) and np.all(out[[4, 9, 30]] == 7.0)
