"""Appends of more than the caches hold (2^28 bytes), which go past them in chunks of another order: bit for bit what stepwise float32
gives, for every storage type and pairing, and nothing else written."""
import numpy as np
import pytest

from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer
from paged_case import Paged, from_storage, rotated, to_storage
from test_gpu_paged_append import tokens_of

pytestmark = pytest.mark.gpu


def noise(tag, shape):
    """Numbers that are cheap to make and differ along every axis that a wrong index could confuse."""
    n = int(np.prod(shape))
    return np.resize(synth.normal(51, tag, (1 << 20) - 3), n).reshape(shape)


# (dtype, hq, hkv, d, rotary, interleaved)
CASES = [("f32", 8, 4, 128, 128, False), ("f16", 8, 4, 128, 128, False), ("bf16", 8, 4, 128, 64, False), ("f32", 8, 4, 128, 64, True), ("f16", 6, 3, 128, 128, True), ("bf16", 8, 4, 128, 32, True),
         ("f32", 0, 12, 64, 0, False), ("f16", 0, 8, 128, 0, False), ("bf16", 0, 8, 256, 0, True), ("f16", 5, 1, 72, 24, False), ("bf16", 4, 4, 72, 72, True), ("f32", 4, 2, 80, 40, False),
         ("bf16", 4, 2, 256, 256, False), ("f16", 17, 1, 64, 64, False), ("f32", 3, 5, 24, 8, False), ("f16", 9, 9, 8, 8, True)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_stepwise_float32(hip, case):
    dtype, hq, hkv, d, rotary, inter = case
    t = 2 ** 28 // (d * (8 * hq + 2 * hkv * (4 + (4 if dtype == "f32" else 2)))) + 37
    lens, new = [t // 3 + 40, 11, t - t // 3 - 5], [t // 3, 5, t - t // 3 - 5]
    n = [-(-x // 16) for x in lens]
    p = Paged.__new__(Paged)  # without sequences of its own
    p.lens, p.hkv, p.d, p.page, p.dtype, p.lead = lens, hkv, d, 16, dtype, 0
    p.max_pages, total = max(n), sum(n) + 2
    p.cache = hip.paged_cache(total, 16, hkv, d, 3, p.max_pages, dtype)
    order, p.table = np.argsort(synth.uniform(51, "pages", (total,))), np.full((3, p.max_pages), -7, np.int32)
    for s in range(3):
        p.table[s, :n[s]] = order[sum(n[:s]):sum(n[:s + 1])]
    p.stores = [np.full(total * p.cache.page_stride, np.nan, np.float32) for _ in range(2)]
    seq, pos = tokens_of(lens, new)
    assert len(seq) == t
    q, k, v = (noise(tag, (t, h, d)) for tag, h in (("q", hq), ("k", hkv), ("v", hkv)))
    cos, sin = hip.rotary_tables(max(lens), rotary) if rotary else (None, None)
    turn = lambda x: rotated(x, pos, cos, sin, rotary, inter, np.float32) if rotary else x
    kc, vc = p.upload()
    bad, out = DeviceBuffer((1,), np.int64), DeviceBuffer.from_host(np.full((t, hq, d), 7.0, np.float32)) if hq else None
    dq, dk, dv, dc, ds = (DeviceBuffer.from_host(x) if x is not None and x.size else None for x in (q, k, v, cos, sin))
    args = (dc, ds, p.dev_table, DeviceBuffer.from_host(seq), DeviceBuffer.from_host(pos))
    desc = hip.paged_append_desc(p.cache, t, hq, rotary, max(lens), inter)
    hip.paged_append(p.cache, desc, dq, dk, dv, *args, out, kc, vc, bad)
    hip.synchronize()
    assert bad.to_host()[0] == -1
    rows = [p.index(s, np.arange(lens[s] - new[s], lens[s])) for s in range(3)]
    turned = turn(k)
    for got, x in zip(p.download(), (turned, v)):
        want = from_storage(to_storage(x, dtype), dtype)
        for s in range(3):
            mine = np.flatnonzero(seq == s)
            mine = mine[np.argsort(pos[mine])]
            assert np.array_equal(got[rows[s]], want[mine])
            got[rows[s]] = np.nan
        assert np.all(np.isnan(got))  # nothing else was written
    if hq:
        want = turn(q)
        assert np.array_equal(out.to_host(), want)
        hip.paged_append(p.cache, desc, dq, dk, dv, *args, dq, kc, vc)
        hip.synchronize()
        assert np.array_equal(dq.to_host(), want)

