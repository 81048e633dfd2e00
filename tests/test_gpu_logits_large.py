"""Logits at the ends of what a call takes."""
import numpy as np
import pytest

from frankentorch_amd import _lib
from frankentorch_amd.device import DeviceBuffer
from test_gpu_logits import ALL, make, plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 2048, 2 ** 31 - 2047])
def test_a_history_of_as_many_tokens_as_a_length_can_say(hip, n):
    """The last tokens lie where a 32-bit index of the next stretch of the scan would be over its range. One row of eight tokens: 8 GiB
    of history, all of token 3 but the first and the last ones."""
    lib, vocab = _lib.load(), 8
    history = DeviceBuffer((n,), np.int32)
    start = np.full(1 << 22, 3, np.int32)
    assert lib.fth_memcpy_h2d(history.ptr, start.ctypes.data, start.nbytes) == 0
    at = start.size
    while at < n:
        more = min(at, n - at)
        assert lib.fth_memcpy_d2d(history.view(at).ptr, history.ptr, 4 * more) == 0
        at += more
    ends = np.array([5, 6, 1], np.int32)
    assert lib.fth_memcpy_h2d(history.ptr, ends.ctypes.data, 8) == 0
    assert lib.fth_memcpy_h2d(history.view(n - 1).ptr, ends[2:].ctypes.data, 4) == 0
    x, out, bad = np.zeros((1, vocab), np.float32), DeviceBuffer((1, vocab)), DeviceBuffer((1,), np.int64)
    one = lambda v, t: DeviceBuffer.from_host(np.array([v], t))
    hip.logits_process(hip.logits_desc(1, vocab, n), DeviceBuffer.from_host(x), history, one(n, np.int32), one(1, np.int32), None, one(0.5, np.float32), one(0.25, np.float32),
                       None, None, out, bad)
    hip.synchronize()
    assert bad.to_host()[0] == -1
    want = np.zeros(vocab, np.float32)
    want[3] = np.float32(-0.5) * np.float32(n - 3) - np.float32(0.25)  # counts are rounded to fp32
    want[[6, 1]] = -0.75
    assert np.array_equal(out.to_host()[0], want)


@pytest.mark.parametrize("rows,vocab,width", [(130, 65537, 900), (260, 32769, 300), (1030, 4097, 40), (700, 8195, 0), (40, 65537, 500), (2048, 1000, 20), (2048, 1024, 33)])
@pytest.mark.parametrize("shared", [False, True])
def test_two_steps_a_stretch_and_outputs_past_the_caches(hip, rows, vocab, width, shared):
    """From 2048 steps of 4096 logits on a workgroup takes two of them, and from 2^21 logits on outputs go past the caches."""
    m = make(61, rows, vocab, width)
    edge = np.array([0, 4095, 4096, 8191, 8192, vocab - 1], np.int32)
    m["history"][:, :6] = edge[edge < vocab][np.arange(min(6, width)) % len(edge[edge < vocab])] if width else 0
    bad = DeviceBuffer((1,), np.int64)
    want = plain(m, ALL, np.float32, shared)
    assert np.array_equal(run(hip, m, ALL, shared, bad=bad), want) and bad.to_host()[0] == -1
    assert np.array_equal(run(hip, m, ALL, shared, in_place=True), want)
    assert np.array_equal(run(hip, m, ALL, shared, pad=3, lead=1), want)
    use = ("bias", "mask")  # no history: one step a stretch
    assert np.array_equal(run(hip, m, use, shared), plain(m, use, np.float32, shared))


def test_invalid_rows_among_many(hip):
    m = make(62, 130, 65537, 64)
    m["hlen"][:], m["plen"][:] = 64, 20
    m["history"][7, 63], m["history"][99, 0], m["hlen"][129] = 65537, -1, 65
    want = plain({**m, "history": np.clip(m["history"], 0, 65536), "hlen": np.minimum(m["hlen"], 64)}, ALL, np.float32)
    bad = DeviceBuffer((1,), np.int64)
    got = run(hip, m, ALL, bad=bad)
    hurt = [7, 99, 129]
    assert bad.to_host()[0] == 7 and np.all(got[hurt] == 7.0)
    assert np.array_equal(np.delete(got, hurt, 0), np.delete(want, hurt, 0))
