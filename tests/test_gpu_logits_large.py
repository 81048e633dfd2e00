"""Logits at the ends of what a call takes."""
import numpy as np
import pytest

from frankentorch_amd import _lib
from frankentorch_amd.device import DeviceBuffer

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
