"""Attention whose K and V are loaded past the caches, which goes by the bound on the lengths, and the head sizes and pages that no
other batch reaches: every storage type, in shares of one length and end to end, against the definition in 64 bits."""
import numpy as np
import pytest

from conftest import TOL_GEMM_F32, rel_err
from paged_case import Paged, attention
from test_gpu_paged_sdpa import queries, run
from test_gpu_paged_sdpa_batches import lengths, long_lengths

from frankentorch_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


def check(hip, p, hq, new, max_len):
    size = 4 if p.dtype == "f32" else 2
    assert 2 * len(p.lens) * max_len * p.hkv * p.d * size > 500 << 20 and max_len <= p.max_pages * p.page
    q, bad = queries(p, hq, new), DeviceBuffer((1,), np.int64)
    got = run(hip, p, q, 0.1, max_len=max_len, bad=bad)
    assert bad.to_host()[0] == -1
    ref = attention(q, p.k, p.v, 0.1, p.lens)
    for s, n in enumerate(p.lens):
        assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if ref[s].any() else not got[s].any(), n
    assert np.all(got[ref == 0] == 0)
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, 0.1, max_len=max_len).view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_few_long_sequences(hip, dtype, d):
    lens = [40000, 0, 1, 24999, 33]  # over two shares, and inside one
    check(hip, Paged(71, lens, 2, d, 32, dtype, room=1 << 15), 6, 2, 1 << 20)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_short_sequences(hip, dtype, d):
    check(hip, Paged(72, lengths(72, 64, 1500, 1), 4, d, 16, dtype, room=8192), 8, 1, 1 << 17)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_long_sequences(hip, dtype, d):
    """576 KB a sequence and K/V head: shared out end to end."""
    longest = (576 << 10) // (2 * d * (4 if dtype == "f32" else 2)) * 2
    check(hip, Paged(73, long_lengths(73, 56, longest, 1), 4, d, 16, dtype, room=8192), 8, 1, 1 << 17)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_more_sequences_than_are_shared_out_end_to_end(hip, dtype, d):
    check(hip, Paged(74, lengths(74, 257, 700, 1), 1, d, 16, dtype, room=2048), 4, 1, 1 << 15)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 40, 128, 104, 256, 200])
@pytest.mark.parametrize("page", [16, 24])
def test_head_sizes_and_pages_in_batches_that_fill_the_chip(hip, dtype, d, page):
    """Head sizes below those that the tiles are made for and pages that are no multiple of 16, cut by sequence and end to end."""
    batches = [lengths(75, 64, 900, 3)]
    if page == 24 and d != 64:
        batches.append(long_lengths(75, 120, (576 << 10) // (2 * d * (4 if dtype == "f32" else 2)) * 2, 3))
    for lens in batches:
        hkv = 4 if len(lens) == 64 else 2
        p = Paged(75, lens, hkv, d, page, dtype, room=300)
        q = queries(p, 2 * hkv, 3)
        got, ref = run(hip, p, q, 0.1), attention(q, p.k, p.v, 0.1, lens)
        for s, n in enumerate(lens):
            assert rel_err(got[s], ref[s]) <= TOL_GEMM_F32 if ref[s].any() else not got[s].any(), n
        assert np.all(got[ref == 0] == 0)
