"""Appends to and attention over an 8-bit cache whose pages lie more than 4 GiB apart, codes and scales: bit for bit as in a small one."""
import math

import numpy as np
import pytest

from conftest import TOL_GEMM_F32, rel_err
from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer, paged_cache, paged_scales, rotary_tables

pytestmark = pytest.mark.gpu

PAGES, PAGE, HEADS, D, QUERIES = 1100, 16, 2, 64, 6


@pytest.mark.parametrize("block,page_stride", [(16, 1 << 22), (4, 1 << 22), (1, 1 << 22), (16, (1 << 22) + 1)])
def test_far_pages(hip, block, page_stride):
    """The last stride is none that vectors take."""
    lens = [70, 33, 512]
    width = -(-max(lens) // PAGE)
    table = (1 + np.random.RandomState(1).permutation(PAGES - 3)[:3 * width]).reshape(3, width).astype(np.int32)
    table[0, :3] = PAGES - 1, 0, PAGES - 2  # (the ends of the pool)
    tokens = [(s, i) for s, n in enumerate(lens) for i in range(n)]
    seqs, positions = (DeviceBuffer.from_host(np.array(x, np.int32)) for x in zip(*tokens))
    proj = DeviceBuffer.from_host(synth.normal(2, "p", (len(tokens), (QUERIES + 2 * HEADS) * D)))
    cos, sin = (DeviceBuffer.from_host(x) for x in rotary_tables(600, D))
    dev_table, dev_lens = DeviceBuffer.from_host(table), DeviceBuffer.from_host(np.array(lens, np.int32))
    q = DeviceBuffer.from_host(synth.normal(3, "q", (3, 1, QUERIES, D)))
    results = []
    for stride, scale_stride in ((HEADS * PAGE * D, HEADS * PAGE // block), (page_stride, 1 << 20)):
        cache = paged_cache(PAGES, PAGE, HEADS, D, 3, width, "e4m3")
        scales = paged_scales(cache, block)
        cache.page_stride, scales.page_stride = stride, scale_stride
        assert stride < 1 << 22 or PAGES * stride > 1 << 32 and 4 * PAGES * scale_stride > 1 << 32
        pools = [DeviceBuffer((PAGES * stride,), np.uint8) for _ in range(2)] + [DeviceBuffer((PAGES * scale_stride,)) for _ in range(2)]
        desc = hip.paged_append_desc(cache, len(tokens), QUERIES, D, 600, row_stride=(QUERIES + 2 * HEADS) * D)
        rotated, out, bad = DeviceBuffer((len(tokens), QUERIES, D)), DeviceBuffer((3, 1, QUERIES, D)), DeviceBuffer((1,), np.int64)
        hip.paged_append_scaled(cache, scales, desc, proj, proj.view(QUERIES * D), proj.view((QUERIES + HEADS) * D), cos, sin, dev_table, seqs, positions, rotated, *pools, bad_index=bad)
        hip.synchronize()
        assert bad.to_host()[0] == -1
        hip.paged_sdpa_scaled(cache, scales, hip.paged_sdpa_desc(cache, QUERIES, 1), 1 / math.sqrt(D), q, *pools, dev_table, dev_lens, out, bad_index=bad)
        hip.synchronize()
        assert bad.to_host()[0] == -1
        results.append([rotated.to_host(), out.to_host()])
        del pools
    assert np.array_equal(results[0][0], results[1][0])
    if page_stride % 16 == 0:
        assert np.array_equal(results[0][1].view(np.uint32), results[1][1].view(np.uint32))
    else:  # another kernel: each is within TOL_GEMM_F32 of the definition
        assert rel_err(results[0][1], results[1][1]) <= 2 * TOL_GEMM_F32
