"""Extents that the paged cache's calls refuse because a number inside would not hold them, without a device. No pointer here is
ever followed."""
import ctypes as C

import pytest

from frankentorch_amd import _lib, device
from test_generation_abi import INVALID, OK, OVERFLOW, append, attend, cache


@pytest.mark.parametrize("page_size", [1 << 31, 1 << 32, 3 << 32, (1 << 32) + 16, 1 << 57])
@pytest.mark.parametrize("rows", [0, 1])
def test_pages_longer_than_any_position(page_size, rows):
    """Also where a table without columns leaves no position at all, and where queries alone are rotated."""
    kw = dict(page_size=page_size, max_pages=0, table_stride=0, num_pages=0, head_dim=1, row_stride=1, head_stride=1, page_stride=1)
    c = cache(**kw)
    d = device.paged_append_desc(c, rows, 4, 0, 100)
    lib = _lib.load()
    assert lib.fth_dev_paged_append_f32(C.byref(c), C.byref(d), 4096, None, None, None, None, None, None, 4096, 8192, None, None, None, None) == OVERFLOW
    assert attend(cache(**kw), rows) == OVERFLOW
    assert lib.fth_dev_paged_sdpa_workspace_bytes(C.byref(c), C.byref(device.paged_sdpa_desc(c, 4))) == 0
    kw["page_size"] = (1 << 31) - 1
    assert attend(cache(**kw), 0) in OK


@pytest.mark.parametrize("q_heads", [(1 << 63) - 1, (1 << 63) - 2, (1 << 62), (1 << 20) + 1, 1 << 20])
def test_heads_whose_sum_overflows(q_heads):
    """Queries and K/V heads together are at most 2^20, also where their sum is no 64-bit number."""
    for tokens in (0, 1):
        assert append(cache(), tokens, q_heads=q_heads) == OVERFLOW
    assert append(cache(), 0, q_heads=(1 << 20) - 2) in OK
