"""Large batches over 8-bit caches, whose sequences are cut end to end into even shares, in every form of the kernels: head sizes that fill them and not,
scales by sixteen positions, by four, by one and looked up by every lane, one row tile and several."""
import numpy as np
import pytest

from conftest import TOL_GEMM_F32
from scaled_case import Scaled, values
from test_gpu_paged_sdpa_scaled import queries, run

pytestmark = pytest.mark.gpu

# (seqs, longest, hq, hkv, new, d, page, block, dtype); a K/V head and sequence has 576 KB and more on average, and there are 256 row tiles of them at least
CASES = [
    (32, 12000, 8, 8, 1, 64, 16, 4, "e4m3"), (32, 12000, 8, 8, 2, 64, 32, 16, "i8"), (32, 12000, 8, 8, 1, 64, 24, 8, "i8"),
    (32, 9000, 8, 8, 1, 80, 16, 16, "e4m3"), (32, 9000, 8, 8, 1, 96, 16, 1, "i8"),
    (32, 6000, 16, 8, 1, 128, 32, 8, "i8"), (32, 6000, 8, 8, 4, 128, 40, 40, "e4m3"), (16, 6000, 24, 8, 8, 128, 16, 16, "e4m3"), (16, 6000, 160, 8, 1, 128, 16, 16, "i8"),
    (16, 6000, 40, 8, 7, 128, 16, 4, "e4m3"), (16, 6000, 40, 8, 7, 128, 8, 8, "i8"),
    (32, 3000, 8, 8, 1, 256, 16, 16, "e4m3"), (32, 3000, 8, 8, 3, 256, 16, 1, "i8"), (32, 3500, 8, 8, 1, 208, 64, 64, "i8"), (16, 3000, 160, 8, 1, 256, 48, 12, "e4m3"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_even_shares(hip, case):
    seqs, longest, hq, hkv, new, d, page, block, dtype = case
    lens = [longest - (i * 7919) % (longest // 2) for i in range(seqs)]
    lens[seqs // 2], lens[seqs // 2 + 1] = 0, 1
    p = Scaled(81, seqs, hkv, d, page, block, dtype, -(-longest // page))
    rng = np.random.RandomState(3)
    p.codes = [rng.randint(0, 256, c.size, dtype=np.uint8) for c in p.codes]
    for c in p.codes:  # no code that stands for no number
        c[c == 128] = 1
        if dtype == "e4m3":
            c[(c & 127) == 127] = 2
    p.scales = [np.exp(rng.normal(-4.0, 0.3, x.size)).astype(np.float32) for x in p.scales]
    q = queries(seqs, new, hq, d)
    got = run(hip, p, q, 0.02, lens)
    assert np.array_equal(got.view(np.uint32), run(hip, p, q, 0.02, lens).view(np.uint32))
    assert not got[seqs // 2].any()
    group = hq // hkv
    for s in (0, 1, seqs // 2 + 1, seqs - 1):
        for hk in (0, hkv - 1):
            pages = p.table[s].astype(np.int64)
            rows = (p.lead + pages[:, None] * p.cache.page_stride + hk * p.cache.head_stride + np.arange(page) * p.cache.row_stride).reshape(-1)[:lens[s]]
            sc = (pages[:, None] * p.sc.page_stride + hk * p.sc.head_stride + np.arange(page) // block).reshape(-1)[:lens[s]]
            k, v = (values(p.codes[w][rows[:, None] + np.arange(d)].ravel(), dtype).reshape(-1, d) * p.scales[w][sc][:, None].astype(np.float64) for w in range(2))
            for i in range(new):
                sees = lens[s] - new + 1 + i
                for h in sorted({hk * group, hk * group + group - 1}):
                    if sees <= 0:
                        assert not got[s, i, h].any()
                        continue
                    x = k[:sees] @ q[s, i, h].astype(np.float64) * float(np.float32(0.02))
                    w = np.exp(x - x.max())
                    ref = (w[:, None] * v[:sees]).sum(0) / w.sum()
                    size = (w[:, None] * np.abs(v[:sees])).sum(0) / w.sum()
                    assert np.all(np.abs(got[s, i, h] - ref) <= TOL_GEMM_F32 * size), (s, i, h)
