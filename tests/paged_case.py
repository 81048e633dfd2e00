"""Paged caches for the tests, built on the host: storage types as numpy arrays (bf16 as its 16 bits), pages in no order, NaN in
everything that no sequence owns, and the operators written out in 64 bits."""
import numpy as np

from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer, paged_cache


def bf16_bits(x):
    """float32 -> bf16, to nearest even, as uint16 (NaN stays NaN)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_storage(x, dtype):
    if dtype == "bf16":
        return bf16_bits(x)
    with np.errstate(over="ignore"):
        return np.ascontiguousarray(x, np.float32).astype(np.float16 if dtype == "f16" else np.float32)


def from_storage(a, dtype):
    return (a.astype(np.uint32) << 16).view(np.float32) if dtype == "bf16" else a.astype(np.float32)


class Paged:
    """Sequences of the given lengths (rows of K and V that the storage type holds exactly), scattered over pages.

    `pad`: elements between rows, `lead`: elements before the first page, `heads_inside`: rows of all heads of a position side
    by side (page, position, head) in place of (page, head, position)."""

    def __init__(self, seed, lens, hkv, d, page, dtype, pad=0, lead=0, heads_inside=False, spare=2, room=1, std=1.0):
        self.lens, self.hkv, self.d, self.page, self.dtype = list(lens), hkv, d, page, dtype
        n = [-(-max(x, 0) // page) for x in lens]
        self.max_pages, total = max(n + [0]) + room, sum(n) + spare
        self.cache = c = paged_cache(total, page, hkv, d, len(lens), self.max_pages, dtype)
        if heads_inside:
            c.head_stride, c.row_stride = d + pad, hkv * (d + pad)
        else:
            c.row_stride, c.head_stride = d + pad, page * (d + pad)
        c.page_stride = hkv * page * (d + pad)
        order = np.argsort(synth.uniform(seed, "pages", (total,)))
        self.table = np.full((len(lens), self.max_pages), -7, np.int32)
        self.k, self.v, at = [], [], 0
        self.stores = [np.full(lead + total * c.page_stride, np.nan, np.float32) for _ in range(2)]
        self.lead = lead
        for s, x in enumerate(lens):
            self.table[s, :n[s]] = order[at:at + n[s]]
            at += n[s]
            rows = []
            for which, store in zip("kv", self.stores):
                r = synth.normal(seed, "%s%d" % (which, s), (hkv, max(x, 0), d), 0.0, std)
                r = from_storage(to_storage(r, dtype), dtype)
                rows.append(r)
                if x > 0:
                    store[self.index(s, np.arange(x))] = r.transpose(1, 0, 2)
            self.k.append(rows[0])
            self.v.append(rows[1])

    def index(self, s, positions):
        """Storage indexes [positions, kv_heads, d] of rows of sequence s."""
        c = self.cache
        row = self.table[s, positions // self.page].astype(np.int64) * c.page_stride + positions % self.page * c.row_stride + self.lead
        return row[:, None, None] + np.arange(self.hkv)[:, None] * c.head_stride + np.arange(self.d)

    def upload(self):
        self.buffers = [DeviceBuffer.from_host(to_storage(x, self.dtype)) for x in self.stores]
        self.dev_table = DeviceBuffer.from_host(self.table)
        return [b.view(self.lead) for b in self.buffers]

    def download(self):
        return [from_storage(b.to_host(), self.dtype) for b in self.buffers]


def attention(q, k, v, scale, lens):
    """64-bit attention of q [num_seqs, new, hq, d] over lists of k, v [hkv, len, d]; zeros where nothing is seen."""
    out = np.zeros(q.shape, np.float64)
    new, hq = q.shape[1], q.shape[2]
    for s, n in enumerate(lens):
        for i in range(new):
            sees = n - new + i + 1
            for h in range(hq if sees > 0 else 0):
                hk = h // (hq // k[s].shape[0])
                with np.errstate(all="ignore"):
                    x = k[s][hk, :sees].astype(np.float64) @ q[s, i, h].astype(np.float64) * float(scale)
                    w = np.exp(x - x.max())
                    out[s, i, h] = (w[:, None] * v[s][hk, :sees].astype(np.float64)).sum(0) / w.sum()
    return out


def rotated(x, positions, cosines, sines, rotary, interleaved, dtype):
    """The rotation in `dtype`, each product and sum rounded to it; x [tokens, heads, d]."""
    y = x.astype(dtype).copy()
    c, s = (t[positions].astype(dtype)[:, None] for t in (cosines, sines))
    first = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    a, b = x[..., first].astype(dtype), x[..., second].astype(dtype)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y
