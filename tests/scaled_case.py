"""Paged caches of 8-bit numbers for the tests: the two types and the append's rules written out with numpy."""
import numpy as np

from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer, paged_cache, paged_scales

LARGEST = {"i8": 127.0, "e4m3": 448.0}


def _e4m3_values():
    bits = np.arange(256)
    sign, e, m = np.where(bits & 128, -1.0, 1.0), (bits >> 3) & 15, bits & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v[(bits & 127) == 127] = np.nan
    return sign * v


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]  # ascending, code = index


def values(codes, dtype):
    """What uint8 codes stand for, before their scale (float64)."""
    return codes.view(np.int8).astype(np.float64) if dtype == "i8" else E4M3[codes]


def codes(x, dtype):
    """Numbers within the type's range to the nearest code, ties to the even one; 0 for what is not finite."""
    x = np.where(np.isfinite(x), x, 0.0).astype(np.float64)
    if dtype == "i8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(x), 448.0)
    lo = np.clip(np.searchsorted(_POSITIVE, a, side="right") - 1, 0, 126)
    hi = np.minimum(lo + 1, 126)
    below, over = a - _POSITIVE[lo], _POSITIVE[hi] - a
    up = (over < below) | ((over == below) & (lo % 2 == 1))
    c = np.where((hi > lo) & up, hi, lo).astype(np.uint8)
    return np.where(np.signbit(x), c | 128, c).astype(np.uint8)


def needed_scale(largest, dtype):
    """The smallest power of two, 2^-126 at least, whose LARGEST multiples reach `largest`."""
    if largest == 0:
        return 0.0
    if not np.isfinite(largest):
        return np.nan
    e = -126
    while LARGEST[dtype] * 2.0 ** e < largest:
        e += 1
    return 2.0 ** e


class Scaled:
    """Caches of pages in no order, kept on the host as codes and scales next to the device's. Whatever no sequence owns holds the
    codes of the largest number (e4m3: NaN) and NaN scales. `lens`: positions that are filled already, through `append`."""

    def __init__(self, seed, seqs, hkv, d, page, block, dtype, max_pages, pad=0, lead=0, heads_inside=False, scale_pad=0):
        self.hkv, self.d, self.page, self.block, self.dtype = hkv, d, page, block, dtype
        total = seqs * max_pages + 2
        self.cache = c = paged_cache(total, page, hkv, d, seqs, max_pages, dtype)
        if heads_inside:
            c.head_stride, c.row_stride = d + pad, hkv * (d + pad)
        else:
            c.row_stride, c.head_stride = d + pad, page * (d + pad)
        c.page_stride = hkv * page * (d + pad)
        self.sc = s = paged_scales(c, block)
        s.head_stride += scale_pad
        s.page_stride = hkv * s.head_stride
        self.table = np.argsort(synth.uniform(seed, "pages", (total,)))[:seqs * max_pages].reshape(seqs, max_pages).astype(np.int32)
        self.lead = lead
        junk = 127 if dtype == "e4m3" else 128
        self.codes = [np.full(lead + total * c.page_stride, junk, np.uint8) for _ in range(2)]
        self.scales = [np.full(total * s.page_stride, np.nan, np.float32) for _ in range(2)]

    def row_at(self, s, pos, h):
        c = self.cache
        return self.lead + int(self.table[s, pos // self.page]) * c.page_stride + h * c.head_stride + (pos % self.page) * c.row_stride

    def scale_at(self, s, pos, h):
        return int(self.table[s, pos // self.page]) * self.sc.page_stride + h * self.sc.head_stride + (pos % self.page) // self.block

    def append(self, which, s, pos, x):
        """Rows x [tokens, heads, d] of K (0) or V (1) from position pos on, all of one block, by the rules."""
        cod, sc = self.codes[which], self.scales[which]
        start = pos - pos % self.block
        for h in range(self.hkv):
            at = self.scale_at(s, pos, h)
            had = float(sc[at]) if pos > start else 0.0
            need = needed_scale(np.max(np.abs(x[:, h])) if np.all(np.isfinite(x[:, h])) else np.inf, self.dtype)
            now = np.nan if np.isnan(had) or np.isnan(need) else max(had, need)
            per = 1.0 / now if now > 0 else 0.0
            if not now == had:
                for p in range(start, pos):
                    r = self.row_at(s, p, h)
                    cod[r:r + self.d] = codes(values(cod[r:r + self.d], self.dtype) * (had * per), self.dtype)
            sc[at] = now
            for i in range(len(x)):
                r = self.row_at(s, pos + i, h)
                with np.errstate(invalid="ignore"):
                    cod[r:r + self.d] = codes(x[i, h].astype(np.float64) * per, self.dtype)

    def rows(self, which, s, n):
        """What the first n positions of a sequence stand for: [heads, n, d], exactly, in float64."""
        out = np.zeros((self.hkv, n, self.d))
        for p in range(n):
            for h in range(self.hkv):
                r = self.row_at(s, p, h)
                out[h, p] = values(self.codes[which][r:r + self.d], self.dtype) * float(self.scales[which][self.scale_at(s, p, h)])
        return out

    def fill(self, seed, lens, std=1.0, spread=0.7):
        """Random rows in the first lens[s] positions of each sequence, whole blocks at a time."""
        for which in range(2):
            for s, n in enumerate(lens):
                n = max(n, 0)
                x = synth.normal(seed, "%d.%d" % (which, s), (n, self.hkv, self.d), 0.0, std) * np.exp(synth.normal(seed, "s%d.%d" % (which, s), (n, self.hkv, 1), 0.0, spread))
                for p0 in range(0, n, self.block):
                    rows = x[p0:p0 + self.block]
                    for h in range(self.hkv):
                        need = needed_scale(np.max(np.abs(rows[:, h])), self.dtype)
                        self.scales[which][self.scale_at(s, p0, h)] = need
                        for i in range(len(rows)):
                            r = self.row_at(s, p0 + i, h)
                            self.codes[which][r:r + self.d] = codes(rows[i, h].astype(np.float64) / need, self.dtype)
        return self

    def upload(self):
        self.buffers = [DeviceBuffer.from_host(x) for x in self.codes]
        self.scale_buffers = [DeviceBuffer.from_host(x) for x in self.scales]
        self.dev_table = DeviceBuffer.from_host(self.table)
        return [b.view(self.lead) for b in self.buffers] + self.scale_buffers
