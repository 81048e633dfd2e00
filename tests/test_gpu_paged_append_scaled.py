"""Appends to a cache of 8-bit numbers against the rules written out block by block: codes, scales and rotated queries bit for bit."""
import numpy as np
import pytest

from frankentorch_amd import _lib, synth
from frankentorch_amd.core import check
from frankentorch_amd.device import DeviceBuffer, Stream, rotary_tables
from paged_case import rotated
from scaled_case import Scaled

pytestmark = pytest.mark.gpu


class Call:
    """One append of tokens at (sequence, position) with the operands of a packed projection, on the device and by the rules."""

    def __init__(self, p, seed, places, hq=0, rotary=0, interleaved=False, max_pos=0, pad=0, lead=0, std=1.0):
        self.p, self.hq, self.rotary, self.inter, self.max_pos, self.lead = p, hq, rotary, interleaved, max_pos, lead
        self.seqs, self.positions = (np.array([x[i] for x in places], np.int32) for i in range(2))
        t, width = len(places), (hq + 2 * p.hkv) * p.d + pad
        self.proj = synth.normal(seed, "proj", (t, width), 0.0, std) * np.exp(synth.normal(seed, "size", (t, 1), 0.0, 1.0)).astype(np.float32)
        self.pitch = width
        self.cos, self.sin = rotary_tables(max_pos, rotary) if rotary else (None, None)

    def heads(self, first, n):
        return self.proj[:, first * self.p.d:(first + n) * self.p.d].reshape(len(self.proj), n, self.p.d)

    def expect(self):
        """The rules on the host's cache; the rotated queries."""
        p, hq = self.p, self.hq
        q, k, v = self.heads(0, hq), self.heads(hq, p.hkv), self.heads(hq + p.hkv, p.hkv)
        if self.rotary:
            where = np.clip(self.positions, 0, self.max_pos - 1)
            q, k = (rotated(x, where, self.cos, self.sin, self.rotary, self.inter, np.float32) for x in (q, k))
        t = 0
        while t < len(self.positions):  # a run: the tokens of one block
            s, pos, n = self.seqs[t], self.positions[t], 1
            while t + n < len(self.positions) and self.seqs[t + n] == s and self.positions[t + n] == pos + n and (pos + n) % p.block:
                n += 1
            p.append(0, s, pos, k[t:t + n])
            p.append(1, s, pos, v[t:t + n])
            t += n
        return q

    def run(self, hip, device, bad=None, stream=None, in_place=False):
        p = self.p
        buf = DeviceBuffer.from_host(np.concatenate([np.zeros(self.lead, np.float32), self.proj.ravel()]))
        desc = hip.paged_append_desc(p.cache, len(self.proj), self.hq, self.rotary, self.max_pos, self.inter, row_stride=self.pitch)
        out = DeviceBuffer.from_host(np.full((len(self.proj), max(self.hq, 1), p.d), 7.0, np.float32))
        if in_place:
            desc.out_row_stride = self.pitch
        cos, sin = (None if x is None else DeviceBuffer.from_host(x) for x in (self.cos, self.sin))
        at = lambda heads: buf.view(self.lead + heads * p.d)
        q = at(0) if self.hq else None
        hip.paged_append_scaled(p.cache, p.sc, desc, q, at(self.hq), at(self.hq + p.hkv), cos, sin, p.dev_table, DeviceBuffer.from_host(self.seqs),
                                DeviceBuffer.from_host(self.positions), (q if in_place else out) if self.hq else None, *device, bad_index=bad, stream=stream)
        hip.synchronize()
        return buf.to_host()[self.lead:].reshape(self.proj.shape)[:, :self.hq * p.d].reshape(-1, self.hq, p.d) if in_place else out.to_host()


def same(p):
    for got, want in zip(p.buffers, p.codes):
        # -0 and 0 are one number
        got = got.to_host()
        zero = lambda x: np.where(x == 128, 0, x) if p.dtype == "e4m3" else x
        assert np.array_equal(zero(got), zero(want))
    for got, want in zip(p.scale_buffers, p.scales):
        assert np.array_equal(got.to_host(), want, equal_nan=True)


def ragged(counts, starts):
    return [(s, a + i) for s, (n, a) in enumerate(zip(counts, starts)) for i in range(n)]


# (counts, starts, hq, hkv, d, page, block, rotary, interleaved, dtype)
CASES = [
    ([1], [0], 0, 1, 64, 16, 16, 0, False, "e4m3"), ([1, 1, 1], [3, 16, 31], 4, 2, 64, 16, 16, 64, False, "i8"), ([16, 15, 17], [0, 1, 15], 2, 2, 64, 16, 16, 0, False, "e4m3"),
    ([33, 0, 70], [5, 0, 30], 8, 2, 128, 16, 16, 128, False, "e4m3"), ([100, 3], [0, 47], 4, 4, 128, 48, 48, 64, True, "i8"), ([40, 41], [9, 90], 4, 1, 128, 32, 1, 128, True, "e4m3"),
    ([130, 64], [0, 64], 12, 12, 64, 64, 64, 0, False, "i8"), ([300], [17], 2, 1, 128, 256, 256, 128, False, "e4m3"), ([21, 9], [2, 6], 3, 3, 80, 8, 4, 40, False, "i8"),
    ([50, 20], [0, 5], 4, 2, 256, 16, 8, 256, False, "e4m3"), ([30, 7], [1, 3], 2, 1, 20, 6, 3, 10, True, "i8"), ([11, 5], [0, 2], 2, 2, 7, 5, 5, 6, False, "e4m3"),
    ([60], [3], 1, 1, 1, 16, 2, 0, False, "i8"), ([90, 31], [7, 0], 32, 8, 128, 24, 24, 128, False, "e4m3"), ([47, 1, 2], [0, 600, 5], 5, 1, 96, 128, 128, 32, True, "i8"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_by_the_rules(hip, case):
    counts, starts, hq, hkv, d, page, block, rotary, inter, dtype = case
    p = Scaled(31, len(counts), hkv, d, page, block, dtype, -(-max(a + n for a, n in zip(starts, counts)) // page)).fill(32, starts)
    device = p.upload()
    call = Call(p, 33, ragged(counts, starts), hq, rotary, inter, 1000 if rotary else 0)
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    got, want = call.run(hip, device, bad), call.expect()
    same(p)
    if hq:
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    assert bad.to_host()[0] == -1


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("pad,lead,heads_inside,scale_pad,operand_pad,operand_lead", [(0, 0, True, 0, 0, 0), (8, 16, False, 3, 4, 4), (3, 0, False, 0, 0, 0), (0, 1, False, 1, 0, 0),
                                                                                    (0, 0, False, 0, 3, 0), (4, 4, True, 0, 0, 1)])
def test_layouts_and_alignments(hip, dtype, pad, lead, heads_inside, scale_pad, operand_pad, operand_lead):
    p = Scaled(34, 3, 2, 64, 16, 8, dtype, 5, pad, lead, heads_inside, scale_pad).fill(35, [9, 0, 20])
    device = p.upload()
    for in_place in (False, True):
        call = Call(p, 36, ragged([20, 3, 11], [9, 0, 20]), 4, 32, False, 80, operand_pad, operand_lead)
        got, want = call.run(hip, device, in_place=in_place), call.expect()
        same(p)  # nothing between the rows is written
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_token_by_token_gives_a_prompts_scales(hip, dtype):
    """Steps of one token, each of which may raise the scale of what the block holds, against one call; and back again after a cut."""
    n = 70
    one, steps = (Scaled(37, 1, 2, 64, 32, 16, dtype, 3) for _ in range(2))
    whole = Call(one, 38, ragged([n], [0]))
    whole.proj *= np.exp(np.linspace(-3, 3, n))[:, None].astype(np.float32)  # scales grow in every block
    whole.run(hip, one.upload())
    device = steps.upload()
    for i in list(range(n)) + list(range(40, n)):  # cut back to 40 positions once, and on from there
        call = Call(steps, 38, [(0, i)])
        call.proj = whole.proj[i:i + 1]
        call.run(hip, device)
        call.expect()
    same(steps)
    for a, b in zip(one.scale_buffers, steps.scale_buffers):
        a, b = a.to_host(), b.to_host()
        cut = one.scale_at(0, 40, 0), one.scale_at(0, 40, 1)  # a block that was cut keeps the scale that it had grown to
        keep = np.ones(a.shape, bool)
        keep[list(cut)] = False
        assert np.array_equal(a[keep], b[keep], equal_nan=True)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_zeros_smallest_and_largest(hip, dtype):
    """Blocks of zeros, elements at both ends of float32, at the border of a scale and halfway between two codes."""
    p = Scaled(39, 1, 1, 64, 16, 4, dtype, 4)
    device = p.upload()
    call = Call(p, 40, ragged([24], [0]))
    x = call.proj[:, :64]
    top = 127.0 if dtype == "i8" else 448.0
    x[0:4] = 0.0
    x[4] = np.float32(1e-45)
    x[5:8] *= np.float32(1e-38)
    x[8:12] *= np.float32(1e36)
    x[12:16] = 0.5
    x[12, 0] = top                                  # the largest code exactly
    x[13, :16] = np.arange(16) + 0.5                # ties
    x[14, :16] = np.nextafter(np.arange(16, dtype=np.float32) + 0.5, 0)
    x[16:20] = 0.25
    x[16, 0] = np.nextafter(np.float32(top), np.float32(1e9))  # just above it: the next scale
    x[20:24] = -np.abs(x[20:24])
    call.proj[:, 64:] = x[::-1]
    call.run(hip, device)
    call.expect()
    same(p)
    step = Call(p, 41, [(0, 24), (0, 25)])  # a zero first, then something: a scale that begins at 0
    step.proj[0] = 0.0
    for i in range(2):
        part = Call(p, 41, [(0, 24 + i)])
        part.proj = step.proj[i:i + 1]
        part.run(hip, device)
        part.expect()
    same(p)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_makes_its_block_nan(hip, dtype, value):
    p = Scaled(42, 1, 2, 64, 16, 8, dtype, 4).fill(43, [20])
    device = p.upload()
    call = Call(p, 44, ragged([25], [20]))
    call.proj[1, 5] = value          # K, head 0, position 21: into a block that holds four rows
    call.proj[12, 3 * 64 + 9] = value  # V, head 1, position 32, the first of its block
    call.run(hip, device)
    call.expect()
    same(p)
    assert np.isnan(p.scales[0]).any()
    again = Call(p, 45, ragged([8], [32]))  # the block anew
    again.run(hip, device)
    again.expect()
    same(p)
    assert np.isfinite(p.scales[1][p.scale_at(0, 32, 1)])


def test_what_is_left_out_and_reported(hip):
    """Padding, places that do not exist, and tokens that do not follow each other in their block."""
    p = Scaled(46, 3, 2, 64, 16, 16, "e4m3", 3).fill(47, [4, 4, 0])
    p.table[1, 2] = 99
    device = p.upload()
    bad = DeviceBuffer.from_host(np.array([0], np.int64))
    places = [(0, -1), (0, 4), (0, 5), (2, -1), (2, 0), (1, 4), (7, 0), (1, 40), (0, 48), (-1, 3)]
    call = Call(p, 48, places, hq=2, rotary=64, max_pos=60)
    got = call.run(hip, device, bad)
    keep = [1, 2, 4, 5]
    assert bad.to_host()[0] == 6
    fine = Call(p, 48, places, hq=2, rotary=64, max_pos=60)
    fine.proj, fine.seqs, fine.positions = fine.proj[keep], fine.seqs[keep], fine.positions[keep]
    want = fine.expect()
    assert np.array_equal(got[keep], want)
    same(p)
    for t in (0, 3, 6, 7, 8, 9):
        assert np.all(got[t] == 7.0)


def test_runs_that_do_not_ascend_are_reported(hip):
    p = Scaled(49, 2, 1, 64, 16, 16, "i8", 2).fill(50, [3, 0])
    device = p.upload()
    bad = DeviceBuffer.from_host(np.array([0], np.int64))
    places = [(0, 3), (0, 4), (0, 4), (1, 0), (1, 1), (0, 16), (0, 18)]  # the second (0, 4) and (0, 18) are left out
    call = Call(p, 51, places)
    call.run(hip, device, bad)
    keep = [0, 1, 3, 4, 5]
    call.proj, call.seqs, call.positions = call.proj[keep], call.seqs[keep], call.positions[keep]
    call.expect()
    same(p)
    assert bad.to_host()[0] == 2


def test_queries_alone_and_nothing(hip):
    """With k and v NULL the call is the rotation of queries; no tokens are nothing to do."""
    p = Scaled(52, 1, 1, 64, 16, 16, "i8", 2)
    device = p.upload()
    x = synth.normal(53, "q", (5, 3, 64))
    pos = np.array([0, 9, -1, 31, 2], np.int32)
    cos, sin = rotary_tables(40, 64)
    out = DeviceBuffer.from_host(np.full(x.shape, 7.0, np.float32))
    desc = hip.paged_append_desc(p.cache, 5, 3, 64, 40)
    hip.paged_append_scaled(p.cache, p.sc, desc, DeviceBuffer.from_host(x), None, None, DeviceBuffer.from_host(cos), DeviceBuffer.from_host(sin), None, None,
                            DeviceBuffer.from_host(pos), out, None, None, None, None)
    hip.synchronize()
    want = rotated(x, np.maximum(pos, 0), cos, sin, 64, False, np.float32)
    want[2] = 7.0
    assert np.array_equal(out.to_host(), want)
    desc.tokens = 0
    hip.paged_append_scaled(p.cache, p.sc, desc, None, *device[:2], None, None, None, None, None, None, *device)
    hip.synchronize()
    same(p)


def test_streams_and_graphs(hip):
    """A captured step, replayed on another stream with other positions and values each time, against the rules."""
    from test_gpu_stream_scratch import Graph

    p = Scaled(54, 4, 2, 64, 16, 16, "e4m3", 4).fill(55, [30, 16, 0, 15])
    device = p.upload()
    home, side = Stream(), Stream()
    cos, sin = rotary_tables(128, 64)
    desc = hip.paged_append_desc(p.cache, 4, 2, 64, 128, row_stride=6 * 64)
    proj, cosines, sines, seqs, where = (DeviceBuffer.from_host(a) for a in (np.zeros((4, 6 * 64), np.float32), cos, sin, np.arange(4, dtype=np.int32), np.full(4, -1, np.int32)))
    out = DeviceBuffer((4, 2, 64))

    def call(stream):
        hip.paged_append_scaled(p.cache, p.sc, desc, proj, proj.view(128), proj.view(256), cosines, sines, p.dev_table, seqs, where, out, *device, stream=stream)

    call(home.handle)
    home.synchronize()
    graph = Graph(home, call)
    for step in range(20):
        positions = np.array([30, 16, 0, 15], np.int32) + step
        positions[step % 4] = -1 if step == 19 else positions[step % 4]
        one = Call(p, 56 + step, [(s, int(x)) for s, x in enumerate(positions)], 2, 64, False, 128)
        for b, a in ((proj, one.proj), (where, positions)):
            check(_lib.load().fth_memcpy_h2d(b.ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes))
        if step % 3:
            graph.replay(side)
            side.synchronize()
        else:
            call(home.handle)
            home.synchronize()
        keep = positions >= 0
        one.proj, one.seqs, one.positions = one.proj[keep], one.seqs[keep], one.positions[keep]
        assert np.array_equal(out.to_host()[keep], one.expect())
    same(p)
    graph.free()
