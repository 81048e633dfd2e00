"""Penalties, biases and masks on logits: bit for bit what stepwise float32 gives, near 64 bits, for every set of steps."""
import numpy as np
import pytest

from frankentorch_amd import _lib, synth
from frankentorch_amd.device import DeviceBuffer, Stream

pytestmark = pytest.mark.gpu


def make(seed, rows, vocab, width):
    u = lambda tag, *a: synth.uniform(seed, tag, *a)
    x = synth.normal(seed, "x", (rows, vocab), 0.0, 3.0)
    history = (u("h", (rows, width)) ** 3 * vocab).astype(np.int32) if width else np.zeros((rows, 0), np.int32)
    hlen = np.minimum(width, (u("hl", (rows,)) * (width + 1)).astype(np.int32)).astype(np.int32)
    plen = np.minimum(hlen, (u("pl", (rows,)) * (hlen + 1)).astype(np.int32)).astype(np.int32)
    rep, freq, pres = u("r", (rows,), 0.8, 1.5), u("f", (rows,), -0.2, 0.7), u("p", (rows,), -0.2, 0.7)
    bias = np.where(u("b", (rows, vocab)) < 0.1, synth.normal(seed, "bv", (rows, vocab)), 0).astype(np.float32)
    mask = (u("m", (rows, vocab)) < 0.3)
    if rows > 2:
        mask[1] = False  # nothing is allowed
        mask[2] = True
    return dict(x=x, history=history, hlen=hlen, plen=plen, rep=rep, freq=freq, pres=pres, bias=bias, mask=mask)


def words(mask):
    rows, vocab = mask.shape
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint8)
    bits[:, :vocab] = mask
    bits[:, vocab:] = np.arange(bits.shape[1] - vocab) % 2  # bits past the vocabulary mean nothing
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def plain(m, use, kind, shared=False):
    x, vocab = m["x"].astype(kind), m["x"].shape[1]
    out = np.empty_like(x)
    for r in range(len(x)):
        z = x[r].copy()
        seen = np.zeros(vocab, bool)
        seen[m["history"][r, : m["hlen"][r]]] = True
        made = np.bincount(m["history"][r, m["plen"][r]: m["hlen"][r]], minlength=vocab)
        with np.errstate(invalid="ignore", over="ignore"):
            if "rep" in use:
                rep = kind(m["rep"][r])
                z = np.where(seen, np.where(z > 0, z / rep, z * rep), z)
            if "freq" in use:
                z = np.where(made > 0, z - kind(m["freq"][r]) * made.astype(kind), z)
            if "pres" in use:
                z = np.where(made > 0, z - kind(m["pres"][r]), z)
            if "bias" in use:
                z = z + m["bias"][0 if shared else r].astype(kind)
        if "mask" in use:
            z = np.where(m["mask"][r], z, -np.inf)
        out[r] = z
    return out


def run(hip, m, use, shared=False, in_place=False, bad=None, pad=0, lead=0, stream=None):
    rows, vocab = m["x"].shape
    desc = hip.logits_desc(rows, vocab, m["history"].shape[1], shared)
    desc.logits_stride = desc.out_stride = vocab + pad
    store = np.full(lead + rows * (vocab + pad), 7.0, np.float32)
    store[lead:].reshape(rows, -1)[:, :vocab] = m["x"]
    x, out = DeviceBuffer.from_host(store), DeviceBuffer.from_host(np.full_like(store, 7.0))
    if in_place:
        out = x
    put = lambda n: DeviceBuffer.from_host(np.ascontiguousarray(m[n])) if n in use else None
    hist = {"rep", "freq", "pres"} & set(use)
    h = [DeviceBuffer.from_host(m[n]) if hist else None for n in ("history", "hlen", "plen")]
    bias = None if "bias" not in use else DeviceBuffer.from_host(np.ascontiguousarray(m["bias"][0] if shared else m["bias"]))
    mask = DeviceBuffer.from_host(words(m["mask"])) if "mask" in use else None
    hip.logits_process(desc, x.view(lead), *h, put("rep"), put("freq"), put("pres"), bias, mask, out.view(lead), bad, stream)
    hip.synchronize()
    got = out.to_host()
    assert np.all(got[:lead] == 7.0) and np.all(got[lead:].reshape(rows, -1)[:, vocab:] == 7.0)
    return got[lead:].reshape(rows, -1)[:, :vocab]


ALL = ("rep", "freq", "pres", "bias", "mask")


@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (1, 31, 5), (3, 32, 0), (4, 33, 40), (2, 1000, 1), (5, 4095, 300), (3, 4096, 2000), (3, 4097, 5000), (1, 50257, 200), (7, 50257, 1024),
                                              (4, 8193, 17), (3, 16385, 4096), (40, 12345, 777), (2, 131071, 9000)])
def test_against_stepwise_float32(hip, rows, vocab, width):
    m = make(41, rows, vocab, width)
    bad = DeviceBuffer((1,), np.int64)
    got = run(hip, m, ALL, bad=bad)
    assert bad.to_host()[0] == -1
    assert np.array_equal(got, plain(m, ALL, np.float32))
    ref = plain(m, ALL, np.float64)
    fine = np.isfinite(ref)
    # five roundings of numbers below |x| rep + |f| n + |p| + |b|
    size = np.abs(m["x"]).max() * 1.5 + 0.7 * (width + 1) + np.abs(m["bias"]).max() + 1
    assert np.all(np.abs(got[fine] - ref[fine]) <= 5 * 2.0 ** -24 * size)
    assert np.array_equal(run(hip, m, ALL, in_place=True), got)


@pytest.mark.parametrize("use", [(), ("rep",), ("freq",), ("pres",), ("bias",), ("mask",), ("rep", "mask"), ("freq", "pres"), ("bias", "mask"), ("rep", "bias")])
@pytest.mark.parametrize("shared,pad,lead", [(False, 0, 0), (True, 3, 0), (False, 1, 1), (True, 0, 2), (True, 4, 4)])
def test_every_step_alone_and_any_stride(hip, use, shared, pad, lead):
    m = make(42, 5, 4999, 333)
    assert np.array_equal(run(hip, m, use, shared, pad=pad, lead=lead), plain(m, use, np.float32, shared))


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 29, 30, 61, 4093, 4094, 4095, 4096, 4097, 8189, 8192, 8195])
@pytest.mark.parametrize("pad,lead", [(0, 0), (0, 1), (1, 2), (2, 3), (4, 0), (3, 1)])
def test_rows_that_start_anywhere(hip, vocab, pad, lead):
    m = make(45, 6, vocab, 50)
    want = plain(m, ALL, np.float32)
    assert np.array_equal(run(hip, m, ALL, pad=pad, lead=lead), want)
    assert np.array_equal(run(hip, m, ALL, pad=pad, lead=lead, in_place=True), want)
    m["history"][3, 0], m["hlen"][3] = -1 - lead, max(m["hlen"][3], 1)  # just before the row
    bad = DeviceBuffer((1,), np.int64)
    got = run(hip, m, ALL, pad=pad, lead=lead, bad=bad)
    assert bad.to_host()[0] == 3 and np.all(got[3] == 7.0) and np.array_equal(np.delete(got, 3, 0), np.delete(want, 3, 0))


def test_values_that_are_not_finite(hip):
    """A masked place is -inf whatever was there; NaN and infinities elsewhere go through the steps."""
    m = make(43, 3, 500, 60)
    m["x"][:, ::7], m["x"][:, 1::7], m["x"][:, 2::7] = np.nan, np.inf, -np.inf
    m["bias"][:, ::11] = -np.inf
    got, ref = run(hip, m, ALL), plain(m, ALL, np.float32)
    assert np.array_equal(got, ref, equal_nan=True)
    assert np.all(got[~m["mask"]] == -np.inf)


def test_many_counts_of_one_token(hip):
    m = make(44, 2, 100, 70000)
    m["history"][:] = 42
    m["hlen"][:], m["plen"][:] = 70000, (0, 69999)
    assert np.array_equal(run(hip, m, ("freq",)), plain(m, ("freq",), np.float32))


@pytest.mark.parametrize("vocab", [700, 50257])
def test_invalid_rows_are_left_alone(hip, vocab):
    m = make(45, 8, vocab, 50)
    m["hlen"][:], m["plen"][:] = 50, 10
    bad = DeviceBuffer((1,), np.int64)
    m["history"][6, 49], m["history"][4, 0], m["history"][3, 20] = vocab, -1, 2 ** 31 - 1
    m["hlen"][5], m["plen"][5] = 51, 0
    m["plen"][7] = 51
    ref = plain({**m, "history": np.clip(m["history"], 0, vocab - 1), "hlen": np.minimum(m["hlen"], 50), "plen": np.minimum(m["plen"], 50)}, ALL, np.float32)
    got = run(hip, m, ALL, bad=bad)
    assert bad.to_host()[0] == 3
    assert np.all(got[3:] == 7.0) and np.array_equal(got[:3], ref[:3])
    m["hlen"][1], m["plen"][0] = -1, -1
    run(hip, m, ALL, bad=bad)
    assert bad.to_host()[0] == 0
    m["history"][:, 45:] = -5  # past the length: not looked at
    m["hlen"][:], m["plen"][:] = 45, 45
    m["history"][4, 0] = m["history"][3, 20] = 9
    got = run(hip, m, ALL, bad=bad)
    assert bad.to_host()[0] == -1
    assert np.array_equal(got, plain({**m, "history": np.clip(m["history"], 0, vocab - 1)}, ALL, np.float32))


def test_stream_and_graph(hip):
    from test_gpu_stream_scratch import Graph

    m = make(46, 4, 50257, 128)
    desc = hip.logits_desc(4, 50257, 128)
    bufs = [DeviceBuffer.from_host(np.ascontiguousarray(a)) for a in (m["x"], m["history"], m["hlen"], m["plen"], m["rep"], m["freq"], m["pres"], m["bias"], words(m["mask"]))]
    out, bad, home, side = DeviceBuffer(m["x"].shape), DeviceBuffer((1,), np.int64), Stream(), Stream()
    call = lambda stream: hip.logits_process(desc, *bufs, out, bad, stream)
    call(home.handle)
    home.synchronize()
    graph = Graph(home, call)
    for n in (128, 5, 0, 77):
        m["hlen"][:], m["plen"][:] = n, n // 2
        for b, a in ((bufs[2], m["hlen"]), (bufs[3], m["plen"])):
            _lib.load().fth_memcpy_h2d(b.ptr, a.ctypes.data, a.nbytes)
        graph.replay(side)
        hip.synchronize()
        assert bad.to_host()[0] == -1 and np.array_equal(out.to_host(), plain(m, ALL, np.float32))
    graph.free()


def test_no_rows(hip):
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    for rows, vocab in ((0, 10), (3, 0)):
        hip.logits_process(hip.logits_desc(rows, vocab), None, None, None, None, None, None, None, None, None, None, bad)
        assert bad.to_host()[0] == -1
