"""Sampling against the definition in 64 bits: the order with its ties, each filter alone and together, what lies at borders, sizes
around the workgroups' pieces, rows that cannot be sampled, and the distribution that the tokens follow."""
import math
from fractions import Fraction

import numpy as np
import pytest

from frankentorch_amd import synth
from frankentorch_amd.device import DeviceBuffer, Stream

pytestmark = pytest.mark.gpu


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(kept tokens in the order of the vocabulary, their weights as multiples of 2^-45 of the largest) of one row, by the definition."""
    order = np.lexsort((np.arange(len(x)), -x))
    with np.errstate(all="ignore"):
        w = np.exp((x[order].astype(np.float64) - float(x.max())) / (float(np.float32(temperature)) if temperature > 0 else 1.0))
    whole = np.rint(w * 2.0 ** 45).astype(np.int64)  # at most 2^17 tokens: their sum fits
    n = 1 if temperature == 0 else int(top_k) if 0 < top_k < len(x) else len(x)
    if top_p < 1:
        upto = np.cumsum(whole[:n])
        n = min(n, int(np.searchsorted(upto, max(1, math.ceil(Fraction(float(np.float32(top_p))) * int(upto[-1]))))) + 1)
    n = min(n, max(1, int((w >= float(np.float32(min_p))).sum())))
    back = np.argsort(order[:n])
    return order[:n][back], whole[:n][back]


def expected(x, u, **kw):
    v, w = kept(x, **kw)
    upto = np.cumsum(w)
    total = int(upto[-1])
    i = int(np.searchsorted(upto, math.floor(Fraction(float(u)) * total), side="right"))
    return int(v[i]), math.log(int(w[i]) / total)


def call(hip, x, u, temperature=None, top_k=None, top_p=None, min_p=None, bad=None, stride=None, lead=0, stream=None, logprobs=True):
    rows, vocab = x.shape
    desc = hip.sample_desc(rows, vocab)
    desc.logits_stride = stride or vocab
    store = np.full(lead + rows * desc.logits_stride, np.nan, np.float32)
    for r in range(rows):
        store[lead + r * desc.logits_stride:][:vocab] = x[r]
    up = lambda a, t: None if a is None else DeviceBuffer.from_host(np.broadcast_to(np.asarray(a, t), (rows,)).copy())
    tokens, lp = DeviceBuffer.from_host(np.full(rows + 2, 77, np.int32)), DeviceBuffer.from_host(np.full(rows + 2, 7.0, np.float32))
    buf = DeviceBuffer.from_host(store)
    hip.sample(desc, buf.view(lead), up(temperature, np.float32), up(top_k, np.int32), up(top_p, np.float32), up(min_p, np.float32), up(u, np.float64), tokens.view(1),
               lp.view(1) if logprobs else None, bad_index=bad, stream=stream)
    hip.synchronize()
    t, l = tokens.to_host(), lp.to_host()
    assert t[0] == t[-1] == 77 and l[0] == l[-1] == 7.0
    return t[1:-1], l[1:-1]


def agree(hip, x, u, **kw):
    t, l = call(hip, x, u, **kw)
    for r in range(len(x)):
        kw_r = {n: (v if np.ndim(v) == 0 else v[r]) for n, v in kw.items() if v is not None and n in ("temperature", "top_k", "top_p", "min_p")}
        token, lp = expected(x[r], u[r], **kw_r)
        if t[r] != token:
            # Weights and sums are held to 2^-45 of the largest weight: where the number is that near to a border, the token on its other side
            v, w = kept(x[r], **kw_r)
            i = int(np.searchsorted(v, t[r]))
            assert i < len(v) and v[i] == t[r], (r, t[r], token, kw_r)
            before, total = int(w[:i].sum()), int(w.sum())
            assert before - len(x[r]) <= u[r] * total <= before + int(w[i]) + len(x[r]), (r, t[r], token, kw_r)
            lp = math.log(max(int(w[i]), 1) / total) if w[i] > 0 else None
        # a rounding of the result, and 2^-24 of the probability where its logarithm is near 0
        assert lp is None or abs(l[r] - lp) <= 2.0 ** -23 * max(1.0, abs(lp)), (r, l[r], lp, kw_r)


def logits(seed, rows, vocab, std=2.0, peak=8.0, ties=False):
    x = synth.normal(seed, "x", (rows, vocab), 0.0, std)
    x += np.where(synth.uniform(seed, "which", (rows, vocab)) < 0.01, synth.uniform(seed, "peak", (rows, vocab)) * peak, 0.0).astype(np.float32)
    return (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32) if ties else x


def numbers(seed, rows):
    return np.random.RandomState(seed).random_sample(rows)


VOCABS = [1, 2, 3, 5, 63, 64, 65, 127, 255, 257, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8193, 16384, 32768, 50257, 65537, 131071]
SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.8, top_k=40, top_p=0.95),
            dict(temperature=1.3, top_p=0.99, min_p=0.001), dict(top_k=700, top_p=0.5), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0), dict(top_k=3000), dict(top_p=0.9999)]


@pytest.mark.parametrize("vocab", VOCABS)
def test_sizes(hip, vocab):
    x = logits(vocab, len(SETTINGS), vocab)
    every = {n: [s.get(n, d) for s in SETTINGS] for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    for seed in range(3):
        agree(hip, x, numbers(seed, len(SETTINGS)), **{n: np.array(v) for n, v in every.items()})


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_each_setting(hip, kw):
    """What is not given is left out; ties at the borders of all filters."""
    for ties in (False, True):
        x = logits(3, 40, 3001, ties=ties)
        agree(hip, x, numbers(4, 40), **{n: (np.full(40, v) if n != "top_k" else np.full(40, v, np.int32)) for n, v in kw.items()})


def test_equal_logits(hip):
    """All equal, or two values: the order is the index, and every filter cuts inside the equal ones."""
    for vocab in (10, 1000, 5000, 50257):
        x = np.zeros((12, vocab), np.float32)
        x[6:, ::3] = -1.0
        x[3, :] = -0.0
        x[4, ::2] = -0.0
        u = numbers(5, 12)
        u[0], u[1] = 0.0, np.nextafter(1.0, 0.0)
        for kw in (dict(), dict(top_k=7), dict(top_p=0.4), dict(top_k=vocab // 2 + 1, top_p=0.7), dict(min_p=0.5), dict(min_p=1.0)):
            agree(hip, x, u, **{n: np.full(12, v) for n, v in kw.items()})


@pytest.mark.parametrize("vocab", [70, 5000, 50257])
def test_the_ends_of_the_numbers(hip, vocab):
    """0 gives the first kept token, the largest number below 1 the last; tokens at -inf or far below are never chosen."""
    x = logits(6, 8, vocab)
    x[:, :vocab // 4] = -np.inf
    x[2, 5] = 3.0
    x[3, vocab - 1] = -np.inf
    x[4] = -np.inf
    x[4, 33] = -5.0
    x[5, :] = np.float32(-3.4028235e38)  # the type's lowest value in masked places
    x[5, 11], x[5, 40] = 1.0, 1.5
    x[6, :] = np.float32(-3.4028235e38)  # and nothing else
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.01), dict(temperature=1e-3), dict(temperature=50.0)):
        for u in (0.0, np.nextafter(1.0, 0.0), 0.5):
            agree(hip, x, np.full(8, u), **{n: np.full(8, v) for n, v in kw.items()})


def test_extreme_values_and_temperatures(hip):
    x = logits(7, 6, 3000)
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(1e-30)
    x[2, 7], x[2, 8] = 3.4028235e38, -3.4028235e38
    x[3] -= np.float32(1e6)
    for t in (1.0, 1e-30, 1e-45, 1e30, 0.01):
        agree(hip, x, numbers(8, 6), temperature=np.full(6, t, np.float32))
        agree(hip, x, numbers(9, 6), temperature=np.full(6, t, np.float32), top_k=np.full(6, 9), top_p=np.full(6, 0.8, np.float32))


def test_rows_that_cannot_be_sampled(hip):
    n = 16
    x = logits(10, n, 2500)
    kw = dict(temperature=np.full(n, 0.9, np.float32), top_k=np.full(n, 30, np.int32), top_p=np.full(n, 0.9, np.float32), min_p=np.full(n, 0.01, np.float32))
    u = numbers(11, n)
    good = [expected(x[r], u[r], **{m: v[r] for m, v in kw.items()}) for r in range(n)]
    x[1, 2400] = np.nan
    x[2, 0] = np.inf
    x[3] = -np.inf
    kw["temperature"][4], kw["temperature"][5], kw["temperature"][6] = -0.5, np.nan, np.inf
    kw["top_k"][7], kw["top_p"][8], kw["top_p"][9], kw["min_p"][10], kw["min_p"][11], kw["min_p"][12] = -1, -0.1, np.nan, -0.1, 1.5, np.nan
    u[13], u[14], u[15] = 1.0, -0.25, np.nan
    bad = DeviceBuffer.from_host(np.array([0], np.int64))
    t, l = call(hip, x, u, bad=bad, **kw)
    assert t[0] == good[0][0] and t[1:].tolist() == [-1] * (n - 1) and np.all(np.isnan(l[1:])) and bad.to_host()[0] == 1
    t, l = call(hip, x[:1], u[:1], bad=bad, **{m: v[:1] for m, v in kw.items()})
    assert t[0] == good[0][0] and bad.to_host()[0] == -1


@pytest.mark.parametrize("stride,lead", [(3000, 0), (3001, 1), (3003, 2), (4096, 3), (3004, 5)])
def test_strides_and_alignments(hip, stride, lead):
    x = logits(12, 9, 3000)
    for kw in (dict(), dict(top_k=np.full(9, 25), top_p=np.full(9, 0.9))):
        agree(hip, x, numbers(13, 9), stride=stride, lead=lead, **kw)


def test_many_rows_and_repeats(hip):
    """More rows than compute units; runs repeat bit for bit, and a row does not depend on its batch."""
    x, u = logits(14, 700, 1500, ties=True), numbers(15, 700)
    kw = dict(temperature=np.linspace(0.5, 1.5, 700).astype(np.float32), top_k=np.arange(700) % 90, top_p=np.linspace(0.3, 1.1, 700).astype(np.float32))
    agree(hip, x, u, **kw)
    a, b = call(hip, x, u, **kw), call(hip, x, u, **kw)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.uint32), b[1].view(np.uint32))
    c = call(hip, x[100:101], u[100:101], **{n: v[100:101] for n, v in kw.items()})
    assert c[0][0] == a[0][100] and c[1][0] == a[1][100]
    assert np.array_equal(call(hip, x, u, logprobs=False, **kw)[0], a[0])


def test_the_distribution(hip):
    """Many draws from one row: every kept token about as often as its probability says (a chi-square of 60 classes stays below 130
    but for one case in a million), no other token ever."""
    one = logits(16, 1, 4000)
    rows = 20000
    x, u = np.repeat(one, rows, 0), (np.arange(rows) + 0.5) / rows
    t, _ = call(hip, x, u, top_k=np.full(rows, 60), top_p=np.full(rows, 0.999))
    v, w = kept(one[0], top_k=60, top_p=0.999)
    share = w / w.sum() * rows
    got = np.array([(t == token).sum() for token in v])
    assert got.sum() == rows
    assert np.sum((got - share) ** 2 / share) < 130
    assert np.all(np.abs(got - share) <= 1.0 + 1e-6)  # even numbers: off by less than one


def test_streams_and_graphs(hip):
    from frankentorch_amd import _lib
    from frankentorch_amd.core import check
    from test_gpu_stream_scratch import Graph

    rows, vocab = 5, 20000
    desc = hip.sample_desc(rows, vocab)
    x, u = DeviceBuffer((rows, vocab)), DeviceBuffer((rows,), np.float64)
    k, p = DeviceBuffer.from_host(np.array([0, 5, 300, 0, 1], np.int32)), DeviceBuffer.from_host(np.array([1.0, 0.9, 0.5, 0.95, 1.0], np.float32))
    tokens = [DeviceBuffer((rows,), np.int32) for _ in range(2)]
    work = [hip.sample_workspace(desc) for _ in range(2)]
    home, side = Stream(), Stream()

    def launch(i, stream):
        hip.sample(desc, x, None, k, p, None, u, tokens[i], workspace=work[i], stream=stream)

    def put(seed):
        values, at = logits(seed, rows, vocab), numbers(seed, rows)
        for b, a in ((x, values), (u, at)):
            check(_lib.load().fth_memcpy_h2d(b.ptr, a.ctypes.data, a.nbytes))
        return values, at

    put(1)
    launch(0, home.handle)
    home.synchronize()
    graph = Graph(home, lambda stream: launch(0, stream))
    for seed in range(20, 30):
        values, at = put(seed)
        graph.replay(side)
        side.synchronize()
        launch(1, home.handle)
        home.synchronize()
        want = [expected(values[r], at[r], top_k=[0, 5, 300, 0, 1][r], top_p=[1.0, 0.9, 0.5, 0.95, 1.0][r])[0] for r in range(rows)]
        assert tokens[0].to_host().tolist() == want and tokens[1].to_host().tolist() == want
    graph.free()
