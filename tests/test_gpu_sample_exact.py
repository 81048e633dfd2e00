"""Sampling against weights in 64 bits that are rounded nowhere: log-probabilities of unlikely tokens, the ends and borders of the numbers,
and vocabularies above 131072 tokens, where a lane of the choice has several pieces of a row and, further on, the row too many to list."""
import math

import numpy as np
import pytest

from frankentorch_amd.device import DeviceBuffer, Stream
from test_gpu_sample import call, numbers

pytestmark = pytest.mark.gpu


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(kept tokens in the order of the vocabulary, their weights) of one row, by the definition."""
    order = np.argsort(-x, kind="stable")
    order = order[:np.count_nonzero(x > -np.inf)]
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((x[order].astype(np.float64) - float(x.max())) / (float(np.float32(temperature)) if temperature > 0 else 1.0))
    n = 1 if temperature == 0 else int(top_k) if 0 < top_k < len(w) else len(w)
    if top_p < 1:
        n = min(n, int(np.searchsorted(np.cumsum(w[:n]), float(np.float32(top_p)) * math.fsum(w[:n]))) + 1)
    n = min(n, max(1, int((w >= float(np.float32(min_p))).sum())))
    back = np.argsort(order[:n])
    return order[:n][back], w[:n][back]


def running(w):
    """Sums up to each weight, in extended precision: in 64 bits those of 2^20 weights are off by more than the kernels' sums are."""
    return np.cumsum(w.astype(np.longdouble))


def agree(hip, x, u, **kw):
    """Every row has a kept token whose stretch of the weights the number lies in, to 2^-46 of their sum (a number rarely lies as near to a border, but
    for those put there), and the logarithm of its share: a rounding to float32, and what fp64 exponentials of up to 2^10 are off by."""
    t, l = call(hip, x, u, **kw)
    memo = {}
    for r in range(len(x)):
        kw_r = {n: (v if np.ndim(v) == 0 else v[r]) for n, v in kw.items() if n in ("temperature", "top_k", "top_p", "min_p")}
        key = (x[r].ctypes.data,) + tuple(sorted((n, float(v)) for n, v in kw_r.items()))
        if key not in memo:
            v, w = kept(x[r], **kw_r)
            memo[key] = v, w, running(w), math.fsum(w)
        v, w, upto, total = memo[key]
        i = int(np.searchsorted(v, t[r]))
        assert i < len(v) and v[i] == t[r] and w[i] > 0, (r, t[r], u[r], kw_r)
        near = total * 2.0 ** -46
        assert upto[i] - w[i] - near <= np.longdouble(u[r]) * total <= upto[i] + near, (r, t[r], u[r], kw_r)
        lp = math.log(w[i] / total)
        assert abs(l[r] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -36, (r, t[r], l[r], lp, kw_r)
    return t, l


@pytest.mark.parametrize("kw", [dict(top_k=41), dict(top_k=500), dict(min_p=1e-30), dict(top_k=45, min_p=1e-27), dict(top_k=20000), dict(top_k=20000, min_p=1e-30), dict()], ids=str)
def test_unlikely_tokens(hip, kw):
    """40 tokens at 2^-20 to 2^-85 of the largest weight stand before all others, and the numbers lead to each of them."""
    vocab = 50257
    x = np.random.RandomState(1).normal(-80.0, 2.0, (1, vocab)).astype(np.float32)
    x[0, :40] = np.linspace(-14.0, -59.0, 40)
    x[0, 20000] = 0.0
    v, w = kept(x[0], **kw)
    assert np.array_equal(v[:40], np.arange(40))
    middle = (running(w) - w / 2)[:40].astype(np.float64) / math.fsum(w)
    u = np.concatenate([[0.0, 2.0 ** -90], middle[::-1], middle, [2.0 ** -10, 0.5]])
    rows = len(u)
    t, l = call(hip, np.repeat(x, rows, 0), u, **{n: np.full(rows, s) for n, s in kw.items()})
    # Sums of fp64 weights, largest 1: the k-th token of a descending line starts where the ones before it end, to 2^-53 of what they weigh
    back = np.argsort(-w[:40])  # (they descend)
    assert np.array_equal(back, np.arange(40))
    for r in range(rows):
        i = int(np.searchsorted(v, t[r]))
        assert v[i] == t[r] and abs(l[r] - math.log(w[i] / math.fsum(w))) <= 2.0 ** -24 * abs(l[r]) + 2.0 ** -36, (r, t[r], l[r])
    assert t[0] == 0 and t[1] == 0
    assert t[2:42].tolist() == t[42:82].tolist()[::-1]
    # to 2^-50 of the likelier ones before it: the first dozen tokens are told apart
    assert t[42:42 + 12].tolist() == list(range(12)) and t[-1] == 20000


def test_the_first_token_that_is_kept(hip):
    """0 and the smallest numbers lead to the first kept token that has any weight, however little."""
    for vocab, at in ((70, 3), (5000, 1), (50257, 31000)):
        for low in (-30.0, -40.0, -100.0, -600.0):
            x = np.full((6, vocab), -np.inf, np.float32)
            x[:, at] = low
            x[:, at + 7] = 1.0
            x[:, at + 9] = 0.5
            u = np.array([0.0, 1e-320, 2.0 ** -1000, 0.0, 0.3, 0.9])
            for kw in (dict(top_k=3), dict(top_k=10, temperature=0.9), dict(top_k=2), dict()):
                t, _ = agree(hip, x, u, **{n: np.full(6, v) for n, v in kw.items()})
                assert t[0] == t[3] == (at if kw.get("top_k") != 2 else at + 7)


def borders(x, rows, seed, **kw):
    """Numbers at and a few units in the last place around borders between kept tokens."""
    v, w = kept(x, **kw)
    rng = np.random.RandomState(seed)
    upto = running(w)
    u = (upto[rng.randint(0, len(v), rows)] / upto[-1]).astype(np.float64)
    return np.clip(u + rng.randint(-4, 5, rows) * np.spacing(u), 0.0, np.nextafter(1.0, 0.0))


@pytest.mark.parametrize("kw", [dict(top_k=3000), dict(top_p=0.9), dict(top_k=12000), dict(min_p=0.001), dict(temperature=2.0)], ids=str)
def test_numbers_at_borders(hip, kw):
    rows, vocab = 600, 20000
    x = np.random.RandomState(3).normal(0.0, 1.5, (1, vocab)).astype(np.float32)
    x[0, ::3] = -np.inf
    u = borders(x[0], rows, 4, **kw)
    agree(hip, np.broadcast_to(x, (rows, vocab)), u, **{n: np.full(rows, v) for n, v in kw.items()})


@pytest.mark.parametrize("seed,std,steps", [(8, 3.0, 0.0), (4, 0.5, 6.0)])
def test_pieces_without_a_token(hip, seed, std, steps):
    """75 pieces a row, two a lane, of whose first every other one is masked; numbers where one lane's weights end and the next one's begin: within a few
    units in the last place of those sums, where a number less the weights before a lane may come out below 0. (The token that the output holds before
    the call is a masked one.)"""
    vocab, piece, lanes = 75 * 2048 - 300, 2048, 38
    rng = np.random.RandomState(seed)
    x = (rng.normal(0.0, std, vocab) + np.repeat(rng.uniform(-steps, 0.0, 75), piece)[:vocab]).astype(np.float32)
    for lane in range(0, lanes, 2):
        x[2 * lane * piece:(2 * lane + 1) * piece] = -np.inf
    w = np.exp(x.astype(np.float64) - float(x.max()))
    upto = running(w)
    u = []
    for lane in range(2, lanes, 2):
        edge = float(upto[2 * lane * piece - 1] / upto[-1])
        u += [edge + k * np.spacing(edge) for k in range(-16, 17)]
    u = np.array(u)
    t, l = agree(hip, np.broadcast_to(x, (len(u), vocab)), u)
    assert np.all(t >= 2048)


LARGE = [131073, 151936, 262145, 524289, 1048577 + 2048]
SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.8, top_k=40, top_p=0.95), dict(top_k=700, top_p=0.5), dict(temperature=0.0),
            dict(top_p=0.0), dict(min_p=1.0), dict(top_k=30000), dict(temperature=1.3, top_p=0.97, min_p=0.0001)]


@pytest.mark.parametrize("vocab", LARGE)
def test_large_vocabularies(hip, vocab):
    """Broad rows, and rows of which whole pieces are masked, the first and the last among them."""
    n = len(SETTINGS)
    every = {m: np.array([s.get(m, d) for s in SETTINGS]) for m, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    rng = np.random.RandomState(vocab)
    x = rng.normal(0.0, 2.0, (n, vocab)).astype(np.float32)
    x[:, rng.randint(0, vocab, 500)] += np.float32(5.0)
    agree(hip, x, numbers(1, n), **every)
    for first in range(0, vocab, 2048):
        if rng.rand() < 0.4 or first == 0 or first + 2048 >= vocab:
            x[:, first:first + 2048] = -np.inf
    for u in (numbers(2, n), np.zeros(n), np.full(n, np.nextafter(1.0, 0.0))):
        agree(hip, x, u, **every)


@pytest.mark.parametrize("vocab", [151936, 1048577 + 2048])
def test_flat_rows_of_large_vocabularies(hip, vocab):
    """All logits alike: the order is the index, and sums are whole numbers."""
    x = np.zeros((4, vocab), np.float32)
    u = np.array([0.0, 0.25, 0.75, np.nextafter(1.0, 0.0)])
    for kw in (dict(), dict(top_k=100001), dict(top_p=0.75), dict(top_k=vocab // 2, top_p=0.5)):
        k = kw.get("top_k", vocab)
        k = math.ceil(float(np.float32(kw.get("top_p", 1.0))) * k)
        t, l = call(hip, x, u, **{n: np.full(4, v) for n, v in kw.items()})
        assert t.tolist() == [0, math.floor(0.25 * k), math.floor(0.75 * k), k - 1]
        assert np.all(np.abs(l + math.log(k)) <= 2.0 ** -24 * math.log(k) + 2.0 ** -36)


def test_rows_that_cannot_be_sampled_in_large_vocabularies(hip):
    vocab = 200001
    x = np.random.RandomState(7).normal(0.0, 2.0, (4, vocab)).astype(np.float32)
    x[1, vocab - 1], x[2, 140000], x[3] = np.nan, np.inf, -np.inf
    bad = DeviceBuffer.from_host(np.array([0], np.int64))
    for kw in (dict(), dict(top_k=np.full(4, 20), top_p=np.full(4, 0.9))):
        t, l = call(hip, x, numbers(8, 4), bad=bad, **kw)
        assert t[0] >= 0 and t[1:].tolist() == [-1] * 3 and np.all(np.isnan(l[1:])) and bad.to_host()[0] == 1


def test_two_calls_at_once(hip):
    """Calls on two streams, each with its workspace, give what they give alone."""
    rows, vocab = 24, 50257
    rng = np.random.RandomState(11)
    x = [rng.normal(0.0, 2.0, (rows, vocab)).astype(np.float32) for _ in range(2)]
    u = [numbers(s, rows) for s in (21, 22)]
    kw = [dict(top_k=np.full(rows, 40, np.int32), top_p=np.full(rows, 0.9, np.float32)), dict(top_p=np.full(rows, 0.999, np.float32))]
    alone = [call(hip, x[i], u[i], **kw[i]) for i in range(2)]
    desc = hip.sample_desc(rows, vocab)
    streams = [Stream() for _ in range(2)]
    ops = []
    for i in range(2):
        k, p = (None if kw[i].get(n) is None else DeviceBuffer.from_host(kw[i][n]) for n in ("top_k", "top_p"))
        ops.append([DeviceBuffer.from_host(x[i]), k, p, DeviceBuffer.from_host(u[i])])
    outs = [[(DeviceBuffer((rows,), np.int32), DeviceBuffer((rows,))) for _ in range(10)] for _ in range(2)]
    work = [hip.sample_workspace(desc) for _ in range(2)]
    hip.synchronize()
    for n in range(10):
        for i in range(2):
            logits, k, p, number = ops[i]
            hip.sample(desc, logits, None, k, p, None, number, *outs[i][n], workspace=work[i], stream=streams[i].handle)
    for s in streams:
        s.synchronize()
    for i in range(2):
        for tokens, lp in outs[i]:
            assert np.array_equal(tokens.to_host(), alone[i][0]) and np.array_equal(lp.to_host().view(np.uint32), alone[i][1].view(np.uint32))
