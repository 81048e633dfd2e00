"""Sampling from rows that few candidates do not decide: nuclei of thousands of tokens, borders inside crowded ranges of logits, many ties,
against the definition in 64 bits."""
import numpy as np
import pytest

from frankentorch_amd import synth
from test_gpu_sample import agree, numbers

pytestmark = pytest.mark.gpu

SETTINGS = [dict(top_p=0.9), dict(top_p=0.5), dict(top_p=0.999), dict(top_k=5000), dict(top_k=20000, top_p=0.9), dict(top_k=9000, top_p=0.3, min_p=0.01),
            dict(min_p=0.002), dict(temperature=6.0, top_p=0.95), dict(temperature=0.3, top_p=0.97), dict(top_k=300, top_p=0.8)]


def run(hip, x, seed):
    rows = len(SETTINGS)
    assert len(x) == rows
    every = {n: np.array([s.get(n, d) for s in SETTINGS]) for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    agree(hip, x, numbers(seed, rows), **every)


@pytest.mark.parametrize("vocab", [7169, 20000, 50257, 131071])
@pytest.mark.parametrize("std", [0.01, 0.5, 2.0])
def test_broad_rows(hip, vocab, std):
    x = synth.normal(vocab, "x", (len(SETTINGS), vocab), 0.0, std)
    for seed in range(2):
        run(hip, x, seed)


@pytest.mark.parametrize("step", [0.5, 0.0625, 2.0 ** -12])
def test_ties(hip, step):
    """Logits on a grid: each border lies among hundreds to thousands of equal ones."""
    x = synth.normal(5, "x", (len(SETTINGS), 50257), 0.0, 1.0)
    run(hip, (np.round(x / step) * step).astype(np.float32), 6)


@pytest.mark.parametrize("crowd", [255, 256, 257, 1023, 1025, 7167, 7168, 7169, 9000])
def test_a_crowd_behind_one(hip, crowd):
    """One token far ahead and `crowd` equal or nearly equal ones, in which all borders lie; the rest is masked."""
    x = np.full((len(SETTINGS), 30011), -np.inf, np.float32)
    at = np.random.RandomState(crowd).permutation(30011)[:crowd + 1]
    x[:, at[0]] = 5.0
    x[:, at[1:]] = 1.0
    x[::2, at[1::2]] += np.float32(2.0 ** -20)
    run(hip, x, crowd)


def test_every_range_of_the_row(hip):
    """Numbers from end to end of a row whose every token is kept: the first, the last, and those around the ends of what wavefronts take."""
    u = np.array([0.0, 1e-12, 0.25, 0.5, 0.75, 0.999999, 1 - 2.0 ** -53, 0.1, 0.9, 1.0 / 3])
    for vocab in (16385, 50257):
        x = synth.uniform(vocab, "x", (len(u), vocab)).astype(np.float32) * np.float32(0.001)
        agree(hip, x, u, top_p=np.full(len(u), 0.99999))
