"""Attention over a paged cache where its result is decided by few keys, or by keys of small weight: each output by itself against 64
bits. Scores are single products of numbers that every storage type holds, so that what is left is the softmax's own error."""
import numpy as np
import pytest

from conftest import TOL_GEMM_F32
from paged_case import Paged, attention, from_storage, to_storage
from test_gpu_paged_sdpa import run

from frankentorch_amd import synth

pytestmark = pytest.mark.gpu

FAR = -1000.0  # exp(FAR) is zero


def scored(seed, lens, scores, d, page, dtype, values, hkv=1):
    """A cache whose first key column is scores[s][position] and the others zero, with V from values[s] [len, d]."""
    p = Paged(seed, lens, hkv, d, page, dtype)
    for s in range(len(lens)):
        p.k[s][:] = 0
        p.k[s][:, :, 0] = from_storage(to_storage(np.asarray(scores[s], np.float32), dtype), dtype)
        p.v[s][:] = from_storage(to_storage(np.asarray(values[s], np.float32), dtype), dtype)
        for x, store in ((p.k, p.stores[0]), (p.v, p.stores[1])):
            store[p.index(s, np.arange(lens[s]))] = x[s].transpose(1, 0, 2)
    return p


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("i,j,n", [(0, 1, 2), (0, 1, 3), (3, 20, 30), (0, 40, 64), (0, 128, 150), (128, 0, 150), (5, 700, 900), (700, 5, 900), (0, 5000, 5100)])
def test_two_weights(hip, dtype, i, j, n):
    """Keys i and j alone have weights, of scores in [-1, 1]: in one tile, in two wavefronts, in two tiles of one wavefront, in two
    shares. In units of 2^-24: a score times log2 e is below 1.45 and rounded by 1 for each key, log2 e itself is off by 0.65 on their
    difference, which is rounded by 2: the exponent is off by 4.65, the weight by 3.25, and exp2 adds 2; the sum, the two
    products of a join on both sides and the division add 5 to the relative error of an output."""
    seqs = 4 if n > 1000 else 150
    a = np.round(synth.uniform(41, "a", (seqs, 2), -1.0, 1.0) * 64) / 64
    scores, values = np.full((seqs, n), FAR), np.full((seqs, n, 64), 5.0)
    scores[:, i], scores[:, j] = a[:, 0], a[:, 1]
    values[:, i], values[:, j] = np.arange(64) % 3 == 0, np.arange(64) % 3 == 1
    p = scored(41, [n] * seqs, scores, 64, 16, dtype, values)
    q = np.zeros((seqs, 1, 1, 64), np.float32)
    q[..., 0] = 1
    got, ref = run(hip, p, q, 1.0), attention(q, p.k, p.v, 1.0, p.lens)
    assert np.all(got[ref == 0] == 0)
    assert np.max(np.abs(got - ref)[ref != 0] / ref[ref != 0]) <= 10.25 * 2.0 ** -24


@pytest.mark.parametrize("dtype,page,d", [("f32", 16, 64), ("f16", 16, 64), ("bf16", 16, 64), ("f16", 5, 64), ("f16", 16, 128), ("f16", 16, 256), ("f16", 16, 40), ("f16", 16, 7)])
@pytest.mark.parametrize("n", [2, 33, 512, 1500])
def test_values_under_small_weights(hip, dtype, page, d, n):
    """One key has nearly all the weight and zeros in V: the outputs are those of the keys 5 to 80 nats below it, relative to themselves as
    exact as any."""
    depths = [5, 12, 16, 20, 25, 28, 40, 60, 80]
    for heavy in {0, n // 2, n - 1}:
        scores = -np.array(depths, np.float64)[:, None] + synth.uniform(42, "s", (len(depths), n), -1.0, 1.0)
        scores[:, heavy] = 0
        values = synth.normal(42, "v", (len(depths), n, d))
        values[:, heavy] = 0
        p = scored(42, [n] * len(depths), scores, d, page, dtype, values)
        q = np.zeros((len(depths), 2, 3, d), np.float32)
        q[..., 0] = np.array([1, 0.5, 0.75], np.float32)
        if heavy == n - 1:
            q[:, 0] = 0  # the first of the two tokens does not see the key
        got, ref = run(hip, p, q, 1.0), attention(q, p.k, p.v, 1.0, p.lens)
        for s, depth in enumerate(depths):
            for h in range(3):
                size = np.abs(ref[s, 1, h]).max()
                assert np.abs(got - ref)[s, 1, h].max() <= TOL_GEMM_F32 * size, (heavy, depth, h)


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("f16", 64), ("bf16", 64), ("f16", 128), ("f16", 256)])
@pytest.mark.parametrize("n", [64, 700])
@pytest.mark.parametrize("order", ["mixed", "rising", "falling"])
def test_weights_of_every_size(hip, dtype, d, n, order):
    """Scores from 0 down to -80; column c of V is zero under all keys above -80 c / d and positive under the others: it is decided by weights of
    one size, which differs from column to column."""
    scores = -80.0 * synth.uniform(43, "s", (3, n))
    if order != "mixed":
        scores = np.sort(scores, 1) if order == "rising" else -np.sort(-scores, 1)
    scores = from_storage(to_storage(scores.astype(np.float32), dtype), dtype).astype(np.float64)
    values = 0.5 + synth.uniform(43, "v", (3, n, d))
    values[scores[:, :, None] > -80.0 * np.arange(d) / d] = 0
    p = scored(43, [n] * 3, scores, d, 16, dtype, values)
    q = np.zeros((3, 1, 2, d), np.float32)
    q[..., 0] = 1
    got, ref = run(hip, p, q, 1.0), attention(q, p.k, p.v, 1.0, p.lens)
    assert np.all(got[ref == 0] == 0)
    assert np.max(np.abs(got - ref)[ref != 0] / ref[ref != 0]) <= TOL_GEMM_F32
