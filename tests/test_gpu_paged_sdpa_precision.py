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
