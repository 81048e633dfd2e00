"""A decoder goes on as if nothing had been asked after calls that it refused or that failed."""
import numpy as np
import pytest

from frankentorch_amd.generate import PagedDecoder
from test_gpu_generate import HEADS, VOCAB, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary", [None, 16])
def test_refused_and_failed_calls_leave_no_trace(hip, rotary):
    w = weights(65)
    w = (w[0], None if rotary else w[1], *w[2:])
    make = lambda: PagedDecoder(*w, HEADS, 3, 5, max_len=40, rotary_dim=rotary)
    model, other = make(), make()
    prompts = [[5, 6, 7], list(range(30, 60))]
    for bad in ([1] * 41, [1] * 48, [1, VOCAB], [-1], [2.5], []):
        with pytest.raises(ValueError):
            model.prefill(0, bad)
    with pytest.raises(MemoryError):
        model.generate([[1] * 30, [2] * 30, [3] * 30], 3)
    with pytest.raises(ValueError):
        model.generate([[1, 2], [3]], 5, allowed=lambda r, tokens: np.full(VOCAB, len(tokens) != 3))
    assert model.generate(prompts, 8, repetition=1.2) == other.generate(prompts, 8, repetition=1.2)
    for m in (model, other):
        m.prefill(1, list(range(40)))
        m.release(1)
        m.prefill(0, prompts[1])
        m.prefill(-1, prompts[0])
    for bad in (([0, 2], [1]), ([0, 2], [1, VOCAB]), ([2, -1], [1, 2]), ([1], [1])):
        with pytest.raises(ValueError):
            model.step(*bad)
    assert np.array_equal(model.step([0, 2], [3, 4]).to_host()[:2 * VOCAB], other.step([0, -1], [3, 4]).to_host()[:2 * VOCAB])
