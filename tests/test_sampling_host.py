"""What sampled generation decides on the host: settings for all prompts or each, what is refused, which numbers a prompt gets. The
device is left out, as in the tests of greedy generation."""
import numpy as np
import pytest

from frankentorch_amd import device, generate
from frankentorch_amd.generate import PagedKVCache
from test_generation_host import VOCAB, HostBuffer, make  # noqa: F401 (a fixture)


@pytest.fixture
def calls(monkeypatch, make):  # noqa: F811
    """The arguments of every device.sample call, as arrays of its rows; the token is the number's place in the vocabulary."""
    seen = []

    def sample(desc, logits, temperature, top_k, top_p, min_p, uniform, tokens, logprobs=None, workspace=None):
        m = desc.rows
        seen.append({n: b.array[:m].copy() for n, b in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p), ("uniform", uniform))})
        tokens.array[:m] = (uniform.array[:m] * VOCAB).astype(np.int32)

    class Desc:
        def __init__(self, rows, vocab):
            self.rows, self.vocab = rows, vocab

    monkeypatch.setattr(device, "sample", sample)
    monkeypatch.setattr(device, "sample_desc", Desc)
    monkeypatch.setattr(device, "sample_workspace", lambda desc: HostBuffer((1,)))
    return seen


def test_settings_reach_their_rows(make, calls):  # noqa: F811
    model = make()
    out = model.generate([[1], [2, 3], [4]], 3, temperature=[0.5, 0.0, 1.5], top_k=7, top_p=[1.0, 0.9, 0.8], min_p=0.1, stop=-1)
    assert len(calls) == 3 + 2  # a prompt each, then steps of all
    assert calls[1]["temperature"].tolist() == [0.0] and calls[4]["temperature"].tolist() == [0.5, 0.0, 1.5]
    assert calls[4]["top_k"].tolist() == [7, 7, 7] and calls[4]["min_p"].tolist() == [np.float32(0.1)] * 3
    assert calls[4]["top_p"].tolist() == np.array([1.0, 0.9, 0.8], np.float32).tolist()
    assert all(len(o) == 3 for o in out)


def test_numbers_do_not_depend_on_the_others(make, calls):  # noqa: F811
    both = make().generate([[1], [2]], 4, temperature=1.0, seed=5)
    one = make().generate([[1]], 4, temperature=1.0, seed=5)
    other = make().generate([[1]], 4, temperature=1.0, seed=6)
    assert both[0] == one[0] != other[0] and both[0] != both[1]


def test_greedy_does_not_sample(make, calls):  # noqa: F811
    assert make().generate([[1], [2]], 3, top_k=5) == [[7] * 3] * 2 and not calls


def test_refusals_take_nothing(make, calls):  # noqa: F811
    model = make()
    pages = len(model.kv.free)
    for kw in (dict(temperature=-1.0), dict(temperature=np.nan), dict(temperature=np.inf), dict(temperature=1.0, top_k=-1), dict(temperature=1.0, top_p=-0.1), dict(temperature=1.0, top_p=np.nan),
               dict(temperature=1.0, min_p=1.5), dict(temperature=1.0, min_p=-0.1), dict(temperature=[1.0, 1.0]), dict(temperature=1.0, top_k=[1, 2, 3, 4])):
        with pytest.raises(ValueError):
            model.generate([[1], [2], [3]], 2, **kw)
    assert not calls and len(model.kv.free) == pages


def test_a_row_that_cannot_be_sampled(make, calls, monkeypatch):  # noqa: F811
    model = make()
    pages = len(model.kv.free)
    monkeypatch.setattr(device, "sample", lambda desc, logits, t, k, p, m, u, tokens, *a, **kw: tokens.array.fill(-1))
    with pytest.raises(ValueError, match="prompt 0"):
        model.generate([[1], [2]], 2, temperature=1.0)
    assert len(model.kv.free) == pages and not model.length.any()


def test_caches_of_eight_bits(monkeypatch):
    monkeypatch.setattr(generate, "DeviceBuffer", HostBuffer)
    for dtype in ("i8", "e4m3"):
        kv = PagedKVCache(2, 5, 16, 3, 32, 4, 64, dtype)
        assert kv.scales.block == 16 and kv.k[1].array.dtype == np.uint8 and kv.v_scales[0].array.shape == (15,)
        assert PagedKVCache(1, 5, 16, 3, 32, 4, 64, dtype, scale_block=4).k_scales[0].array.shape == (60,)
        for block in (0, 3, 32, -16):
            with pytest.raises(ValueError):
                PagedKVCache(1, 5, 16, 3, 32, 4, 64, dtype, scale_block=block)
    assert PagedKVCache(1, 5, 16, 3, 32, 4, 64, "bf16").scales is None
    with pytest.raises(ValueError):
        PagedKVCache(1, 5, 16, 3, 32, 4, 64, "bf16", scale_block=16)
