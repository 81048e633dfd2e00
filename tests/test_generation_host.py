"""What generation decides on the host: which prompts, tokens and sequences it takes, and what it holds after an error. The device
is left out: buffers are host arrays, the forward is a stand-in that gives logits of zeros."""
import numpy as np
import pytest

from frankentorch_amd import device, generate
from frankentorch_amd.generate import PagedDecoder

VOCAB, D, HEADS, FFN = 50, 32, 2, 64


class HostBuffer:
    def __init__(self, shape, dtype=np.float32):
        self.array = np.zeros(shape, dtype)
        self.shape, self.dtype, self.size, self.nbytes, self.ptr = self.array.shape, self.array.dtype, self.array.size, self.array.nbytes, 64

    @classmethod
    def from_host(cls, array):
        buf = cls(np.shape(array), np.asarray(array).dtype)
        buf.array[...] = array
        return buf

    def to_host(self):
        return self.array.copy()

    def view(self, offset):
        return self


def put(buf, array):
    array = np.ascontiguousarray(array, buf.dtype)
    buf.array.reshape(-1)[:array.size] = array.reshape(-1)
    return buf


@pytest.fixture
def make(monkeypatch):
    """make(max_seqs, num_pages, max_len, rotation): a decoder whose forward notes its tokens in `seen`."""
    monkeypatch.setattr(generate, "DeviceBuffer", HostBuffer)
    monkeypatch.setattr(generate, "_put", put)
    monkeypatch.setattr(device, "synchronize", lambda: None)
    monkeypatch.setattr(device, "logits_process", lambda *a, **k: None)
    monkeypatch.setattr(device, "argmax", lambda x, m, vocab, inner, best: best.array.fill(7))

    def make(max_seqs=3, num_pages=12, max_len=20, rotation=False):
        z = lambda *s: np.zeros(s, np.float32)
        layer = dict(ln1_w=z(D), ln1_b=z(D), wq=z(D, D), bq=z(D), wk=z(D, D), bk=z(D), wv=z(D, D), bv=z(D), wo=z(D, D), bo=z(D), ln2_w=z(D), ln2_b=z(D), w1=z(FFN, D),
                     b1=z(FFN), w2=z(D, FFN), b2=z(D))
        model = PagedDecoder(z(VOCAB, D), None if rotation else z(max_len, D), [layer], z(D), z(D), HEADS, max_seqs, num_pages, max_len=max_len)
        model.seen = []

        def forward(ids, seqs, positions, attend, prompt=False):
            model.seen.append((np.asarray(ids).tolist(), list(seqs), np.asarray(positions).tolist()))
            return HostBuffer((max(len(ids), 1), D))

        model._forward, model._gemm = forward, lambda *a, **k: None
        return model

    return make


def state(model):
    return len(model.kv.free), model.length.tolist(), model.kv.rows.tolist()


@pytest.mark.parametrize("rotation", [False, True])
@pytest.mark.parametrize("length", [21, 25, 32, 33, 40])
def test_prompts_longer_than_max_len_are_refused(make, length, rotation):
    """max_len is no multiple of the page: the pages would hold 32 positions, the positions' table has 20."""
    model = make(max_len=20, rotation=rotation)
    before = state(model)
    with pytest.raises(ValueError):
        model.prefill(0, [1] * length)
    assert state(model) == before and not model.seen
    model.prefill(0, [1] * 20)
    assert model.length[0] == 20


@pytest.mark.parametrize("bad", [-1, VOCAB, VOCAB + 1000, -2 ** 40, 2 ** 40, 1.5, float("nan"), float("inf")], ids=str)
def test_tokens_outside_the_vocabulary_are_refused(make, bad):
    model = make()
    before = state(model)
    for prompt in ([bad], [1, 2, bad], [bad, 3]):
        with pytest.raises(ValueError):
            model.prefill(0, prompt)
    assert state(model) == before and not model.seen
    model.prefill(0, [0, VOCAB - 1])
    model.prefill(1, [5.0])
    before = state(model)
    for tokens in ([bad, 1], [1, bad]):
        with pytest.raises(ValueError):
            model.step([0, 1], tokens)
    assert state(model) == before and len(model.seen) == 2
    model.step([0, 1], [VOCAB - 1, 0])
    with pytest.raises(ValueError):
        make().generate([[1], [2, bad]], 3)


@pytest.mark.parametrize("seqs,tokens", [([0, 1], [3]), ([0], [3, 4]), ([0, 1], []), ([0, 1], [[3, 4]]), ([0, -3], [3, 4]), ([-1, 2], [3, 4]), ([0, 3], [3, 4]), ([0, -4], [3, 4])], ids=str)
def test_steps_of_sequences_and_tokens_that_do_not_pair_up(make, seqs, tokens):
    """A token for every sequence; no sequence twice, whichever end of the batch its number counts from; none that is not there."""
    model = make(max_seqs=3)
    for s in range(3):
        model.prefill(s, [s + 1])
    before = state(model)
    with pytest.raises((ValueError, IndexError)):
        model.step(seqs, tokens)
    assert state(model) == before and len(model.seen) == 3


def test_a_sequence_counted_from_the_end_is_the_same_one(make):
    model = make(max_seqs=3)
    model.prefill(-1, [1, 2])
    model.step([-1], [3])
    model.step([2], [4])
    assert model.length.tolist() == [0, 0, 4] and model.seen[1][1] == [2] and model.seen[2][2] == [3]
    with pytest.raises(IndexError):
        model.prefill(3, [1])


def test_generate_gives_back_what_it_took(make):
    """After an error in the middle the pages are free and the next call goes through."""
    model = make(max_seqs=3, num_pages=5, max_len=64)
    empty = state(model)
    with pytest.raises(MemoryError):  # three prompts fit, their growth does not
        model.generate([[1] * 16, [2] * 16, [3] * 32], 30)
    assert state(model) == empty
    with pytest.raises(MemoryError):  # the third prompt does not fit
        model.generate([[1] * 30, [2] * 30, [3] * 33], 2)
    assert state(model) == empty

    def allowed(r, tokens):
        if len(tokens) == 6:
            raise KeyError("a grammar's own error")
        return None

    with pytest.raises(KeyError):
        model.generate([[1] * 3, [2] * 4], 9, allowed=allowed)
    assert state(model) == empty
    with pytest.raises(ValueError):
        model.generate([[1], [2] * 65], 2)
    assert state(model) == empty
    with pytest.raises(ValueError):  # more than max_seqs
        model.generate([[1]] * 4, 2)
    assert state(model) == empty
    assert model.generate([[1] * 16, [2]], 3) == [[7] * 3] * 2 and state(model) == empty


def test_generate_leaves_sequences_that_others_hold(make):
    model = make(max_seqs=3)
    model.prefill(1, [4] * 17)
    held = state(model)
    assert model.generate([[1], [2]], 0) == [[], []] and state(model) == held
    with pytest.raises(ValueError):
        model.generate([[1], [2]], 3)
    assert state(model) == held
    assert model.generate([[1]], 3) == [[7] * 3] and state(model) == held


def test_a_prompt_whose_forward_fails_leaves_nothing(make):
    model = make()
    empty = state(model)

    def forward(*a, **k):
        raise MemoryError("no room for the activations")

    model._forward = forward
    with pytest.raises(MemoryError):
        model.prefill(1, [1] * 18)
    assert state(model) == empty


def test_a_step_that_fails_adds_no_position(make):
    """Neither a pool that runs dry nor an error on the way to the kernels counts a position whose keys were never stored."""
    model = make(max_seqs=2, num_pages=3)
    model.prefill(0, [1] * 16)
    model.prefill(1, [2] * 16)
    with pytest.raises(MemoryError):
        model.step([0, 1], [3, 4])
    assert model.length.tolist() == [16, 16]
    forward = model._forward

    def fails(*a, **k):
        raise RuntimeError("no launch")

    model._forward = fails
    with pytest.raises(RuntimeError):
        model.step([0], [3])
    assert model.length.tolist() == [16, 16]
    model._forward = forward
    model.step([0], [3])
    assert model.length.tolist() == [17, 16] and model.seen[-1] == ([3], [0], [16])


def test_a_mask_that_allows_no_token_is_an_error(make):
    """There is no token to choose: all logits are minus infinity and the argmax would give token 0."""
    model = make()
    empty = state(model)
    for after in (2, 4):
        with pytest.raises(ValueError, match="prompt 1"):
            model.generate([[1, 2], [3, 4]], 5, allowed=lambda r, tokens: np.full(VOCAB, r == 0 or len(tokens) != after))
        assert state(model) == empty
    one = np.zeros(VOCAB, bool)
    one[VOCAB - 1] = True
    assert len(model.generate([[1, 2]], 5, allowed=lambda r, tokens: one)[0]) == 5


def test_columns_of_tokens(make):
    """An array with one token a row is those tokens; more than one a row are not."""
    model = make()
    model.prefill(0, np.array([[4], [5], [6]]))
    model.prefill(1, np.array([7]))
    model.step([0, 1], np.array([[8], [9]], np.int32))
    assert model.length.tolist() == [4, 2, 0] and [s[0] for s in model.seen] == [[4, 5, 6], [7], [8, 9]]
    for wrong in ([[1, 2], [3, 4]], [[1, 2]]):
        with pytest.raises(ValueError):
            model.prefill(2, np.array(wrong))
        with pytest.raises(ValueError):
            model.step([0, 1], np.array(wrong))
    assert model.length.tolist() == [4, 2, 0]
