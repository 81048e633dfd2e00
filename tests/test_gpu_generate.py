"""Generation on the paged cache: logits of prompts and steps against the dense forward of the same decoder (learned positions)
and against a plain decoder in 64 bits (rotation, fewer K/V heads, 16-bit caches); the choice of tokens against plain penalties."""
import numpy as np
import pytest

from conftest import rel_err
from frankentorch_amd import fused, synth
from frankentorch_amd.device import DeviceBuffer
from frankentorch_amd.generate import PagedDecoder, PagedKVCache
from paged_case import from_storage, rotated, to_storage

pytestmark = pytest.mark.gpu

VOCAB, D, HEADS, FFN, LAYERS, MAX = 503, 128, 4, 256, 2, 96


def weights(seed, kv_heads=HEADS):
    n = lambda tag, *s: synth.normal(seed, tag, s, 0.0, 0.08)
    kv = kv_heads * (D // HEADS)
    layers = [{"ln1_w": 1 + n("a%d" % i, D), "ln1_b": n("b%d" % i, D), "wq": n("c%d" % i, D, D), "bq": n("d%d" % i, D), "wk": n("e%d" % i, kv, D), "bk": n("f%d" % i, kv),
               "wv": n("g%d" % i, kv, D), "bv": n("h%d" % i, kv), "wo": n("i%d" % i, D, D), "bo": n("j%d" % i, D), "ln2_w": 1 + n("k%d" % i, D), "ln2_b": n("l%d" % i, D),
               "w1": n("m%d" % i, FFN, D), "b1": n("n%d" % i, FFN), "w2": n("o%d" % i, D, FFN), "b2": n("p%d" % i, D)} for i in range(LAYERS)]
    return n("wte", VOCAB, D) * 3, n("wpe", MAX, D), layers, 1 + n("lnf", D), n("lnfb", D)


def plain(w, tokens, kv_heads, rotary, interleaved, cache, tables):
    """Logits [len(tokens), vocab] in 64 bits; the first one is the prompt, all others read keys and values rounded to the
    cache's type."""
    wte, wpe, layers, lw, lb = w
    t, hd = len(tokens), D // HEADS
    norm = lambda x, g, b: (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5) * g + b
    x = wte.astype(np.float64)[tokens]
    if not rotary:
        x = x + wpe[:t]
    for p in layers:
        h = norm(x, p["ln1_w"], p["ln1_b"])
        q, k, v = ((h @ p["w" + n].T.astype(np.float64) + p["b" + n]).reshape(t, -1, hd) for n in "qkv")
        if rotary:
            q, k = (rotated(z, np.arange(t), *tables, rotary, interleaved, np.float64) for z in (q, k))
        stored = [from_storage(to_storage(z.astype(np.float32), cache), cache).astype(np.float64) for z in (k, v)] if cache != "f32" else [k, v]
        out = np.zeros((t, HEADS, hd))
        for i in range(t):
            for hh in range(HEADS):
                g = hh // (HEADS // kv_heads)
                kk, vv = stored if i else (k, v)  # the prompt's attention reads its own projection
                s = kk[:i + 1, g] @ q[i, hh] / np.sqrt(hd)
                e = np.exp(s - s.max())
                out[i, hh] = e @ vv[:i + 1, g] / e.sum()
        x = x + out.reshape(t, D) @ p["wo"].T + p["bo"]
        h = norm(x, p["ln2_w"], p["ln2_b"]) @ p["w1"].T + p["b1"]
        h = 0.5 * h * (1 + np.tanh(np.sqrt(2 / np.pi) * (h + 0.044715 * h ** 3)))
        x = x + h @ p["w2"].T + p["b2"]
    return norm(x, lw, lb) @ wte.T.astype(np.float64)


@pytest.mark.parametrize("page", [16, 5])
def test_steps_give_the_logits_of_the_dense_forward(hip, page):
    """Prompts of ragged lengths, then tokens one by one: every row of logits is the dense decoder's at that position."""
    w = weights(61)
    model = PagedDecoder(*w, HEADS, max_seqs=4, num_pages=4 * -(-MAX // page), page_size=page)
    dense = fused.Gpt2Hip(*w, HEADS, 1e-5, gelu_tanh=True)
    seqs = [synth.uniform(61, "s%d" % i, (n,), 0, VOCAB).astype(int).tolist() for i, n in enumerate((40, 7, 1, 64))]
    start = (23, 6, 1, 40)

    def reference(tokens):
        ids, out = DeviceBuffer.from_host(np.array(tokens, np.float64)), DeviceBuffer((len(tokens), VOCAB))
        dense.forward_dev(ids, 1, len(tokens), out, None)
        return out.to_host()

    refs = [reference(s) for s in seqs]
    for i, n in enumerate(start):
        assert rel_err(model.prefill(i, seqs[i][:n]).to_host()[:VOCAB], refs[i][n - 1]) <= 1e-4
    for k in range(24):
        rows = [i for i in (2, 0, 3, 1) if start[i] + k < len(seqs[i])]
        if not rows:
            break
        got = model.step(rows, [seqs[i][start[i] + k] for i in rows]).to_host()[:len(rows) * VOCAB].reshape(-1, VOCAB)
        for row, i in zip(got, rows):
            assert rel_err(row, refs[i][start[i] + k]) <= 1e-4, (k, i)


@pytest.mark.parametrize("kv_heads,rotary,interleaved,cache", [(4, 32, False, "f32"), (2, 16, True, "f32"), (1, 32, False, "bf16"), (4, 0, False, "f16")])
def test_against_a_plain_decoder(hip, kv_heads, rotary, interleaved, cache):
    """A sequence that starts at its first token goes through the cache alone: the plain decoder rounds where the cache does. The
    bar is four times fp32's through two blocks, and a tenth of the storage type's step where activations may round either way."""
    w = weights(62, kv_heads)
    model = PagedDecoder(w[0], None if rotary else w[1], *w[2:], HEADS, 3, 60, 16, MAX, cache, rotary_dim=rotary or None, interleaved=interleaved)
    tokens = synth.uniform(62, "t", (50,), 0, VOCAB).astype(int).tolist()
    ref = plain(w, tokens, kv_heads, rotary, interleaved, cache, hip.rotary_tables(MAX, rotary) if rotary else None)
    bar = {"f32": 1e-4, "f16": 1e-4 + 2.0 ** -11 / 4, "bf16": 1e-4 + 2.0 ** -8 / 4}[cache]
    got = [model.prefill(1, tokens[:1]).to_host()[:VOCAB]] + [model.step([1], [t]).to_host()[:VOCAB] for t in tokens[1:]]
    assert rel_err(np.array(got), ref) <= bar
    if cache == "f32":  # and the same from a prompt
        model.release(1)
        assert rel_err(model.prefill(0, tokens).to_host()[:VOCAB], ref[-1]) <= bar


def test_generate(hip):
    """Greedy tokens with penalties, a bias and a mask are the plain choice on the decoder's own logits; pages come back."""
    w = weights(63)
    model = PagedDecoder(*w, HEADS, 3, 3 * MAX // 16)
    prompts = [[5, 6, 7, 5, 9], [100], list(range(30, 60))]
    bias = synth.normal(63, "bias", (VOCAB,), 0.0, 0.2)
    allowed = lambda r, tokens: None if r == 0 else np.arange(VOCAB) % 3 == len(tokens) % 3
    pages = len(model.kv.free)
    out = model.generate(prompts, 20, repetition=1.3, frequency=0.2, presence=0.1, bias=bias, allowed=allowed)
    assert len(model.kv.free) == pages and [len(o) for o in out] == [20, 20, 20]
    other = PagedDecoder(*w, HEADS, 3, 3 * MAX // 16)
    for r, p in enumerate(prompts):
        tokens = list(p)
        logits = other.prefill(r, p).to_host()[:VOCAB]
        for t in out[r]:
            x = logits.astype(np.float64)
            seen, made = np.unique(tokens), np.bincount(tokens[len(p):], minlength=VOCAB)
            x[seen] = np.where(x[seen] > 0, x[seen] / np.float32(1.3), x[seen] * np.float32(1.3))
            x = x - np.float32(0.2) * made - np.float32(0.1) * (made > 0) + bias
            may = allowed(r, tokens)
            if may is not None:
                assert may[t]
                x = np.where(may, x, -np.inf)
            assert x[t] >= x.max() - 1e-4  # (the batch of another size rounds products otherwise)
            tokens.append(t)
            if len(tokens) < len(p) + 20:
                logits = other.step([r], [t]).to_host()[:VOCAB]
    stop = out[1][7]
    again = model.generate(prompts, 20, repetition=1.3, frequency=0.2, presence=0.1, bias=bias, allowed=allowed, stop=stop)
    for o, a in zip(out, again):
        assert a == (o[:o.index(stop) + 1] if stop in o else o)
    assert model.generate([[1]], 0) == [[]]


def test_pages_and_refusals(hip):
    pool = PagedKVCache(1, 5, 16, 2, 32, 3, 64)
    pool.reserve(0, 33)
    assert np.count_nonzero(pool.rows[0] >= 0) == 3 and len(pool.free) == 2
    with pytest.raises(MemoryError):
        pool.reserve(1, 40)
    assert len(pool.free) == 2 and np.all(pool.rows[1] == -1)
    with pytest.raises(ValueError):
        pool.reserve(1, 65)
    pool.release(0)
    pool.reserve(1, 64)
    assert len(pool.free) == 1 and len(set(pool.rows[1])) == 4
    w = weights(64)
    model = PagedDecoder(*w, HEADS, 2, 12, max_len=20)
    for bad in (lambda: model.prefill(0, []), lambda: model.step([0], [1]), lambda: model.prefill(0, [1] * 40)):
        with pytest.raises(ValueError):
            bad()
    model.prefill(0, [1] * 20)
    for bad in (lambda: model.prefill(0, [1]), lambda: model.step([0], [1]), lambda: model.step([0, 0], [1, 1])):
        with pytest.raises(ValueError):
            bad()
