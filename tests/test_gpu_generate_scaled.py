"""Generation on a cache of 8-bit numbers against a plain decoder that rounds where the cache does, and sampled tokens against the
plain choice on the decoder's own logits."""
import numpy as np
import pytest

from conftest import rel_err
from frankentorch_amd import synth
from frankentorch_amd.generate import PagedDecoder
from paged_case import rotated
from scaled_case import Scaled
from test_gpu_generate import D, HEADS, LAYERS, MAX, VOCAB, weights
from test_gpu_sample import kept

pytestmark = pytest.mark.gpu


def plain(w, tokens, kv_heads, rotary, interleaved, dtype, block, tables):
    """Logits [len(tokens), vocab] in 64 bits of tokens appended one by one; the first reads its own projection, all others the cache."""
    wte, wpe, layers, lw, lb = w
    hd = D // HEADS
    norm = lambda x, g, b: (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5) * g + b
    caches = [Scaled(i, 1, kv_heads, hd, 16, block, dtype, -(-len(tokens) // 16)) for i in range(LAYERS)]
    logits = []
    for pos, token in enumerate(tokens):
        x = wte[token].astype(np.float64) + (0 if rotary else wpe[pos])
        for p, cache in zip(layers, caches):
            h = norm(x, p["ln1_w"], p["ln1_b"])
            q, k, v = ((p["w" + n].astype(np.float64) @ h + p["b" + n]).reshape(1, -1, hd) for n in "qkv")
            if rotary:
                q, k = (rotated(z, np.array([pos]), *tables, rotary, interleaved, np.float64) for z in (q, k))
            cache.append(0, 0, pos, k.astype(np.float32))
            cache.append(1, 0, pos, v.astype(np.float32))
            kk, vv = (k.transpose(1, 0, 2), v.transpose(1, 0, 2)) if pos == 0 else (cache.rows(0, 0, pos + 1), cache.rows(1, 0, pos + 1))
            out = np.zeros((HEADS, hd))
            for hh in range(HEADS):
                g = hh // (HEADS // kv_heads)
                s = kk[g] @ q[0, hh] / np.sqrt(hd)
                e = np.exp(s - s.max())
                out[hh] = e @ vv[g] / e.sum()
            x = x + p["wo"] @ out.reshape(D) + p["bo"]
            h = p["w1"] @ norm(x, p["ln2_w"], p["ln2_b"]) + p["b1"]
            h = 0.5 * h * (1 + np.tanh(np.sqrt(2 / np.pi) * (h + 0.044715 * h ** 3)))
            x = x + p["w2"] @ h + p["b2"]
        logits.append(wte.astype(np.float64) @ norm(x, lw, lb))
    return np.array(logits)


@pytest.mark.parametrize("kv_heads,rotary,interleaved,dtype,block", [(4, 32, False, "e4m3", 16), (2, 16, True, "i8", 16), (1, 32, False, "i8", 1), (4, 0, False, "e4m3", 4)])
def test_against_a_plain_decoder(hip, kv_heads, rotary, interleaved, dtype, block):
    """The bar is that of fp32 through two blocks, and a quarter of the type's step at a block's largest element where activations may
    round either way."""
    w = weights(72, kv_heads)
    model = PagedDecoder(w[0], None if rotary else w[1], *w[2:], HEADS, 3, 60, 16, MAX, dtype, rotary_dim=rotary or None, interleaved=interleaved, scale_block=block)
    tokens = synth.uniform(72, "t", (50,), 0, VOCAB).astype(int).tolist()
    ref = plain(w, tokens, kv_heads, rotary, interleaved, dtype, block, hip.rotary_tables(MAX, rotary) if rotary else None)
    bar = 1e-4 + (2.0 ** -3 if dtype == "e4m3" else 1 / 64) / 4
    got = [model.prefill(1, tokens[:1]).to_host()[:VOCAB]] + [model.step([1], [t]).to_host()[:VOCAB] for t in tokens[1:]]
    assert rel_err(np.array(got), ref) <= bar
    assert np.median(np.max(np.abs(np.array(got) - ref), 1) / np.max(np.abs(ref))) <= 1e-4 + bar / 16  # most tokens round alike


@pytest.mark.parametrize("cache", ["e4m3", "i8", "f32"])
def test_sampled_generation(hip, cache):
    """Each token is where its number falls among the kept ones of the decoder's own logits; runs repeat; pages come back."""
    w = weights(73)
    prompts = [[5, 6, 7, 5, 9], [100], list(range(30, 60))]
    how = dict(temperature=[0.9, 1.4, 0.0], top_k=[0, 40, 3], top_p=[0.95, 1.0, 0.5], min_p=[0.0, 0.02, 0.0])
    model = PagedDecoder(*w, HEADS, 3, 3 * MAX // 16, cache=cache)
    pages = len(model.kv.free)
    out = model.generate(prompts, 20, repetition=1.2, seed=11, **how)
    assert len(model.kv.free) == pages and [len(o) for o in out] == [20] * 3
    assert model.generate(prompts, 20, repetition=1.2, seed=11, **how) == out
    assert model.generate(prompts, 20, repetition=1.2, seed=12, **how)[:2] != out[:2]
    other = PagedDecoder(*w, HEADS, 3, 3 * MAX // 16, cache=cache)
    for r, p in enumerate(prompts):
        rng, tokens = np.random.default_rng([11, r]), list(p)
        logits = other.prefill(r, p).to_host()[:VOCAB]
        for t in out[r]:
            x = logits.copy()
            seen = np.unique(tokens)
            x[seen] = np.where(x[seen] > 0, x[seen] / np.float32(1.2), x[seen] * np.float32(1.2))
            v, weight = kept(x, **{n: a[r] for n, a in how.items()})
            u, i = rng.random(), int(np.searchsorted(v, t))
            if how["temperature"][r] == 0:
                assert x[t] >= x.max() - 1e-4
            else:  # (the batch of another size rounds products otherwise: the borders are within 1e-3 of the kept weight)
                total = float(weight.sum())
                assert i < len(v) and v[i] == t or np.min(np.abs(x - x[t])[v]) < 1e-3
                if i < len(v) and v[i] == t:
                    assert weight[:i].sum() / total - 1e-3 <= u <= weight[:i + 1].sum() / total + 1e-3
            tokens.append(t)
            if len(tokens) < len(p) + 20:
                logits = other.step([r], [t]).to_host()[:VOCAB]


def test_eight_bits_do_not_change_much(hip):
    """The logits of a long prompt and its steps on 8-bit caches are those of the fp32 cache but for the rounding of keys and values."""
    w = weights(74)
    tokens = synth.uniform(74, "t", (MAX,), 0, VOCAB).astype(int).tolist()
    got = {}
    for cache in ("f32", "i8", "e4m3"):
        model = PagedDecoder(w[0], None, *w[2:], HEADS, 1, MAX // 16, max_len=MAX, cache=cache, rotary_dim=32)
        model.prefill(0, tokens[:60])
        got[cache] = np.array([model.step([0], [t]).to_host()[:VOCAB] for t in tokens[60:]])
    size = np.sqrt(np.mean(got["f32"] ** 2))
    # an element of K or V is off by up to a quarter of 2^-6 of its block's largest (i8: the scale may be twice what is needed), by 2^-4 of itself (e4m3)
    assert np.sqrt(np.mean((got["i8"] - got["f32"]) ** 2)) <= 2.0 ** -6 * size
    assert np.sqrt(np.mean((got["e4m3"] - got["f32"]) ** 2)) <= 2.0 ** -4 * size
