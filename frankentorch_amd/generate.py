"""Token-by-token generation on a paged K/V cache: the operators of the device tier put together the way a server runs them.

`PagedKVCache` hands out pages of one pool to sequences; `PagedDecoder` is the GPT-2-shaped decoder of `fused.Gpt2Hip` (pre-LN
blocks, tied head) that keeps keys and values there, so that a new token costs one pass over the weights and one over the
cache instead of a forward over all positions. Prompts run through the dense causal attention and are appended on the way;
after that every step appends one token per sequence, attends over the pages, and readies the logits (penalties, bias, a mask of
allowed tokens) for the argmax. Positions are a learned table (`wpe`) or, without one, a rotation of queries and keys. K/V heads
may be fewer than query heads (rows of `wk`, `wv`).

    python -m frankentorch_amd.generate        # a GPT-2-small-shaped decoder with random weights, a few sequences
"""
from __future__ import annotations

import ctypes as C
from typing import Callable, Optional, Sequence

import numpy as np

from . import _lib, device
from .core import check
from .device import DeviceBuffer


def _put(buf: DeviceBuffer, array) -> DeviceBuffer:
    """Copies a host array to the front of a buffer of its type."""
    array = np.ascontiguousarray(array, buf.dtype)
    if array.size > buf.size:
        raise ValueError("%d elements do not fit %d" % (array.size, buf.size))
    if array.size:
        check(_lib.load().fth_memcpy_h2d(buf.ptr, array.ctypes.data, array.nbytes))
    return buf


class PagedKVCache:
    """Pages of one pool for up to `max_seqs` sequences of up to `max_len` positions, in every layer alike. `cache` is the
    descriptor, `table` the block table on the device (kept in line with `rows` by `sync`)."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int, max_len: int, dtype: str = "f32"):
        width = -(-max_len // page_size)
        self.cache = device.paged_cache(num_pages, page_size, kv_heads, head_dim, max_seqs, width, dtype)
        store = np.float32 if dtype == "f32" else np.uint16
        self.k, self.v = ([DeviceBuffer((num_pages * kv_heads * page_size * head_dim,), store) for _ in range(layers)] for _ in range(2))
        self.rows = np.full((max_seqs, width), -1, np.int32)
        self.table = DeviceBuffer((max_seqs, width), np.int32)
        self.free = list(range(num_pages))[::-1]
        self._dirty = True

    def reserve(self, seq: int, length: int) -> None:
        """Pages for the first `length` positions of a sequence; raises MemoryError, with nothing taken, when the pool has too few."""
        want = -(-length // self.cache.page_size)
        if want > self.rows.shape[1]:
            raise ValueError("sequence %d: %d positions are more than the table holds" % (seq, length))
        have = int(np.count_nonzero(self.rows[seq] >= 0))
        if want - have > len(self.free):
            raise MemoryError("the page pool is empty: %d more needed, %d free" % (want - have, len(self.free)))
        for i in range(have, want):
            self.rows[seq, i] = self.free.pop()
            self._dirty = True

    def release(self, seq: int) -> None:
        """Gives a sequence's pages back (calls that use them are done, or on the stream that later users run on)."""
        self.free.extend(int(p) for p in self.rows[seq][self.rows[seq] >= 0][::-1])
        self.rows[seq] = -1
        self._dirty = True

    def sync(self) -> DeviceBuffer:
        if self._dirty:
            _put(self.table, self.rows)
            self._dirty = False
        return self.table


class PagedDecoder:
    def __init__(self, wte, wpe, layers: Sequence[dict], lnf_w, lnf_b, n_heads: int, max_seqs: int, num_pages: int, page_size: int = 16, max_len: Optional[int] = None,
                 cache: str = "f32", ln_eps: float = 1e-5, gelu_tanh: bool = True, rotary_dim: Optional[int] = None, interleaved: bool = False, rotary_base: float = 10000.0):
        """The weights of `fused.Gpt2Hip`; wpe None: positions by rotation of the first `rotary_dim` elements of a head (default: all)."""
        up = lambda a: DeviceBuffer.from_host(np.ascontiguousarray(a, np.float32))
        self.vocab, self.d = np.shape(wte)
        self.heads, self.hd, self.eps = n_heads, self.d // n_heads, ln_eps
        self.kv_heads = np.shape(layers[0]["wk"])[0] // self.hd
        self.qkv = (n_heads + 2 * self.kv_heads) * self.hd
        self.ffn = np.shape(layers[0]["w1"])[0]
        self.max_len = max_len if max_len is not None else (np.shape(wpe)[0] if wpe is not None else 2048)
        if wpe is not None and self.max_len > np.shape(wpe)[0]:
            raise ValueError("the position table has %d rows, fewer than max_len" % np.shape(wpe)[0])
        self.wte, self.wpe = up(wte), None if wpe is None else up(wpe)
        self.max_pos = 0 if wpe is None else np.shape(wpe)[0]
        self.rotary = 0 if wpe is not None else self.hd if rotary_dim is None else rotary_dim
        self.interleaved = interleaved
        self.cos, self.sin = (up(t) for t in device.rotary_tables(self.max_len, self.rotary, rotary_base)) if self.rotary else (None, None)
        self.lnf = up(lnf_w), up(lnf_b)
        self.layers = []
        for lw in layers:
            packed = {n: up(lw[n]) for n in ("ln1_w", "ln1_b", "wo", "bo", "ln2_w", "ln2_b", "w1", "b1", "w2", "b2")}
            packed["wqkv"] = up(np.concatenate([lw["wq"], lw["wk"], lw["wv"]]))
            packed["bqkv"] = up(np.concatenate([lw["bq"], lw["bk"], lw["bv"]]))
            self.layers.append(packed)
        self.kv = PagedKVCache(len(layers), num_pages, page_size, self.kv_heads, self.hd, max_seqs, self.max_len, cache)
        self.act = device.EPI_GELU_TANH if gelu_tanh else device.EPI_GELU
        self.length = np.zeros(max_seqs, np.int32)  # positions of each sequence that are in the cache
        self._room = {}

    def _buffer(self, name: str, shape, dtype=np.float32) -> DeviceBuffer:
        """A buffer kept from call to call, grown where a call needs more."""
        n = int(np.prod(shape, dtype=np.int64))
        buf = self._room.get(name)
        if buf is None or buf.size < n:
            if buf is not None:
                device.synchronize()  # queued work may still read the old one
            buf = self._room[name] = DeviceBuffer((max(n, 1),), dtype)
        return buf

    def _gemm(self, a, w, out, m, n, k, bias=None, residual=None, act=0):
        epilogue = (device.EPI_BIAS if bias is not None else 0) | act | (device.EPI_RESIDUAL if residual is not None else 0)
        device.gemm(device.gemm_desc(m, n, k, trans_b=True, epilogue=epilogue), a, w, out, bias, residual)

    def _forward(self, ids, seqs, positions, attend: Callable, prompt: bool = False) -> DeviceBuffer:
        """The final hidden states [tokens, d] of tokens at (sequence, position); `attend(layer, qkv, out)` is the attention."""
        t, d, b = len(ids), self.d, self._buffer
        ids64 = _put(b("ids", (t,), np.float64), ids)
        seq_ids, pos = _put(b("seqs", (t,), np.int32), seqs), _put(b("pos", (t,), np.int32), positions)
        x, h, ctx = b("x", (t, d)), b("h", (t, d)), b("ctx", (t, d))
        qkv, up = b("qkv", (t, self.qkv)), b("up", (t, self.ffn))
        table = self.kv.sync()
        device.index_select(self.wte, 1, self.vocab, d, ids64, t, x)
        if self.wpe is not None:
            device.index_select(self.wpe, 1, self.max_pos, d, _put(b("pos64", (t,), np.float64), positions), t, h)
            device.add(x, h, x, t * d)
        turn = append = device.paged_append_desc(self.kv.cache, t, self.heads if self.rotary else 0, self.rotary, self.max_len, self.interleaved, row_stride=self.qkv)
        append.out_row_stride = self.qkv  # queries are rotated in place
        if prompt and self.rotary:  # the dense attention wants the keys rotated as well: they stand beside the queries
            turn = device.paged_append_desc(self.kv.cache, t, self.heads + self.kv_heads, self.rotary, self.max_len, self.interleaved, row_stride=self.qkv)
            turn.out_row_stride = self.qkv
            append = device.paged_append_desc(self.kv.cache, t, row_stride=self.qkv)
        k_at, v_at = self.heads * self.hd, (self.heads + self.kv_heads) * self.hd
        for i, lw in enumerate(self.layers):
            device.layer_norm(x, lw["ln1_w"], lw["ln1_b"], h, t, d, self.eps)
            self._gemm(h, lw["wqkv"], qkv, t, self.qkv, d, lw["bqkv"])
            q = qkv.view(0) if append.q_heads else None
            if turn is not append:
                device.paged_append(self.kv.cache, turn, qkv.view(0), None, None, self.cos, self.sin, None, None, pos, qkv.view(0), None, None)
            device.paged_append(self.kv.cache, append, q, qkv.view(k_at), qkv.view(v_at), self.cos, self.sin, table, seq_ids, pos, q, self.kv.k[i], self.kv.v[i])
            attend(i, qkv, ctx)
            self._gemm(ctx, lw["wo"], x, t, d, d, lw["bo"], x)
            device.layer_norm(x, lw["ln2_w"], lw["ln2_b"], h, t, d, self.eps)
            self._gemm(h, lw["w1"], up, t, self.ffn, d, lw["b1"], act=self.act)
            self._gemm(up, lw["w2"], x, t, d, self.ffn, lw["b2"], x)
        device.layer_norm(x, *self.lnf, h, t, d, self.eps)
        return h

    def _tokens(self, tokens: Sequence[int], n: int) -> np.ndarray:
        """The ids of n tokens, each of which has a row in the embedding."""
        ids = np.asarray(tokens, np.float64)
        if len(ids) != n or ids.size != n:
            raise ValueError("%d tokens are asked for, not an array of %s" % (n, ids.shape))
        ids = ids.reshape(-1)
        with np.errstate(invalid="ignore"):
            wrong = ~((ids >= 0) & (ids < self.vocab) & (ids == np.floor(ids)))
        if wrong.any():
            raise ValueError("token %s is outside the vocabulary of %d" % (ids[wrong][0], self.vocab))
        return ids

    def prefill(self, seq: int, prompt: Sequence[int]) -> DeviceBuffer:
        """A whole prompt into the cache of an empty sequence; the logits [1, vocab] after its last token (a buffer of this object's)."""
        n, seq = len(prompt), range(len(self.length))[seq]  # (the kernels count from the front alone)
        if n == 0 or self.length[seq]:
            raise ValueError("a prompt has at least one token and starts an empty sequence")
        if n > self.max_len:  # (whole pages may hold more positions than the tables have)
            raise ValueError("a prompt of %d tokens is longer than max_len, %d" % (n, self.max_len))
        ids = self._tokens(prompt, n)
        self.kv.reserve(seq, n)
        desc = device.sdpa_desc_gqa(1, self.heads, self.kv_heads, n, n, self.hd, self.hd, True)
        for name, pitch in (("q", self.qkv), ("k", self.qkv), ("v", self.qkv), ("o", self.d)):
            setattr(desc, name + "_batch_stride", n * pitch)
            setattr(desc, name + "_head_stride", self.hd)
            setattr(desc, name + "_row_stride", pitch)
        k_at, v_at = self.heads * self.hd, (self.heads + self.kv_heads) * self.hd

        def attend(layer, qkv, out):
            device.sdpa_forward(desc, device.default_scale(self.hd), qkv.view(0), qkv.view(k_at), qkv.view(v_at), out)

        try:
            hidden = self._forward(ids, [seq] * n, np.arange(n), attend, prompt=True)
            logits = self._buffer("prompt_logits", (1, self.vocab))
            self._gemm(hidden.view((n - 1) * self.d), self.wte, logits, 1, self.vocab, self.d)
        except BaseException:
            self.kv.release(seq)
            raise
        self.length[seq] = n
        return logits

    def step(self, seqs: Sequence[int], tokens: Sequence[int]) -> DeviceBuffer:
        """One more token of each of `seqs`; the logits [len(seqs), vocab] after them, in that order (a buffer of this object's)."""
        n, where = len(seqs), [range(len(self.length))[s] for s in seqs]
        if len(set(where)) != n or any(self.length[s] == 0 for s in where):
            raise ValueError("a step takes different sequences, each after its prompt")
        if any(self.length[s] >= self.max_len for s in where):
            raise ValueError("a sequence is at max_len")
        ids = self._tokens(tokens, n)
        for s in where:
            self.kv.reserve(s, int(self.length[s]) + 1)
        positions = self.length[where]
        # the rows of the batch are its sequences: their rows of the block table, their lengths
        cache = _lib.PagedCache.from_buffer_copy(self.kv.cache)
        cache.num_seqs = n
        table = _put(self._buffer("rows", (n, cache.max_pages), np.int32), self.kv.rows[where])
        lens = _put(self._buffer("lens", (n,), np.int32), positions + 1)
        longest = -(-(int(positions.max()) + 1) // 128) * 128
        desc = device.paged_sdpa_desc(cache, self.heads, 1, min(longest, cache.max_pages * cache.page_size))
        desc.q_seq_stride = desc.q_row_stride = self.qkv
        need = _lib.load().fth_dev_paged_sdpa_workspace_bytes(C.byref(cache), C.byref(desc))
        work = self._buffer("attention", (need // 4 + 4,))

        def attend(layer, qkv, out):
            device.paged_sdpa(cache, desc, device.default_scale(self.hd), qkv, self.kv.k[layer], self.kv.v[layer], table, lens, out, workspace=work)

        hidden = self._forward(ids, where, positions, attend)
        logits = self._buffer("logits", (n, self.vocab))
        self._gemm(hidden, self.wte, logits, n, self.vocab, self.d)
        self.length[where] += 1
        return logits

    def release(self, seq: int) -> None:
        self.kv.release(seq)
        self.length[seq] = 0

    def generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0, bias=None,
                 allowed: Optional[Callable] = None, stop: Optional[int] = None):
        """Greedy continuations of the prompts, one list a prompt. repetition, frequency and presence are as in
        device.logits_process; bias [vocab] or None; allowed(prompt number, tokens so far) gives the tokens that may follow (a
        bool array over the vocabulary) or None for all; a sequence ends with the token `stop`, after `new_tokens`, or at max_len.
        Uses the sequences 0 .. len(prompts) - 1, which have to be empty, and gives them back, after an error too."""
        n = len(prompts)
        if new_tokens > 0 and n > len(self.length):
            raise ValueError("%d prompts are more than max_seqs, %d" % (n, len(self.length)))
        tokens = [list(p) for p in prompts]
        done = [[] for _ in prompts]
        width = max(len(p) for p in prompts) + new_tokens
        fill = lambda value: DeviceBuffer.from_host(np.full(n, value, np.float32))
        penalties = [fill(repetition), fill(frequency), fill(presence)]
        dev_bias = None if bias is None else DeviceBuffer.from_host(np.asarray(bias, np.float32))
        history, counts, given = DeviceBuffer((n, width), np.int32), DeviceBuffer((n,), np.int32), DeviceBuffer((n,), np.int32)
        words = (self.vocab + 31) // 32
        mask, ready, best = DeviceBuffer((n, words), np.uint32), DeviceBuffer((n, self.vocab)), DeviceBuffer((n,))

        def choose(rows, logits):
            """The next token of the sequences `rows` from their logits."""
            m = len(rows)
            desc = device.logits_desc(m, self.vocab, width, shared_bias=True)
            past = np.zeros((m, width), np.int32)
            bits = np.full((m, words * 32), 1, np.uint8)
            for i, r in enumerate(rows):
                past[i, :len(tokens[r])] = tokens[r]
                may = None if allowed is None else allowed(r, tokens[r])
                if may is not None:
                    bits[i, :self.vocab] = np.asarray(may, bool)
                    if not bits[i, :self.vocab].any():
                        raise ValueError("no token may follow prompt %d and the %d tokens after it" % (r, len(done[r])))
            _put(history, past)
            _put(counts, [len(tokens[r]) for r in rows])
            _put(given, [len(prompts[r]) for r in rows])
            if allowed is not None:
                _put(mask, np.packbits(bits, axis=1, bitorder="little").view(np.uint32))
            device.logits_process(desc, logits, history, counts, given, *penalties, dev_bias, mask if allowed is not None else None, ready)
            device.argmax(ready, m, self.vocab, 1, best)
            return best.to_host()[:m].astype(np.int64)

        def note(rows, chosen):
            for r, t in zip(rows, chosen):
                tokens[r].append(int(t))
                done[r].append(int(t))

        started = []
        try:
            for r, p in enumerate(prompts if new_tokens > 0 else []):
                logits = self.prefill(r, p)
                started.append(r)
                note([r], choose([r], logits))
            for _ in range(new_tokens - 1):
                rows = [r for r in range(n) if done[r][-1] != stop and self.length[r] < self.max_len]
                if not rows:
                    break
                note(rows, choose(rows, self.step(rows, [tokens[r][-1] for r in rows])))
        finally:
            for r in started:
                self.release(r)
        return done


def main() -> None:
    import time

    rng = np.random.RandomState(0)
    d, heads, layers, vocab, max_pos, ffn = 768, 12, 12, 50257, 1024, 3072
    w = lambda *s: (rng.standard_normal(s) * 0.02).astype(np.float32)
    one, zero = np.ones(d, np.float32), np.zeros(d, np.float32)
    blocks = [dict(ln1_w=one, ln1_b=zero, wq=w(d, d), bq=zero, wk=w(d, d), bk=zero, wv=w(d, d), bv=zero, wo=w(d, d), bo=zero, ln2_w=one, ln2_b=zero,
                   w1=w(ffn, d), b1=np.zeros(ffn, np.float32), w2=w(d, ffn), b2=zero) for _ in range(layers)]
    batch, new = 8, 64
    model = PagedDecoder(w(vocab, d), w(max_pos, d), blocks, one, zero, heads, batch, batch * max_pos // 16, cache="bf16")
    prompts = [rng.randint(0, vocab, 40 + 60 * i).tolist() for i in range(batch)]
    model.generate(prompts, 4)
    start = time.perf_counter()
    out = model.generate(prompts, new, repetition=1.1, frequency=0.1)
    took = time.perf_counter() - start
    print("%d sequences, %d new tokens each: %.2f ms a step (prompts included), first tokens of each: %s" % (batch, new, 1e3 * took / new, [o[:4] for o in out]))


if __name__ == "__main__":
    main()
