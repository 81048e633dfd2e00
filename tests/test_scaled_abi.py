"""Refusals of the operators on caches of 8-bit numbers and of sampling: they come before any device is asked for, so they need none;
what is accepted gives Unavailable without a device. No pointer here is ever followed."""
import ctypes as C

import pytest

from frankentorch_amd import _lib, device
from test_generation_abi import CACHES, INVALID, OK, OVERFLOW, P


def cache(stored="e4m3", **kw):
    c = device.paged_cache(10, 16, 2, 64, 3, 4, stored)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def scales(c=None, block=8, **kw):
    s = device.paged_scales(c or cache(), block)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def append(c, sc, tokens=0, none=(), **kw):
    d = device.paged_append_desc(c, tokens, 4, 64, 100) if c is not None else _lib.PagedAppendDesc()
    for k, v in kw.items():
        setattr(d, k, v)
    args = {n: P for n in ("q", "k", "v", "cos", "sin", "table", "seq", "pos", "out", "kc", "vc", "ks", "vs")}
    args.update({n: None for n in none if n in args})
    args["q"] = 8192 if args["q"] else None
    return _lib.load().fth_dev_paged_append_scaled_f32(None if c is None else C.byref(c), None if sc is None else C.byref(sc), None if "desc" in none else C.byref(d),
                                                       *args.values(), None, None)


def attend(c, sc, seqs=None, none=(), **kw):
    d = device.paged_sdpa_desc(c, 4, 1) if c is not None else _lib.PagedSdpaDesc()
    for k, v in kw.items():
        setattr(d, k, v)
    if seqs is not None:
        c.num_seqs = seqs
    args = {n: P for n in ("q", "k", "v", "ks", "vs", "table", "lens", "out")}
    args.update({n: None for n in none if n in args})
    ref = lambda x: None if x is None else C.byref(x)
    rc = _lib.load().fth_dev_paged_sdpa_scaled_f32(ref(c), ref(sc), None if "desc" in none else C.byref(d), 1.0, *args.values(), None, None, 0, None)
    if rc and rc != 100 and not none:
        assert _lib.load().fth_dev_paged_sdpa_scaled_workspace_bytes(ref(c), ref(sc), C.byref(d)) == 0
    return rc


@pytest.mark.parametrize("kw,code", [x for x in CACHES if "dtype" not in x[0]] + [(dict(dtype=t), INVALID) for t in (-1, 0, 1, 2, 3, 4, 15, 18)], ids=str)
def test_caches_that_cannot_be(kw, code):
    c = cache(**kw)
    sc = scales() if c.page_size != 16 else scales(block=8)
    assert append(c, sc) == code and attend(c, sc) == code
    assert _lib.last_error().message


def test_eight_bits_and_the_other_calls():
    """The calls without scales take no cache of 8 bits, and the other way round."""
    for dtype in ("i8", "e4m3"):
        c = cache(dtype)
        assert append(c, scales()) in OK and attend(c, scales(), 0) in OK
        d = device.paged_append_desc(c, 0)
        assert _lib.load().fth_dev_paged_append_f32(C.byref(c), C.byref(d), *[None] * 13) == INVALID
        d = device.paged_sdpa_desc(c, 4, 1)
        assert _lib.load().fth_dev_paged_sdpa_f32(C.byref(c), C.byref(d), 1.0, *[None] * 8, 0, None) == INVALID
        assert _lib.load().fth_dev_paged_sdpa_workspace_bytes(C.byref(c), C.byref(d)) == 0


@pytest.mark.parametrize("kw,code", [(dict(block=0), INVALID), (dict(block=-8), INVALID), (dict(block=3), INVALID), (dict(block=17), INVALID), (dict(block=32), INVALID),
                                     (dict(page_stride=0), INVALID), (dict(head_stride=0), INVALID), (dict(head_stride=-1), INVALID), (dict(page_stride=1 << 60), OVERFLOW),
                                     (dict(head_stride=1 << 62), OVERFLOW), (None, INVALID)], ids=str)
def test_scales_that_cannot_be(kw, code):
    sc = None if kw is None else scales(**kw)
    assert append(cache(), sc) == code and attend(cache(), sc) == code


def test_contiguous_scales():
    c = device.paged_cache(10, 48, 3, 64, 3, 4, "i8")
    for block in (1, 3, 16, 48):
        s = device.paged_scales(c, block)
        assert (s.block, s.head_stride, s.page_stride) == (block, 48 // block, 3 * (48 // block))
    assert device.paged_scales(c, 0).head_stride == 0  # refused by the calls


def test_append_refusals():
    sc = scales()
    assert append(None, sc) == INVALID and append(cache(), sc, none=("desc",)) == INVALID
    for kw in (dict(tokens=-1), dict(q_heads=-1), dict(rotary_dim=-2), dict(rotary_dim=63), dict(rotary_dim=66), dict(max_pos=-1), dict(q_row_stride=-1), dict(v_head_stride=-5),
               dict(out_row_stride=(1 << 40) + 1)):
        assert append(cache(), sc, **kw) == INVALID, kw
    assert append(cache(), sc, q_heads=1 << 40) == OVERFLOW and append(cache(), sc, tokens=1 << 31) == OVERFLOW
    for n in ("q", "k", "v", "cos", "sin", "table", "seq", "pos", "out", "kc", "vc", "ks", "vs"):
        assert append(cache(), sc, 1, none=(n,)) == INVALID, n
    assert append(cache(), sc, 1, none=("k", "v", "q", "out"), q_heads=0) == INVALID  # nothing to do
    assert append(cache(), sc, 0, none=("k", "v")) in OK


def test_attention_refusals():
    sc = scales()
    assert attend(cache(), sc, 0) in OK
    assert attend(None, sc, none=("q",)) == INVALID and attend(cache(), sc, none=("desc",)) == INVALID
    for kw in (dict(q_heads=0), dict(q_heads=3), dict(new_tokens=0), dict(new_tokens=9), dict(max_len=-1), dict(max_len=1 << 31), dict(q_seq_stride=-1), dict(o_head_stride=-1)):
        assert attend(cache(), sc, **kw) == INVALID, kw
    assert attend(cache(), sc, 1 << 30, q_heads=4) == OVERFLOW
    for n in ("q", "k", "v", "ks", "vs", "table", "lens", "out"):
        assert attend(cache(), sc, none=(n,)) == INVALID, n
    c = device.paged_cache(5000, 16, 8, 128, 2, 4000, "i8")
    need = _lib.load().fth_dev_paged_sdpa_scaled_workspace_bytes(C.byref(c), C.byref(device.paged_scales(c, 16)), C.byref(device.paged_sdpa_desc(c, 32)))
    assert 0 < need < 1 << 30  # asked for without a device; without it, smaller or askew the call is refused
    args = [1.0, P, P, P, P, P, P, P, P, None]
    for at, n in ((None, need), (4096, need - 1), (4100, need)):
        assert _lib.load().fth_dev_paged_sdpa_scaled_f32(C.byref(c), C.byref(device.paged_scales(c, 16)), C.byref(device.paged_sdpa_desc(c, 32)), *args, at, n, None) == INVALID


def test_sampling_refusals():
    fn = _lib.load().fth_dev_sample_f32

    def call(rows=0, vocab=100, none=(), desc=True, work=True, **kw):
        d = device.sample_desc(rows, vocab)
        for k, v in kw.items():
            setattr(d, k, v)
        args = {n: P for n in ("x", "t", "k", "p", "m", "u", "tokens", "lp")}
        args.update({n: None for n in none if n in args})
        need = _lib.load().fth_dev_sample_workspace_bytes(C.byref(d)) if desc else 0
        return fn(C.byref(d) if desc else None, *args.values(), None, P if work else None, need, None)

    assert call() in OK and call(vocab=0) in OK and call(none=("x", "u", "tokens")) in OK
    assert call(desc=False) == INVALID
    for kw in (dict(rows=-1), dict(vocab=-1), dict(logits_stride=99), dict(rows=1, vocab=0)):
        assert call(**kw) == INVALID, kw
    for kw in (dict(vocab=1 << 31), dict(rows=(1 << 20) + 1), dict(logits_stride=(1 << 40) + 1)):
        assert call(**kw) == OVERFLOW, kw
    for n in ("x", "u", "tokens"):
        assert call(1, none=(n,)) == INVALID, n


def test_struct_layouts():
    assert C.sizeof(_lib.PagedScales) == 3 * 8
    assert C.sizeof(_lib.SampleDesc) == 3 * 8
