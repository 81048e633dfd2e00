"""Refusals of the operators on a paged cache and on logits: they come before any device is asked for, so they need none; what
is accepted gives Unavailable without a device. No pointer here is ever followed."""
import ctypes as C

import pytest

from frankentorch_amd import _lib, device

OK = (0, 100)  # accepted: nothing to do on a device, or no device
P = 4096       # stands for a device pointer
INVALID, OVERFLOW = 105, 102


def cache(**kw):
    c = device.paged_cache(10, 16, 2, 64, 3, 4, "bf16")
    for k, v in kw.items():
        setattr(c, k, v)
    return c


CACHES = [(dict(dtype=0), INVALID), (dict(dtype=4), INVALID), (dict(num_pages=-1), INVALID), (dict(num_seqs=-1), INVALID), (dict(max_pages=-1), INVALID),
          (dict(kv_heads=0), INVALID), (dict(page_size=0), INVALID), (dict(page_size=-16), INVALID), (dict(head_dim=0), INVALID), (dict(head_dim=257, row_stride=257), INVALID),
          (dict(page_stride=63), INVALID), (dict(head_stride=0), INVALID), (dict(row_stride=-64), INVALID), (dict(table_stride=3), INVALID),
          (dict(num_pages=1 << 31), OVERFLOW), (dict(max_pages=1 << 27, table_stride=1 << 27), OVERFLOW), (dict(page_stride=1 << 60), OVERFLOW),
          (dict(page_stride=1 << 62, num_pages=1 << 30), OVERFLOW), (dict(max_pages=1 << 62, table_stride=1 << 62), OVERFLOW), (dict(table_stride=1 << 62), OVERFLOW)]


def append(c, tokens=0, none=(), **kw):
    d = device.paged_append_desc(c, tokens, 4, 64, 100) if c is not None else _lib.PagedAppendDesc()
    for k, v in kw.items():
        setattr(d, k, v)
    args = {n: P for n in ("q", "k", "v", "cos", "sin", "table", "seq", "pos", "out", "kc", "vc")}
    args.update({n: None for n in none})
    args["q"] = 8192 if args["q"] else None
    return _lib.load().fth_dev_paged_append_f32(None if c is None else C.byref(c), None if "desc" in none else C.byref(d), *[args[n] for n in list(args)[:11]], None, None)


def attend(c, seqs=None, none=(), **kw):
    d = device.paged_sdpa_desc(c, 4, 1) if c is not None else _lib.PagedSdpaDesc()
    for k, v in kw.items():
        setattr(d, k, v)
    if seqs is not None:
        c.num_seqs = seqs
    args = {n: P for n in ("q", "k", "v", "table", "lens", "out")}
    args.update({n: None for n in none})
    rc = _lib.load().fth_dev_paged_sdpa_f32(None if c is None else C.byref(c), None if "desc" in none else C.byref(d), 1.0, *[args[n] for n in list(args)[:6]], None, None, 0, None)
    if rc and rc != 100 and not none:
        assert _lib.load().fth_dev_paged_sdpa_workspace_bytes(C.byref(c), C.byref(d)) == 0
    return rc


@pytest.mark.parametrize("kw,code", CACHES, ids=str)
def test_caches_that_cannot_be(kw, code):
    assert append(cache(**kw)) == code
    assert attend(cache(**kw)) == code
    assert _lib.last_error().message


def test_append_refusals():
    assert append(cache()) in OK
    assert append(None) == INVALID and append(cache(), none=("desc",)) == INVALID
    for kw in (dict(tokens=-1), dict(q_heads=-1), dict(rotary_dim=-2), dict(rotary_dim=63), dict(rotary_dim=66), dict(max_pos=-1), dict(q_row_stride=-1), dict(v_head_stride=-5),
               dict(out_row_stride=(1 << 40) + 1)):
        assert append(cache(), **kw) == INVALID, kw
    assert append(cache(), q_heads=1 << 40) == OVERFLOW
    assert append(cache(), tokens=1 << 31) == OVERFLOW
    assert append(cache(), 1, none=("k", "v", "q", "out"), q_heads=0) == INVALID  # nothing to do
    for n in ("q", "k", "v", "cos", "sin", "table", "seq", "pos", "out", "kc", "vc"):
        assert append(cache(), 1, none=(n,)) == INVALID, n


def test_attention_refusals():
    assert attend(cache(), 0) in OK
    assert attend(None, none=("q",)) == INVALID and attend(cache(), none=("desc",)) == INVALID
    for kw in (dict(q_heads=0), dict(q_heads=3), dict(q_heads=-4), dict(new_tokens=0), dict(new_tokens=9), dict(max_len=-1), dict(max_len=1 << 31), dict(q_seq_stride=-1),
               dict(o_head_stride=-1), dict(q_row_stride=(1 << 40) + 1)):
        assert attend(cache(), **kw) == INVALID, kw
    assert attend(cache(), 1 << 30, q_heads=4) == OVERFLOW
    assert attend(cache(), q_heads=1 << 62) == OVERFLOW and attend(cache(), 0, q_heads=1 << 62) == OVERFLOW
    for n in ("q", "k", "v", "table", "lens", "out"):
        assert attend(cache(), none=(n,)) == INVALID, n


def test_the_workspace_is_asked_for_without_a_device():
    c = device.paged_cache(5000, 16, 8, 128, 2, 4000, "bf16")
    need = lambda c, **kw: _lib.load().fth_dev_paged_sdpa_workspace_bytes(C.byref(c), C.byref(device.paged_sdpa_desc(c, 32, **kw)))
    assert 0 <= need(c) < 1 << 30
    assert need(device.paged_cache(0, 16, 8, 128, 0, 0, "f32")) == 0


def test_logits_refusals():
    fn = _lib.load().fth_dev_logits_process_f32

    def call(rows=0, vocab=100, none=(), desc=True, same=False, **kw):
        d = device.logits_desc(rows, vocab, 10)
        for k, v in kw.items():
            setattr(d, k, v)
        args = {n: P for n in ("x", "h", "hl", "pl", "rep", "freq", "pres", "bias", "mask")}
        args.update({n: None for n in none})
        out = P if same else 8192
        return fn(C.byref(d) if desc else None, *[args[n] for n in list(args)[:9]], None if "out" in none else out, None, None)

    assert call() in OK and call(vocab=0) in OK
    assert call(desc=False) == INVALID
    for kw in (dict(rows=-1), dict(vocab=-1), dict(logits_stride=99), dict(out_stride=0), dict(history_stride=-1), dict(bias_stride=99), dict(bias_stride=-1), dict(mask_stride=3)):
        assert call(**kw) == INVALID, kw
    for kw in (dict(vocab=1 << 31), dict(rows=(1 << 20) + 1), dict(logits_stride=(1 << 40) + 1)):
        assert call(**kw) == OVERFLOW, kw
    for n in ("x", "hl", "pl", "out"):
        assert call(1, none=(n,)) == INVALID, n
    assert call(1, same=True, out_stride=101) == INVALID
    # what is not given is not looked at
    assert call(none=("h", "bias", "mask"), history_stride=-1, bias_stride=1, mask_stride=0) in OK


def test_struct_layouts():
    assert C.sizeof(_lib.PagedCache) == 10 * 8 + 8
    assert C.sizeof(_lib.PagedAppendDesc) == 12 * 8 + 8
    assert C.sizeof(_lib.PagedSdpaDesc) == 9 * 8
    assert C.sizeof(_lib.LogitsDesc) == 7 * 8
