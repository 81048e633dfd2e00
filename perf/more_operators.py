"""Timed cases of the 8-bit paged cache and of sampling, each in its plain form and through the library.

  append   keys and values of new tokens into a cache of 8-bit numbers with a scale for each block of tokens and head: rotation,
           the blocks' scales, what a block holds brought to a grown scale, rounding
  attend   attention of one to eight new tokens per sequence over such a cache
  sample   the next token of each row of logits from a given uniform number: temperature, top-k, top-p, min-p

Inputs are torch tensors on the GPU. The plain form is elementary torch operations in float32 (sampling in float64: which side of
a border a number lies on decides the token); with `own` a pass is the library's calls on the same tensors. Lengths are ragged: a
case fixes which lengths there are, the seed which sequence has which, where its pages lie, and every value.
"""
import math
import random

import numpy as np
import torch

own = False

F32, F64, I32, U8 = torch.float32, torch.float64, torch.int32, torch.uint8
_TYPES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
_LARGEST = {"e4m3": 448.0, "i8": 127.0}


# ---- the cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one sequence of a GPT-2-small-shaped decoder, 37 tokens in: one layer's attention in an interactive session (latency)
        dict(name="attend_b1_h12_d64_k37", kind="attend", batch=1, hq=12, hkv=12, d=64, page=16, block=16, new=1, max_len=37, type="e4m3"),
        # eight such sequences, up to the decoder's 1024 positions, whole numbers in the cache
        dict(name="attend_b8_h12_d64_k1024", kind="attend", batch=8, hq=12, hkv=12, d=64, page=16, block=16, new=1, max_len=1024, type="i8"),
        # a serving batch: 64 ragged sequences, four query heads per K/V head
        dict(name="attend_b64_hq32_hkv8_k8191", kind="attend", batch=64, hq=32, hkv=8, d=128, page=16, block=16, new=1, max_len=8191, type="e4m3"),
        # one user with a long document: the length is all there is to share out
        dict(name="attend_b1_hq32_hkv8_k131071", kind="attend", batch=1, hq=32, hkv=8, d=128, page=64, block=64, new=1, max_len=131071, type="e4m3"),
        # four proposed tokens per sequence checked at once, a scale for every token
        dict(name="attend_b16_hq32_hkv8_new4_k3967", kind="attend", batch=16, hq=32, hkv=8, d=128, page=32, block=1, new=4, max_len=3967, type="i8"),
        # a decode step of a serving batch, keys and queries rotated: blocks that hold tokens already (latency)
        dict(name="append_b64_hq32_hkv8", kind="append", batch=64, new=1, start=1500, hq=32, hkv=8, d=128, page=16, block=16, rotary=128, interleaved=False, type="e4m3"),
        # eight prompts of up to 1024 tokens, learned positions
        dict(name="append_b8_s1024_h12_d64", kind="append", batch=8, new=1024, start=0, hq=0, hkv=12, d=64, page=16, block=16, rotary=0, interleaved=False, type="i8"),
        # three long prompts behind what is there, the first half of each head rotated in adjacent pairs, pages of 48 tokens
        dict(name="append_b3_s7001_hq32_hkv8", kind="append", batch=3, new=7001, start=500, hq=32, hkv=8, d=128, page=48, block=48, rotary=64, interleaved=True, type="e4m3"),
        # one row over the GPT-2 vocabulary, the usual settings of a chat (latency)
        dict(name="sample_1x50257", kind="sample", rows=1, vocab=50257, top_k=50, top_p=0.95, min_p=0.0, masked=False, ties=False),
        # a batch of 16 at a temperature alone: every token may come
        dict(name="sample_16x50257", kind="sample", rows=16, vocab=50257, top_k=0, top_p=1.0, min_p=0.0, masked=False, ties=False),
        # a batch of 64 under a grammar, logits of a bf16 product (many are equal), a nucleus and a floor
        dict(name="sample_64x50257", kind="sample", rows=64, vocab=50257, top_k=0, top_p=0.9, min_p=0.02, masked=True, ties=True),
        # a large vocabulary of an odd size, every row with its own settings up to a wide nucleus
        dict(name="sample_200x131071", kind="sample", rows=200, vocab=131071, top_k=1000, top_p=0.98, min_p=0.0, masked=False, ties=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "append", "sample"])
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 200), vocab=_log(rng, 1000, 131071), top_k=rng.choice([0, 0, _log(rng, 1, 5000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 1.0), 3)]), min_p=rng.choice([0.0, 0.0, round(math.exp(rng.uniform(-7.0, -1.0)), 4)]),
                    masked=rng.random() < 0.4, ties=rng.random() < 0.4)
    d = rng.choice([64, 64, 80, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 12])
    hq = hkv * rng.choice([1, 2, 4, 5, 8]) if hkv < 12 else 12
    name = rng.choice(["e4m3", "i8"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 128])
    block = rng.choice([1, page, page, 16 if page % 16 == 0 else 4])
    if kind == "attend":
        batch, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7, 8])
        most = int(5e8) // (batch * hkv * d * 2)  # half a gigabyte of cache
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, d=d, page=page, block=block, new=new, max_len=max(new, _log(rng, 1, min(131071, most))), type=name)
    rotary = rng.choice([0, d, d, d // 2])
    batch = _log(rng, 1, 64)
    most = int(4e8) // (batch * 4 * (hq + 2 * hkv) * d * 2)
    new = 1 if rng.random() < 0.4 else _log(rng, 1, min(8192, most))
    return dict(kind=kind, batch=batch, new=new, start=rng.choice([0, 200, 1500]), hq=hq if rotary else 0, hkv=hkv, d=d, page=page, block=block, rotary=rotary,
                interleaved=rng.random() < 0.4, type=name)


# ---- numbers of 8 bits -----------------------------------------------------------------------------------------------


def _scale_for(largest, name):
    """The smallest power of two (2^-126 at least) whose multiples of the type reach `largest`; 0 for zeros alone, NaN for what is not finite."""
    m, e = torch.frexp(largest)
    top, bits = math.frexp(_LARGEST[name])
    s = torch.ldexp(torch.ones_like(largest), (e - bits + (m > top).to(I32)).clamp(min=-126))
    s = torch.where(largest == 0, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(largest), s, torch.full_like(s, math.nan))


def _per(scale):
    """1 / scale, 0 where the scale is 0 or NaN."""
    return torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))


def _rounded(x, name):
    """float32 to the storage type, to nearest even, as raw bytes; what is not finite becomes 0."""
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).clamp(-_LARGEST[name], _LARGEST[name])
    x = torch.round(x) if name == "i8" else x
    return x.to(_TYPES[name]).view(U8)


def _values(raw, name):
    return raw.view(_TYPES[name]).to(F32)


# ---- inputs ----------------------------------------------------------------------------------------------------------


class _Maker:
    """Seeded inputs: one generator on the GPU and one on the host."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1000003 * int(seed) + 41)
        self.host = random.Random(7919 * int(seed) + 5)
        self.np = np.random.RandomState((7919 * int(seed) + 5) % (1 << 32))

    def normal(self, shape, std=1.0):
        t = torch.randn(shape, generator=self.g, device="cuda")
        return t if std == 1.0 else t.mul_(std)

    def uniform(self, shape, lo, hi, dtype=F32):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=dtype).mul_(hi - lo).add_(lo)

    def cache(self, pages, hkv, page, d, block, name):
        """A filled cache [pages, hkv, page, d] and its scales [pages, hkv, page / block]: rows whose size differs from token to token."""
        x = self.normal((pages, hkv, page, d)).mul_(self.normal((pages, hkv, page, 1), 0.5).exp_())
        s = _scale_for(x.reshape(pages, hkv, page // block, block * d).abs().amax(-1), name)
        x = x.mul_(_per(s).repeat_interleave(block, 2)[..., None])
        return _rounded(x, name).view(_TYPES[name]), s


def _ints(values):
    return torch.tensor(np.asarray(values, dtype=np.int32), device="cuda")


def _lengths(batch, most, least):
    """`batch` lengths from `most` down to nearly `least`, evenly spread."""
    return [most - (most - least) * b // batch for b in range(batch)]


def _pages(mk, lengths, page, total, width):
    """A block table of pages in no order, -1 behind a sequence's own."""
    counts = [-(-n // page) for n in lengths]
    order = mk.np.permutation(total).astype(np.int32)
    table = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return _ints(table)


def _attend_lengths(case):
    return _lengths(case["batch"], case["max_len"], max(case["new"], case["max_len"] // 8))


def _prepare_attend(case, mk):
    lengths = _attend_lengths(case)
    mk.host.shuffle(lengths)
    total, width = sum(-(-n // case["page"]) for n in lengths) + 3, -(-case["max_len"] // case["page"])
    s = dict(q=mk.normal((case["batch"], case["new"], case["hq"], case["d"]), 1.5), table=_pages(mk, lengths, case["page"], total, width), width=width, total=total,
             lens=_ints(lengths), scale=1.0 / math.sqrt(case["d"]))
    for n in ("k", "v"):
        s[n], s[n + "_scales"] = mk.cache(total, case["hkv"], case["page"], case["d"], case["block"], case["type"])
    return dict(s, out=torch.empty_like(s["q"]))


def _append_counts(case):
    return _lengths(case["batch"], case["new"], max(1, case["new"] // 4))


def _prepare_append(case, mk):
    counts = _append_counts(case)
    mk.host.shuffle(counts)
    starts = [mk.host.randint(case["start"] // 2, case["start"]) for _ in counts]
    width = -(-(case["start"] + case["new"]) // case["page"])
    total = case["batch"] * width + 3
    table = _pages(mk, [a + n for a, n in zip(starts, counts)], case["page"], total, width)
    tokens, d, hq, hkv = sum(counts), case["d"], case["hq"], case["hkv"]
    proj = mk.normal((tokens, (max(hq, hkv) + 2 * hkv) * d))  # the packed projection of the step: queries, keys, values
    proj.mul_(mk.normal((tokens, 1), 0.5).exp_())
    k_at = (max(hq, hkv)) * d
    s = dict(q=proj[:, : hq * d], k=proj[:, k_at:k_at + hkv * d], v=proj[:, k_at + hkv * d:], pitch=proj.shape[1], tokens=tokens, table=table, width=width, total=total,
             seq_ids=_ints(np.repeat(np.arange(len(counts)), counts)), positions=_ints(np.concatenate([a + np.arange(n) for a, n in zip(starts, counts)])))
    for n in ("k", "v"):
        s[n + "_cache"], s[n + "_scales"] = mk.cache(total, hkv, case["page"], d, case["block"], case["type"])
    s["q_out"] = torch.empty((tokens, hq, d), device="cuda")
    s["cos"] = s["sin"] = None
    if case["rotary"]:
        s["max_pos"] = case["start"] + case["new"]
        angle = torch.arange(s["max_pos"], device="cuda", dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=F64) / case["rotary"])
        s["cos"], s["sin"] = angle.cos().to(F32), angle.sin().to(F32)
    return s


def _prepare_sample(case, mk):
    rows, vocab = case["rows"], case["vocab"]
    # what a model answers: a broad crowd of unlikely tokens, one in a hundred well above it
    x = mk.normal((rows, vocab), 2.0)
    x += mk.uniform((rows, vocab), 0.0, 11.0) * (mk.uniform((rows, vocab), 0.0, 1.0) < 0.01)
    if case["ties"]:
        x = x.to(torch.bfloat16).to(F32)
    if case["masked"]:
        x = x.masked_fill(mk.uniform((rows, vocab), 0.0, 1.0) < 0.9, -math.inf)
        x[:, 7] = 1.0  # something is always allowed
    full = lambda value, dtype: torch.full((rows,), value, device="cuda", dtype=dtype)
    # requests of one batch have settings of their own; the first row has the case's
    vary = mk.uniform((rows,), 0.5, 1.0)
    vary[0] = 1.0
    return dict(logits=x, temperature=mk.uniform((rows,), 0.6, 1.2), top_k=(full(case["top_k"], F32) * vary).ceil().to(I32), top_p=full(case["top_p"], F32) * vary if case["top_p"] < 1 else full(1.0, F32),
                min_p=full(case["min_p"], F32) * vary, uniform=mk.uniform((rows,), 0.0, 1.0, F64), tokens=torch.empty((rows,), device="cuda", dtype=I32),
                logprobs=torch.empty((rows,), device="cuda"))


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _sequences(case, cache, scales, table):
    """The pages of every sequence one after the other, as the values they stand for: [batch, heads, positions, d] in float32."""
    at = table.clamp(min=0).long()
    x = _values(cache.view(U8)[at], case["type"]) * scales[at].repeat_interleave(case["block"], 3)[..., None]
    b, p, h, n, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * n, d)


def _plain_attend(case, s):
    b, new, hq, d = s["q"].shape
    hkv = case["hkv"]
    k, v = (_sequences(case, s[n], s[n + "_scales"], s["table"]) for n in ("k", "v"))
    at = torch.arange(k.shape[2], device="cuda")
    lens = s["lens"].long()
    v.masked_fill_((at >= lens[:, None])[:, None, :, None], 0.0)
    q = s["q"].permute(0, 2, 1, 3).reshape(b, hkv, hq // hkv * new, d)
    scores = torch.matmul(k, q.transpose(2, 3).contiguous()).transpose(2, 3) * s["scale"]
    seen = lens[:, None] - new + 1 + torch.arange(new, device="cuda")  # keys that each of the new tokens sees
    hidden = (at >= seen[:, :, None])[:, None, None]
    scores = scores.reshape(b, hkv, hq // hkv, new, -1).masked_fill(hidden, -math.inf)
    w = (scores - scores.amax(-1, keepdim=True)).exp()
    w = w / w.sum(-1, keepdim=True)
    out = torch.matmul(w.reshape(b, hkv, hq // hkv * new, -1), v)
    return out.reshape(b, hq, new, d).permute(0, 2, 1, 3).contiguous()


def _rotate(x, cos, sin, rotary, interleaved):
    """The rotation of x [tokens, heads, d] by cos, sin [tokens, rotary / 2] of each token's position."""
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., rotary:]], -1)
    a, b = x[..., : rotary // 2], x[..., rotary // 2:rotary]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rotary:]], -1)


def _store(case, cache, scales, x, page, row):
    """Rows x [tokens, heads, d] at (page, row) of each token. The blocks that they fall into get the scale that the largest of them
    needs, if what is before the first of them does not have a larger one; what is before is rounded to that scale."""
    name, block, hkv = case["type"], case["block"], case["hkv"]
    pages, _, size, d = cache.shape
    per_page = size // block
    number = page * per_page + row // block  # the block of each token
    tokens = torch.arange(x.shape[0], device="cuda")
    blocks, member = torch.unique(number, return_inverse=True)
    first = torch.full(blocks.shape, block, device="cuda", dtype=torch.int64).scatter_reduce_(0, member, row % block, "amin")
    needs = torch.zeros((blocks.shape[0], hkv), device="cuda").scatter_reduce_(0, member[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
    p, i = blocks // per_page, blocks % per_page
    had = scales[p, :, i] * (first > 0)[:, None].to(F32)
    now = torch.maximum(had, _scale_for(needs, name))
    raw = cache.view(U8).view(pages, hkv, per_page, block, d)
    old = raw[p, :, i]
    kept = _rounded(_values(old, name) * (had * _per(now))[..., None, None], name)
    before = (torch.arange(block, device="cuda") < first[:, None])[:, None, :, None]
    raw[p, :, i] = torch.where(before, kept, old)
    cache.view(U8)[page, :, row] = _rounded(x * _per(now)[member][..., None], name)
    scales[p, :, i] = now


def _plain_append(case, s):
    t, d, pos = s["tokens"], case["d"], s["positions"].long()
    q, k, v = (s[n].reshape(t, -1, d) for n in ("q", "k", "v"))
    if case["rotary"]:
        cos, sin = s["cos"][pos], s["sin"][pos]
        q, k = (_rotate(x, cos, sin, case["rotary"], case["interleaved"]) for x in (q, k))
    page, row = s["table"][s["seq_ids"].long(), pos // case["page"]].long(), pos % case["page"]
    _store(case, s["k_cache"], s["k_scales"], k, page, row)
    _store(case, s["v_cache"], s["v_scales"], v, page, row)
    return _appended(case, s, q)


def _appended(case, s, q):
    """What is held after an append: the 8-bit numbers' values and the scales that they are times, each apart (their products would be another pass over the whole cache)."""
    return {**{n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}, **({"q": q} if case["hq"] else {})}


def _plain_sample(case, s):
    x, rows, vocab = s["logits"], case["rows"], case["vocab"]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal ones: the lowest index first
    w = ((x.to(F64) - x[:, :1].to(F64)) / s["temperature"].to(F64)[:, None]).exp()
    at = torch.arange(vocab, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"].long().clamp(max=vocab), torch.full_like(s["top_k"], vocab).long())
    w = w * (at < k[:, None])
    upto = w.cumsum(1)
    p = s["top_p"].to(F64)[:, None]
    need = p * upto[:, -1:]
    inside = (upto - w < need) | (p >= 1) | (at == 0)  # one more as long as those before it do not reach the share
    w = w * inside * ((w >= s["min_p"].to(F64)[:, None]) | (at == 0))
    total = w.sum(1)
    w = torch.zeros_like(w).scatter_(1, order, w)  # back to the order of the vocabulary
    run_up = w.cumsum(1)
    token = (run_up <= (s["uniform"] * total)[:, None]).sum(1)
    last = (vocab - 1 - (w.flip(1) > 0).to(I32).argmax(1)).to(token.dtype)
    token = torch.minimum(token, last)
    return {"tokens": token.to(I32), "logprobs": (w.gather(1, token[:, None])[:, 0] / total).log().to(F32)}


# ---- the library's calls ---------------------------------------------------------------------------------------------


class _Tensor:
    """A torch tensor as the device tier takes its operands."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _plan(case, s):
    """Descriptors, operands and workspace, made once and kept, as a program would."""
    from frankentorch_amd import device

    p = {n: _Tensor(x) for n, x in s.items() if isinstance(x, torch.Tensor)}
    if case["kind"] == "sample":
        p["desc"] = device.sample_desc(case["rows"], case["vocab"])
        p["ws"] = device.sample_workspace(p["desc"])
        return p
    p["cache"] = device.paged_cache(s["total"], case["page"], case["hkv"], case["d"], case["batch"], s["width"], case["type"])
    p["scales"] = device.paged_scales(p["cache"], case["block"])
    if case["kind"] == "attend":
        p["desc"] = device.paged_sdpa_desc(p["cache"], case["hq"], case["new"], case["max_len"])
        p["ws"] = device.paged_sdpa_scaled_workspace(p["cache"], p["scales"], p["desc"])
    else:
        p["desc"] = device.paged_append_desc(p["cache"], s["tokens"], case["hq"], case["rotary"], s.get("max_pos", 0), case["interleaved"], row_stride=s["pitch"])
    return p


def _own(case, s):
    from frankentorch_amd import device

    p = s.get("plan")
    if p is None:
        p = s["plan"] = _plan(case, s)
    if case["kind"] == "attend":
        device.paged_sdpa_scaled(p["cache"], p["scales"], p["desc"], s["scale"], p["q"], p["k"], p["v"], p["k_scales"], p["v_scales"], p["table"], p["lens"], p["out"],
                                 workspace=p["ws"])
        return s["out"]
    if case["kind"] == "append":
        device.paged_append_scaled(p["cache"], p["scales"], p["desc"], p["q"] if case["hq"] else None, p["k"], p["v"], p.get("cos"), p.get("sin"), p["table"], p["seq_ids"],
                                   p["positions"], p["q_out"] if case["hq"] else None, p["k_cache"], p["v_cache"], p["k_scales"], p["v_scales"])
        return _appended(case, s, s["q_out"])
    device.sample(p["desc"], p["logits"], p["temperature"], p["top_k"], p["top_p"], p["min_p"], p["uniform"], p["tokens"], p["logprobs"], workspace=p["ws"])
    return {"tokens": s["tokens"], "logprobs": s["logprobs"]}


# ---- 64 bits, from the definitions ------------------------------------------------------------------------------------


def _exact_attend(case, s):
    page, hkv, new = case["page"], case["hkv"], case["new"]
    group = case["hq"] // hkv
    out = torch.zeros(s["q"].shape, device="cuda", dtype=F64)
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, : -(-n // page)].long()
        rows = torch.arange(page, device="cuda") // case["block"]
        k, v = ((s[c].view(U8)[ids].view(_TYPES[case["type"]]).to(F64) * s[c + "_scales"].to(F64)[ids][:, :, rows, None]).transpose(0, 1).reshape(hkv, -1, case["d"])[:, :n]
                for c in ("k", "v"))
        for i in range(new):
            sees = n - new + 1 + i
            for g in range(group if sees > 0 else 0):
                heads = torch.arange(hkv, device="cuda") * group + g
                score = (k[:, :sees] * s["q"][b, i, heads].to(F64)[:, None]).sum(-1) * s["scale"]
                w = torch.exp(score - score.max(-1, keepdim=True).values)
                out[b, i, heads] = (w[..., None] * v[:, :sees]).sum(1) / w.sum(-1, keepdim=True)
    return out


def _grid(x, name):
    """x (float64, within the type's range) on the grid of the 8-bit type, to nearest even."""
    if name == "i8":
        return x.round()
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x)[1].clamp(min=-5) - 4)  # 3 bits behind the first; 2^-9 at least
    return (x / step).round() * step


def _exact_append(case, s):
    t, d, rotary, page, name, block = s["tokens"], case["d"], case["rotary"], case["page"], case["type"], case["block"]
    pos = s["positions"].long()
    pages = s["table"].long()[s["seq_ids"].long(), pos // page]

    def turned(x):
        z = x.to(F64).reshape(t, -1, d).clone()
        if rotary:
            first = torch.arange(0, rotary, 2, device="cuda") if case["interleaved"] else torch.arange(rotary // 2, device="cuda")
            second = first + (1 if case["interleaved"] else rotary // 2)
            turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[pos][:, None]
            w = torch.complex(z[..., first], z[..., second]) * turn
            z[..., first], z[..., second] = w.real, w.imag
        return z

    def stored(cache, scales, x):
        codes = cache.view(U8).view(_TYPES[name]).to(F64).transpose(1, 2).reshape(-1, case["hkv"], d).clone()  # [page x row, head, d]
        sc = scales.to(F64).transpose(1, 2).reshape(-1, case["hkv"]).clone()                                   # [page x block, head]
        at = pages * page + pos % page
        codes = codes.reshape(-1, block, case["hkv"], d)
        fresh = torch.zeros_like(codes).reshape(-1, case["hkv"], d)
        fresh[at] = x
        new = torch.zeros(codes.shape[0] * block, dtype=torch.bool, device="cuda")
        new[at] = True
        fresh, new = fresh.reshape(codes.shape), new.reshape(-1, block)
        touched = new.any(1)
        before = (new.to(I32).cumsum(1) == 0) & touched[:, None]
        largest = fresh.abs().amax((1, 3))
        want = torch.exp2(torch.ceil(torch.log2(largest / _LARGEST[name]).clamp(min=-126)))
        want[largest == 0] = 0.0
        now = torch.where(touched[:, None], torch.maximum(want, sc * before.any(1)[:, None]), sc)
        per = torch.where(now > 0, 1 / now, torch.zeros_like(now))[:, None, :, None]
        codes = torch.where(before[..., None, None], _grid(codes * sc[:, None, :, None] * per, name), codes)
        codes = torch.where(new[..., None, None], _grid(fresh * per, name), codes)
        codes = codes.reshape(cache.shape[0], page, case["hkv"], d).transpose(1, 2).contiguous()
        return codes, now.reshape(cache.shape[0], page // block, case["hkv"]).transpose(1, 2).contiguous()

    out = {}
    for n, x in (("k", turned(s["k"])), ("v", s["v"].to(F64).reshape(t, -1, d))):
        out[n + "_cache"], out[n + "_scales"] = stored(s[n + "_cache"], s[n + "_scales"], x)
    return {**out, **({"q": turned(s["q"])} if case["hq"] else {})}


def _exact_sample(case, s):
    x, tokens, logprobs = s["logits"].cpu().numpy(), [], []
    t, k, p, m, u = (s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    for r in range(case["rows"]):
        order = np.lexsort((np.arange(case["vocab"]), -x[r]))
        w = np.exp((x[r][order].astype(np.float64) - float(x[r].max())) / t[r])
        n = int(k[r]) if k[r] > 0 else len(w)
        w = w[:n]
        if p[r] < 1:
            w = w[: int(np.searchsorted(np.cumsum(w), p[r] * math.fsum(w))) + 1]
        w = w[: max(1, int((w >= m[r]).sum()))]
        total = math.fsum(w)
        by_index = np.argsort(order[: len(w)])
        chosen = min(int(np.searchsorted(np.cumsum(w[by_index]), u[r] * total, side="right")), len(w) - 1)
        tokens.append(int(order[by_index[chosen]]))
        logprobs.append(math.log(w[by_index[chosen]] / total))
    return {"tokens": torch.tensor(tokens, dtype=I32), "logprobs": torch.tensor(logprobs, dtype=F64)}


# ---- entry points ------------------------------------------------------------------------------------------------------

_PREPARE = {"attend": _prepare_attend, "append": _prepare_append, "sample": _prepare_sample}
_PLAIN = {"attend": _plain_attend, "append": _plain_append, "sample": _plain_sample}
_EXACT = {"attend": _exact_attend, "append": _exact_append, "sample": _exact_sample}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, _Maker(seed)), case=case)


def run(state):
    case = state["case"]
    return _own(case, state) if own else _PLAIN[case["kind"]](case, state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, _PREPARE[case["kind"]](case, _Maker(seed)))


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["rows"], "flops": 4 * n}
    d, block = case["d"], case["block"]
    if case["kind"] == "attend":
        lengths = _attend_lengths(case)
        keys, blocks = sum(lengths), sum(-(-n // block) for n in lengths)
        q = 4 * case["batch"] * case["new"] * case["hq"] * d
        return {"bytes": 2 * case["hkv"] * (keys * d + 4 * blocks) + 2 * q, "flops": 4 * keys * case["new"] * case["hq"] * d}
    counts = _append_counts(case)
    tokens, blocks = sum(counts), sum(-(-n // block) for n in counts)
    tables = 4 * case["rotary"] * min(tokens, case["start"] + case["new"])
    return {"bytes": tokens * (8 * case["hq"] * d + 2 * case["hkv"] * d * 5 + 12) + 8 * case["hkv"] * blocks + tables,
            "flops": 3 * tokens * case["rotary"] * (case["hq"] + case["hkv"]) + 4 * tokens * case["hkv"] * d}
