"""Timed cases of the operators that generate text token by token, each in its plain form and through the library.

  append   keys and values of new tokens into a paged cache, the position rotation of keys and queries applied on the way
  attend   attention of one to eight new tokens per sequence over the paged cache
  logits   penalties for repeated tokens, biases and a grammar's mask on the logits of a step

Inputs are torch tensors on the GPU. The plain form is elementary torch operations in float32, rounded once to the type of
the output; with `own` a pass is the library's calls on the same tensors. Lengths are ragged: a case fixes which lengths
there are, the seed which sequence has which, where its pages lie, and every value.
"""
import math
import random

import numpy as np
import torch

own = False

F32, F64, I32 = torch.float32, torch.float64, torch.int32
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one sequence of a GPT-2-small-shaped decoder, 37 tokens in: one layer's attention in an interactive session (latency)
        dict(name="attend_b1_h12_d64_k37", kind="attend", batch=1, hq=12, hkv=12, d=64, page=16, new=1, max_len=37, type="f32"),
        # eight such sequences, up to the decoder's 1024 positions, an fp32 cache
        dict(name="attend_b8_h12_d64_k1024", kind="attend", batch=8, hq=12, hkv=12, d=64, page=16, new=1, max_len=1024, type="f32"),
        # a serving batch: 64 ragged sequences, four query heads per K/V head, a cache in 16 bits
        dict(name="attend_b64_hq32_hkv8_k8191", kind="attend", batch=64, hq=32, hkv=8, d=128, page=16, new=1, max_len=8191, type="bf16"),
        # one user with a long document: the length is all there is to share out
        dict(name="attend_b1_hq32_hkv8_k131071", kind="attend", batch=1, hq=32, hkv=8, d=128, page=64, new=1, max_len=131071, type="bf16"),
        # four proposed tokens per sequence checked at once
        dict(name="attend_b16_hq32_hkv8_new4_k3967", kind="attend", batch=16, hq=32, hkv=8, d=128, page=32, new=4, max_len=3967, type="f16"),
        # one token's keys and values of one layer of the GPT-2-small-shaped decoder, learned positions (latency)
        dict(name="append_b1_h12_d64", kind="append", batch=1, new=1, start=900, hq=0, hkv=12, d=64, page=16, rotary=0, interleaved=False, type="f32"),
        # a decode step of a serving batch, keys and queries rotated
        dict(name="append_b64_hq32_hkv8", kind="append", batch=64, new=1, start=1500, hq=32, hkv=8, d=128, page=16, rotary=128, interleaved=False, type="bf16"),
        # eight prompts of up to 1024 tokens into the fp32 cache
        dict(name="append_b8_s1024_h12_d64", kind="append", batch=8, new=1024, start=0, hq=0, hkv=12, d=64, page=16, rotary=0, interleaved=False, type="f32"),
        # three long prompts, the first half of each head rotated in adjacent pairs, pages of 48 tokens
        dict(name="append_b3_s7001_hq32_hkv8", kind="append", batch=3, new=7001, start=500, hq=32, hkv=8, d=128, page=48, rotary=64, interleaved=True, type="f16"),
        # one row over the GPT-2 vocabulary (latency)
        dict(name="logits_1x50257", kind="logits", rows=1, vocab=50257, history=200, bias="none", mask=False),
        # a batch of 64 under a grammar, one bias for all
        dict(name="logits_64x50257", kind="logits", rows=64, vocab=50257, history=1024, bias="shared", mask=True),
        # a large vocabulary of an odd size, a bias per row, long histories
        dict(name="logits_200x131071", kind="logits", rows=200, vocab=131071, history=8000, bias="rows", mask=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "append", "logits"])
    if kind == "logits":
        rows = _log(rng, 1, 200)
        return dict(kind=kind, rows=rows, vocab=_log(rng, 1000, 131071), history=_log(rng, 1, 8000), bias=rng.choice(["none", "shared", "rows"]),
                    mask=rng.random() < 0.6)
    d = rng.choice([64, 64, 80, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 12])
    hq = hkv * rng.choice([1, 2, 4, 5, 8]) if hkv < 12 else 12
    name = rng.choice(["f32", "f16", "bf16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 128])
    if kind == "attend":
        batch, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7, 8])
        size = 4 if name == "f32" else 2
        most = int(5e8) // (batch * hkv * d * 2 * size)  # half a gigabyte of cache
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, d=d, page=page, new=new, max_len=max(new, _log(rng, 1, min(131071, most))), type=name)
    rotary = rng.choice([0, d, d, d // 2])
    batch = _log(rng, 1, 64)
    most = int(4e8) // (batch * 4 * (hq + 2 * hkv) * d * 2)
    new = 1 if rng.random() < 0.4 else _log(rng, 1, min(8192, most))
    return dict(kind=kind, batch=batch, new=new, start=rng.choice([0, 200, 1500]), hq=hq if rotary else 0, hkv=hkv, d=d, page=page, rotary=rotary,
                interleaved=rng.random() < 0.4, type=name)


# ---- inputs ----------------------------------------------------------------------------------------------------------


class _Maker:
    """Seeded inputs: one generator on the GPU and one on the host."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1000003 * int(seed) + 29)
        self.host = random.Random(7919 * int(seed) + 3)
        self.np = np.random.RandomState((7919 * int(seed) + 3) % (1 << 32))

    def normal(self, shape, std=1.0, dtype=F32):
        t = torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)
        return t if std == 1.0 else t.mul_(std)

    def uniform(self, shape, lo, hi):
        return torch.rand(shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)


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
    table = _pages(mk, lengths, case["page"], total, width)
    shape = (total, case["hkv"], case["page"], case["d"])
    q = mk.normal((case["batch"], case["new"], case["hq"], case["d"]), 1.5)
    return dict(q=q, k=mk.normal(shape, dtype=_TYPES[case["type"]]), v=mk.normal(shape, dtype=_TYPES[case["type"]]), table=table, width=width, total=total,
                lens=_ints(lengths), out=torch.empty_like(q), scale=1.0 / math.sqrt(case["d"]))


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
    k_at = (max(hq, hkv)) * d
    s = dict(q=proj[:, : hq * d], k=proj[:, k_at:k_at + hkv * d], v=proj[:, k_at + hkv * d:], pitch=proj.shape[1], tokens=tokens, table=table, width=width, total=total,
             seq_ids=_ints(np.repeat(np.arange(len(counts)), counts)), positions=_ints(np.concatenate([a + np.arange(n) for a, n in zip(starts, counts)])))
    shape = (total, hkv, case["page"], d)
    s["k_cache"], s["v_cache"] = (mk.normal(shape, dtype=_TYPES[case["type"]]) for _ in range(2))
    s["q_out"] = torch.empty((tokens, hq, d), device="cuda")
    s["cos"] = s["sin"] = None
    if case["rotary"]:
        s["max_pos"] = case["start"] + case["new"]
        angle = torch.arange(s["max_pos"], device="cuda", dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=F64) / case["rotary"])
        s["cos"], s["sin"] = angle.cos().to(F32), angle.sin().to(F32)
    return s


def _history_lengths(case):
    return _lengths(case["rows"], case["history"], case["history"] // 4)


def _prepare_logits(case, mk):
    rows, vocab, width = case["rows"], case["vocab"], case["history"]
    lengths = _history_lengths(case)
    mk.host.shuffle(lengths)
    # what text looks like: a few tokens come again and again, most are rare
    rank = mk.uniform((rows, width), 0.0, math.log(vocab)).exp().long().clamp(1, vocab) - 1
    s = dict(logits=mk.normal((rows, vocab), 3.0), history=((rank * 7919 + 13) % vocab).to(I32), history_len=_ints(lengths),
             prompt_len=_ints([mk.host.randint(0, n) for n in lengths]), repetition=mk.uniform((rows,), 1.0, 1.3), frequency=mk.uniform((rows,), 0.0, 0.6),
             presence=mk.uniform((rows,), -0.2, 0.6), bias=None, mask=None, out=torch.empty((rows, vocab), device="cuda"))
    if case["bias"] != "none":
        shape = (vocab,) if case["bias"] == "shared" else (rows, vocab)
        s["bias"] = mk.normal(shape, 2.0).mul_((mk.uniform(shape, 0.0, 1.0) < 0.01).to(F32))
    if case["mask"]:
        # every other row is free, the others may go on with few tokens
        words = (vocab + 31) // 32
        few = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=mk.g, device="cuda").to(I32)
        for _ in range(4):
            few &= torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=mk.g, device="cuda").to(I32)
        free = (torch.arange(rows, device="cuda") % 2 == 0)[:, None]
        s["mask"] = torch.where(free, torch.full_like(few, -1), few)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _sequences(cache, table):
    """The pages of every sequence one after the other: [batch, heads, positions, d] in float32."""
    x = cache[table.clamp(min=0).long()]
    b, p, h, n, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * n, d).to(F32)


def _plain_attend(case, s):
    b, new, hq, d = s["q"].shape
    hkv = case["hkv"]
    k, v = _sequences(s["k"], s["table"]), _sequences(s["v"], s["table"])
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


def _plain_append(case, s):
    t, d, pos = s["tokens"], case["d"], s["positions"].long()
    q, k, v = (s[n].reshape(t, -1, d) for n in ("q", "k", "v"))
    if case["rotary"]:
        cos, sin = s["cos"][pos], s["sin"][pos]
        q, k = (_rotate(x, cos, sin, case["rotary"], case["interleaved"]) for x in (q, k))
    page = s["table"][s["seq_ids"].long(), pos // case["page"]].long()
    s["k_cache"][page, :, pos % case["page"]] = k.to(s["k_cache"].dtype)
    s["v_cache"][page, :, pos % case["page"]] = v.to(s["v_cache"].dtype)
    return {"k": s["k_cache"], "v": s["v_cache"], **({"q": q} if case["hq"] else {})}


def _plain_logits(case, s):
    x, history = s["logits"], s["history"].long()
    at = torch.arange(history.shape[1], device="cuda")
    there = at < s["history_len"][:, None]
    count = lambda which: torch.zeros(x.shape, device="cuda", dtype=I32).scatter_add_(1, history, which.to(I32))
    seen, made = count(there) > 0, count(there & (at >= s["prompt_len"][:, None])).to(F32)
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * made
    x = x - s["presence"][:, None] * (made > 0).to(F32)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        v = torch.arange(x.shape[1], device="cuda")
        x = x.masked_fill((s["mask"][:, v // 32] >> (v % 32).to(I32)) & 1 == 0, -math.inf)
    return x


# ---- the library's calls ---------------------------------------------------------------------------------------------


class _Tensor:
    """A torch tensor as the device tier takes its operands."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _plan(case, s):
    """Descriptors, operands and workspace, made once and kept, as a program would."""
    from frankentorch_amd import device

    p = {n: _Tensor(x) for n, x in s.items() if isinstance(x, torch.Tensor)}
    if case["kind"] == "logits":
        p["desc"] = device.logits_desc(case["rows"], case["vocab"], case["history"], shared_bias=case["bias"] == "shared")
        return p
    p["cache"] = device.paged_cache(s["total"], case["page"], case["hkv"], case["d"], case["batch"], s["width"], case["type"])
    if case["kind"] == "attend":
        p["desc"] = device.paged_sdpa_desc(p["cache"], case["hq"], case["new"], case["max_len"])
        p["ws"] = device.paged_sdpa_workspace(p["cache"], p["desc"])
    else:
        p["desc"] = device.paged_append_desc(p["cache"], s["tokens"], case["hq"], case["rotary"], s.get("max_pos", 0), case["interleaved"], row_stride=s["pitch"])
    return p


def _own(case, s):
    from frankentorch_amd import device

    p = s.get("plan")
    if p is None:
        p = s["plan"] = _plan(case, s)
    if case["kind"] == "attend":
        device.paged_sdpa(p["cache"], p["desc"], s["scale"], p["q"], p["k"], p["v"], p["table"], p["lens"], p["out"], workspace=p["ws"])
        return s["out"]
    if case["kind"] == "append":
        device.paged_append(p["cache"], p["desc"], p["q"] if case["hq"] else None, p["k"], p["v"], p.get("cos"), p.get("sin"), p["table"], p["seq_ids"], p["positions"],
                            p["q_out"] if case["hq"] else None, p["k_cache"], p["v_cache"])
        return {"k": s["k_cache"], "v": s["v_cache"], **({"q": s["q_out"]} if case["hq"] else {})}
    device.logits_process(p["desc"], p["logits"], p["history"], p["history_len"], p["prompt_len"], p["repetition"], p["frequency"], p["presence"], p.get("bias"),
                          p.get("mask"), p["out"])
    return s["out"]


# ---- 64 bits, from the definitions ------------------------------------------------------------------------------------


def _exact_attend(case, s):
    page, hkv, new = case["page"], case["hkv"], case["new"]
    group = case["hq"] // hkv
    out = torch.zeros(s["q"].shape, device="cuda", dtype=F64)
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, : -(-n // page)].long()
        k, v = (s[c][ids].transpose(0, 1).reshape(hkv, -1, case["d"])[:, :n].to(F64) for c in ("k", "v"))
        for i in range(new):
            sees = n - new + 1 + i
            for g in range(group if sees > 0 else 0):
                heads = torch.arange(hkv, device="cuda") * group + g
                score = (k[:, :sees] * s["q"][b, i, heads].to(F64)[:, None]).sum(-1) * s["scale"]
                w = torch.exp(score - score.max(-1, keepdim=True).values)
                out[b, i, heads] = (w[..., None] * v[:, :sees]).sum(1) / w.sum(-1, keepdim=True)
    return out


def _exact_append(case, s):
    t, d, rotary, page = s["tokens"], case["d"], case["rotary"], case["page"]
    pos = s["positions"].long()
    slot = s["table"].long()[s["seq_ids"].long(), pos // page] * page + pos % page

    def turned(x):
        z = x.to(F64).reshape(t, -1, d).clone()
        if rotary:
            first = torch.arange(0, rotary, 2, device="cuda") if case["interleaved"] else torch.arange(rotary // 2, device="cuda")
            second = first + (1 if case["interleaved"] else rotary // 2)
            turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[pos][:, None]
            w = torch.complex(z[..., first], z[..., second]) * turn
            z[..., first], z[..., second] = w.real, w.imag
        return z

    def stored(cache, x):
        rows = cache.to(F64).transpose(1, 2).reshape(-1, case["hkv"], d).clone()
        rows[slot] = x
        return rows.reshape(cache.shape[0], page, case["hkv"], d).transpose(1, 2).contiguous()

    out = {"k": stored(s["k_cache"], turned(s["k"])), "v": stored(s["v_cache"], s["v"].to(F64).reshape(t, -1, d))}
    return {**out, **({"q": turned(s["q"])} if case["hq"] else {})}


def _exact_logits(case, s):
    out = torch.empty(s["logits"].shape, dtype=F64)
    history, bias = s["history"].cpu().numpy(), None if s["bias"] is None else s["bias"].double().cpu().numpy()
    for r in range(case["rows"]):
        x = s["logits"][r].double().cpu().numpy()
        n, prompt = int(s["history_len"][r]), int(s["prompt_len"][r])
        penalty, per, once = (float(s[name][r]) for name in ("repetition", "frequency", "presence"))
        seen = np.unique(history[r, :n])
        x[seen] = np.where(x[seen] > 0, x[seen] / penalty, x[seen] * penalty)
        made, times = np.unique(history[r, prompt:n], return_counts=True)
        x[made] -= per * times + once
        if bias is not None:
            x += bias if bias.ndim == 1 else bias[r]
        if s["mask"] is not None:
            allowed = np.unpackbits(s["mask"][r].cpu().numpy().view(np.uint8), bitorder="little")[: case["vocab"]]
            x[allowed == 0] = -np.inf
        out[r] = torch.from_numpy(x)
    return out.cuda()


# ---- entry points ------------------------------------------------------------------------------------------------------

_PREPARE = {"attend": _prepare_attend, "append": _prepare_append, "logits": _prepare_logits}
_PLAIN = {"attend": _plain_attend, "append": _plain_append, "logits": _plain_logits}
_EXACT = {"attend": _exact_attend, "append": _exact_append, "logits": _exact_logits}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, _Maker(seed)), case=case)


def run(state):
    case = state["case"]
    return _own(case, state) if own else _PLAIN[case["kind"]](case, state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, _PREPARE[case["kind"]](case, _Maker(seed)))


def work(case):
    if case["kind"] == "logits":
        n, words = case["rows"] * case["vocab"], (case["vocab"] + 31) // 32
        more = {"none": 0, "shared": 4 * case["vocab"], "rows": 4 * n}[case["bias"]] + (4 * case["rows"] * words if case["mask"] else 0)
        return {"bytes": 8 * n + more + 4 * sum(_history_lengths(case)), "flops": 4 * n}
    size, d = _TYPES[case["type"]].itemsize, case["d"]
    if case["kind"] == "attend":
        keys = sum(_attend_lengths(case))
        q = 4 * case["batch"] * case["new"] * case["hq"] * d
        return {"bytes": 2 * keys * case["hkv"] * d * size + 2 * q, "flops": 4 * keys * case["new"] * case["hq"] * d}
    tokens = sum(_append_counts(case))
    tables = 4 * case["rotary"] * min(tokens, case["start"] + case["new"])
    return {"bytes": tokens * (8 * case["hq"] * d + 2 * case["hkv"] * d * (4 + size) + 12) + tables, "flops": 3 * tokens * case["rotary"] * (case["hq"] + case["hkv"])}
