"""Appends to a cache of 8-bit numbers in calls large enough to be cut otherwise: many single tokens, runs over several cuts, long blocks,
tokens left out at the cuts, runs past the rotation tables, and sizes that go past the caches."""
import numpy as np
import pytest

from frankentorch_amd.device import DeviceBuffer
from scaled_case import Scaled
from test_gpu_paged_append_scaled import Call, ragged, same

pytestmark = pytest.mark.gpu

KV, D = 16, 64  # 256 tokens are the last that go one by one, 1024 the last that go by four


def by_the_rules(hip, p, places, keep, first_bad, rotary=0, max_pos=0, inter=False, hq=1):
    """The call with all `places`, and the rules with those that `keep` (a mask) has; every other token's rows stay out of the cache."""
    device = p.upload()
    bad = DeviceBuffer.from_host(np.array([5], np.int64))
    call = Call(p, 91, places, hq, rotary, inter, max_pos)
    got = call.run(hip, device, bad)
    call.proj, call.seqs, call.positions = call.proj[keep], call.seqs[keep], call.positions[keep]
    want = call.expect()
    same(p)
    assert np.array_equal(got[keep].view(np.uint32), want.view(np.uint32))
    assert bad.to_host()[0] == first_bad


@pytest.mark.parametrize("tokens", [256, 257, 700, 1024, 1025, 1300])
@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_single_tokens(hip, tokens, dtype):
    """A step of many sequences, some of which are padding."""
    starts = [(7 * s) % 32 for s in range(tokens)]
    # a fifth of them has something in the block
    p = Scaled(90, tokens, KV, D, 16, 16, dtype, 2).fill(89, [0 if s % 5 else a for s, a in enumerate(starts)])
    starts = [a - a % 16 if s % 5 else a for s, a in enumerate(starts)]
    places = [(s, -1 if s % 11 == 3 else a) for s, a in enumerate(starts)]
    by_the_rules(hip, p, places, np.array([a >= 0 for _, a in places]), -1, 64, 40)


# (page, block, counts, starts)
PROMPTS = [(16, 16, [150, 90, 61], [5, 0, 33]), (48, 48, [150, 90, 61], [5, 0, 33]), (24, 24, [100, 200], [23, 1]), (128, 128, [190, 130], [3, 120]), (16, 8, [300], [4]), (16, 1, [299], [4]),
           (16, 16, [700, 1, 399], [5, 20, 0]), (64, 64, [700, 1, 399], [5, 20, 0]), (256, 256, [1100], [17]), (16, 4, [600, 500], [3, 1]), (32, 1, [1030], [9])]


@pytest.mark.parametrize("page,block,counts,starts", PROMPTS, ids=str)
@pytest.mark.parametrize("dtype,rotary,inter", [("i8", 64, False), ("e4m3", 32, True)])
def test_prompts(hip, page, block, counts, starts, dtype, rotary, inter):
    p = Scaled(92, len(counts), KV, D, page, block, dtype, -(-max(a + n for a, n in zip(starts, counts)) // page)).fill(93, starts)
    places = ragged(counts, starts)
    by_the_rules(hip, p, places, np.ones(len(places), bool), -1, rotary, 1200, inter, hq=3)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("count", [300, 1100])
def test_left_out_at_the_cuts(hip, block, count):
    """Tokens out of order, padding and places that do not exist at the first and last tokens of what a wavefront looks through. (A token out
    of order follows a token of its block in the list: elsewhere it would be that block's second place in the call.)"""
    p = Scaled(94, 2, KV, D, 64, block, "e4m3", -(-count // 64) + 9)
    places, keep = [], []
    at = 0
    for t in range(count):
        kind = {4: "again", 31: "none", 33: "again", 63: "hole", 65: "again", 95: "away", 96: "none", 128: "away", 160: "again"}.get(t)
        if kind is None:
            places.append((0, at))
            at += 1
        else:
            # the place before once more, the one behind a hole, no place, or a sequence that is not there
            assert kind not in ("again", "hole") or (keep[-1] and (at - 1) // block == (at + 1) // block or kind == "again" and keep[-1])
            places.append({"again": (0, at - 1), "hole": (0, at + 1), "none": (0, -1), "away": (5, 0)}[kind])
            at = -(-at // block) * block  # what follows starts a block of its own
        keep.append(kind is None)
    rows = np.array(keep)
    by_the_rules(hip, p, places, rows, 4)


@pytest.mark.parametrize("page,block,tokens", [(16, 16, 40), (64, 64, 40), (64, 64, 300), (64, 64, 1100), (256, 256, 1100), (16, 1, 40)])
def test_runs_past_the_tables(hip, page, block, tokens):
    """The first tokens of a run have an angle, the others none."""
    p = Scaled(95, 1, KV, D, page, block, "i8", -(-tokens // page))
    for max_pos in (tokens - 1, tokens - 9, tokens // 2 + 1):
        places = ragged([tokens], [0])
        by_the_rules(hip, p, places, np.arange(tokens) < max_pos, max_pos, 64, max_pos)


def test_past_the_caches(hip):
    """Rows and queries of more than 256 MB, against the same call from operands at addresses that are taken element by element."""
    n = 6300
    assert n * 128 * (8 * 32 + 10 * 8) > 1 << 28
    results = []
    for lead in (0, 1):
        p = Scaled(96, 2, 8, 128, 64, 32, "e4m3", 50)
        call = Call(p, 97, ragged([n // 2, n // 2], [0, 40]), 32, 128, False, 3200, lead=lead)
        out = call.run(hip, p.upload())
        results.append([out.view(np.uint32)] + [b.to_host().view(np.uint8) for b in p.buffers + p.scale_buffers])
    for a, b in zip(*results):
        assert np.array_equal(a, b)
