"""The paged prefill's plan on the CPU, key by key: the pieces that a token's keys are cut
into follow one another without a gap or an overlap, from the first to the last that it
sees; and long requests are cut whatever else is in the batch."""
import heapq
import random

import numpy as np
import pytest

from test_paged_plan_cpu import PACKED, _plan

STEP_US, SHARED_US, START_US = 1.8, 1.3, 6.0  # the plan's own costs


def _pieces(reqs, hq, hkv, page, causal=1, sms=148):
    """Items of the plan; {(request, token): [(first, end) key tile of each item]}, and the key
    tiles that the token's tile of rows needs."""
    out, items, rows, cq, ck = _plan(reqs, hq, hkv, page, causal, sms)
    owner = {int(cq[b]): b for b in range(len(reqs)) if reqs[b][0] > 0}
    cover, want = {}, {}
    for it in items:
        q_tok, q_len, k_len, _, row, n0, n1, flags, kt0, kt1, _, _ = (int(x) for x in it)
        b = owner[q_tok]
        nq, nk = reqs[b]
        for first, m in ((row, n0), (row + n0, n1)):
            end = min(nk, nk - nq + first + m) if causal else nk
            tiles = -(-max(0, end) // 128)
            for tok in range(first, first + m):
                assert want.setdefault((b, tok), tiles) == tiles
                cover.setdefault((b, tok), []).append((kt0, min(kt1, tiles)))
    return out, items, cover, want


def _exactly_once(cover, want):
    for key, ranges in cover.items():
        at = 0
        for lo, hi in sorted(r for r in ranges if r[0] < r[1]):
            assert lo == at, (key, ranges)
            at = hi
        assert at == want[key], (key, ranges, want[key])


def _batch(rng):
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 7, 8, 16, 130])
    reqs = [(rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 700)]),
             rng.choice([0, rng.randint(1, 300), rng.randint(1, 20000)])) for _ in range(rng.randint(1, 12))]
    return reqs, hq, hkv, rng.choice([16, 32, 64, 128, 256]), rng.randint(0, 1), rng.choice([0, 1, 7, 148])


def test_every_key_tile_once():
    rng = random.Random(1)
    for _ in range(60):
        reqs, hq, hkv, page, causal, sms = _batch(rng)
        _, _, cover, want = _pieces(reqs, hq, hkv, page, causal, sms)
        assert sorted(cover) == [(b, t) for b, (nq, _) in enumerate(reqs) for t in range(nq)]
        _exactly_once(cover, want)


@pytest.mark.parametrize("wrong", ["no keys", "keys twice", "a gap"])
def test_the_check_sees_wrong_items(wrong):
    _, _, cover, want = _pieces([(5, 16001), (1, 9000)], 28, 4, 16)
    cover = {k: list(v) for k, v in cover.items()}
    v = cover[(0, 0)]
    assert len(v) > 2
    v[:] = {"no keys": [(a, a) for a, _ in v], "keys twice": [(0, b) for _, b in v], "a gap": v[:1] + v[2:]}[wrong]
    with pytest.raises(AssertionError):
        _exactly_once(cover, want)


def _limit(share):
    """Items that go to the first free SM end at the mean share and one item's length at the
    latest. The plan tries lengths down to a quarter of the share, each at most 1.5 times the
    next, and takes a shorter one where that gains 3%: 1 + 1.5 / 4 of the share, 3% more, and
    the start of an item (6 us) with a key tile's rounding (1.8 us)."""
    return 1.03 * (1 + 1.5 / 4) * share + 8


def _ends(items, hq, hkv, sms=148):
    """When the last item is done under the plan's costs, and an SM's mean share: items in
    order, each for the first SM that is free."""
    free = [0.0] * sms
    work = 0.0
    for it in items:
        n1, flags, kt0, kt1 = int(it[6]), int(it[7]), int(it[8]), int(it[9])
        cost = (kt1 - kt0) * (STEP_US if n1 else SHARED_US) + START_US
        for _ in range(hkv if flags & PACKED else hq):
            heapq.heappush(free, heapq.heappop(free) + cost)
            work += cost
    return max(free), work / sms


@pytest.mark.parametrize("short", [73, 74, 75, 100, 300, 2000])
@pytest.mark.parametrize("keys", [32768, 131072])
def test_a_long_request_is_cut_among_any_number_of_short_ones(short, keys):
    reqs = [(1, 1000)] * (short // 2) + [(1, keys)] + [(1, 1000)] * (short - short // 2)
    out, items, cover, want = _pieces(reqs, 32, 8, 16)
    _exactly_once(cover, want)
    end, share = _ends(items, 32, 8)
    alone = -(-keys // 128) * SHARED_US  # what it takes uncut
    if alone > 1.1 * share:
        assert out.num_parts > 0
    assert end <= _limit(share), (end, share)


def test_a_long_decode_behind_chunks_is_cut():
    """The chunks' items fill the machine and come first: what follows them adds to their time."""
    reqs = [(2048, 8192)] * 4 + [(1, 131072)] + [(1, 500)] * 10
    out, items, cover, want = _pieces(reqs, 32, 8, 16)
    _exactly_once(cover, want)
    end, share = _ends(items, 32, 8)
    assert out.num_parts > 0 and end <= _limit(share), (end, share)


@pytest.mark.parametrize("reqs,hq,hkv", [([(1, 1000)] * 100, 32, 8), ([(1, 1000)] * 4000, 28, 4), ([(2048, 8192)] * 8, 28, 4),
                                         ([(700, 5000)] * 30, 16, 16), ([(4, 3000 + 10 * i) for i in range(200)], 32, 8)])
def test_even_batches_stay_whole(reqs, hq, hkv):
    out, items, _, _ = _pieces(reqs, hq, hkv, 16)
    end, share = _ends(items, hq, hkv)
    assert out.num_parts == 0 and end <= _limit(share)
