"""The append into an e4m3 cache of batches that mix single tokens, drafts and prompts,
byte for byte and scale for scale: runs of every length next to one another, many scales
that grow at once, windows in which no run begins, with and without rotation and norm."""
import numpy as np
import pytest
import torch

import _e4m3
from _inputs import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _batch(page, hkv, lens, app, layout, seed, padding=0, grow=False):
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // page) for n in lens]
    total = sum(npg) + 3
    indices = torch.randperm(total, generator=g).to(torch.int32)[:sum(npg)].contiguous()
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32)
    bidx = [b for b, a in enumerate(app) for _ in range(a)] + [-1] * padding
    pos = [p for n, a in zip(lens, app) for p in range(n - a, n)] + [0] * padding
    cache = _e4m3.random_cache(total, page, hkv, layout, g)
    k, v = (torch.randn((len(pos), hkv, 128), generator=g)
            * torch.exp2(torch.randint(-6, 7, (len(pos), hkv, 1), generator=g).float()) for _ in range(2))
    if grow:  # every scale under what the new rows need, by different powers
        for s in (cache[1], cache[3]):
            s.copy_(torch.exp2(torch.randint(-20, -12, s.shape, generator=g).float()))
    return (cache, k.bfloat16(), v.bfloat16(), torch.tensor(bidx, dtype=torch.int32), torch.tensor(pos, dtype=torch.int32),
            indptr, indices)


def _check(cache, k, v, bidx, pos, indptr, indices, layout, want_k=None, **kw):
    import atflash
    want = _e4m3.append(*cache, k if want_k is None else want_k, v, bidx, pos, indptr, indices, layout)
    d = [t.to(DEV) for t in cache]
    atflash.append_paged_kv_cache(k.to(DEV), v.to(DEV), bidx.to(DEV), pos.to(DEV), (d[0], d[2]), indices.to(DEV),
                                  indptr.to(DEV), kv_layout=layout, kv_scales=(d[1], d[3]), **kw)
    for x, y in zip(d, want):
        assert np.array_equal(x.cpu().float().double().numpy(), y, equal_nan=True)
    assert atflash.check_device_errors() == 0


# (page, kv heads, lengths after the append, new tokens)
MIXED = [
    (16, 8, [30] * 20 + [45, 90, 33] + [7] * 13, [1] * 20 + [5, 77, 1] + [1] * 13),
    (64, 4, [100] * 33 + [1000, 65, 130] + [64] * 9, [1] * 33 + [900, 2, 17] + [1] * 9),
    (64, 1, [61, 700, 62, 300, 63, 64], [1, 650, 4, 16, 33, 64]),
    (256, 3, [250] * 10 + [900, 256, 257], [1] * 10 + [600, 129, 66]),
    (128, 8, [50, 128, 129, 700], [1, 65, 1, 33]),
    (20, 5, [19] * 40 + [333], [1] * 40 + [300]),
    (1, 2, [5, 9, 1], [1, 8, 1]),
]


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("page,hkv,lens,app", MIXED)
def test_runs_of_every_length(page, hkv, lens, app, grow, layout):
    _check(*_batch(page, hkv, lens, app, layout, page + hkv, grow=grow), layout)


@pytest.mark.parametrize("order", ["sorted_pair", "rotate_half"])
@pytest.mark.parametrize("shift", [0, 11])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("page,hkv,lens,app", MIXED[:6])
def test_with_rotation_and_norm(page, hkv, lens, app, norm, shift, order):
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _batch(page, hkv, lens, app, "NHD", page + hkv, grow=shift > 0)
    cos, sin = (t.to(DEV) for t in rope_tables(1024, 128, 1e4))
    rp = (pos.long() + shift).to(DEV)
    w = (1 + torch.randn(128, generator=torch.Generator().manual_seed(1)) / 8).bfloat16().to(DEV)
    if norm:
        want_k, _ = atflash.qk_norm_rope(k.to(DEV), None, w, None, cos, sin, positions=rp, out_layout=order)
    else:
        want_k = atflash.rope_pack(k.to(DEV)[None], cos, sin, positions=rp, out_layout=order)[0]
    kw = dict(k_norm=(w, 1e-6)) if norm else {}
    if shift:
        kw["rope_positions"] = rp
    _check(cache, k, v, bidx, pos, indptr, indices, "NHD", want_k=want_k.cpu(), rope=(cos, sin), out_layout=order, **kw)


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 147, 148, 149, 700])
@pytest.mark.parametrize("page", [16, 64])
def test_steps_of_single_tokens_and_padding(batch, page):
    lens = [1 + (7 * b) % (3 * page) for b in range(batch)]
    _check(*_batch(page, 2, lens, [1] * batch, "HND", batch, padding=batch % 5, grow=True), "HND")


def test_a_list_with_more_requests_than_tokens():
    # padded page lists: most requests have no new token
    lens = [40] * 300
    _check(*_batch(16, 4, lens, [40 if b % 100 == 3 else 0 for b in range(300)], "NHD", 3), "NHD")
