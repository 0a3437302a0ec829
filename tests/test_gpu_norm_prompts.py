"""Norms and appends of prompts with any number of heads: token counts that are no
multiple of four, few heads, batches whose sequences end inside a group of tokens, strided
and in-place rows, bad tokens between good ones."""
import numpy as np
import pytest
import torch

import _norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tables(n, base=1e6):
    inv = 1.0 / (base ** (torch.arange(0, 128, 2).double() / 128))
    t = torch.arange(n).double()[:, None] * inv[None]
    return torch.cos(t).float(), torch.sin(t).float()


def _weight(g, dtype=torch.bfloat16):
    return (1 + 0.3 * torch.randn(128, generator=g)).to(dtype)


def _check(got, x, w, pos, order, n_pos):
    cos, sin = _tables(n_pos)
    pos = pos.cpu().reshape(-1).clamp(0, n_pos - 1).long()
    rows, size = _norm.norm_rope(x.cpu().float().reshape(-1, *x.shape[-2:]).double().numpy(), w.double().numpy(),
                                 cos[pos].double().numpy(), sin[pos].double().numpy(), 1e-6, order)
    err = np.abs(got.cpu().double().reshape(rows.shape).numpy() - rows)
    assert (err <= _norm.bound(rows, size)).all(), (err - _norm.bound(rows, size)).max()


@pytest.mark.parametrize("order", ["rotate_half", "sorted_pair"])
@pytest.mark.parametrize("tokens,hq,hkv", [(2367, 1, 0), (2369, 1, 0), (2402, 1, 1), (5003, 3, 2), (2500, 4, 1), (2375, 7, 1),
                                           (2370, 12, 4), (1601, 16, 4), (799, 40, 8), (2801, 5, 0)])
def test_any_number_of_heads(tokens, hq, hkv, order):
    import atflash
    g = torch.Generator().manual_seed(tokens)
    qkv = (torch.randn((tokens, hq + 2 * hkv, 128), generator=g) * 3).bfloat16().to(DEV)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    qw, kw = _weight(g).to(DEV), _weight(g).to(DEV)
    pos = torch.randint(0, 600, (tokens,), generator=g).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(600))

    def call(a, b, **kws):
        return atflash.qk_norm_rope(q[a:b], k[a:b] if hkv else None, qw, kw if hkv else None, cos, sin,
                                    positions=pos[a:b], out_layout=order, **kws)
    oq, ok = call(0, tokens)
    _check(oq, q, qw.cpu(), pos, order, 600)
    if hkv:
        _check(ok, k, kw.cpu(), pos, order, 600)
    # the rows do not depend on how many tokens a call has
    parts = [call(a, min(a + 97, tokens)) for a in range(0, tokens, 97)]
    assert torch.equal(oq, torch.cat([p[0] for p in parts]))
    assert not hkv or torch.equal(ok, torch.cat([p[1] for p in parts]))
    # over their own inputs, V and the rows around them untouched
    before = qkv.clone()
    call(0, tokens, q_out=q, k_out=k if hkv else None)
    assert torch.equal(q, oq) and (not hkv or torch.equal(k, ok))
    assert torch.equal(qkv[:, hq + hkv:], before[:, hq + hkv:])


@pytest.mark.parametrize("hq,hkv", [(5, 1), (16, 4)])
def test_batches_whose_sequences_end_inside_a_group(hq, hkv):
    import atflash
    g = torch.Generator().manual_seed(hq)
    B, S = 7, 1003
    q, k = ((torch.randn((B, S, h, 128), generator=g) * 3).bfloat16().to(DEV) for h in (hq, hkv))
    w = _weight(g, torch.float32)
    pos = torch.randint(-5, 700, (B, S), generator=g)
    cos, sin = (t.to(DEV) for t in _tables(600))
    for kw, p in ((dict(positions=pos.to(DEV)), pos), (dict(pos_offset=3), (3 + torch.arange(S))[None].expand(B, S))):
        oq, ok = atflash.qk_norm_rope(q, k, w.to(DEV), w.to(DEV), cos, sin, **kw)
        _check(oq, q, w, p, "rotate_half", 600)
        _check(ok, k, w, p, "rotate_half", 600)


@pytest.mark.parametrize("kind", ["NHD", "HND", "level"])
@pytest.mark.parametrize("page,hkv,lens", [(16, 1, [1201, 900, 310]), (16, 3, [2000, 7, 400]), (64, 2, [2371]),
                                           (128, 5, [1500, 871, 1, 2, 3]), (16, 12, [1301]), (32, 8, [1187, 1186])])
def test_append_of_prompts(page, hkv, lens, kind):
    import atflash
    g = torch.Generator().manual_seed(page + hkv)
    npg = [-(-n // page) for n in lens]
    total = sum(npg) + 2
    indices = torch.randperm(total, generator=g).to(torch.int32)[:sum(npg)].to(DEV)
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32, device=DEV)
    bidx = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], dtype=torch.int32)
    pos = torch.tensor([p for n in lens for p in range(n)], dtype=torch.int32)
    bad = torch.zeros(len(pos), dtype=torch.bool)
    bad[5::401] = True  # padding in between
    bidx[bad] = -1
    bidx, pos = bidx.to(DEV), pos.to(DEV)
    qkv = (torch.randn((len(pos), 3 * hkv, 128), generator=g) * 3).bfloat16().to(DEV)
    k, v, w = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:], _weight(g).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(2400))
    vc = torch.randn((total, page, hkv, 128) if kind != "HND" else (total, hkv, page, 128), generator=g).bfloat16().to(DEV)
    kc = torch.randn((total, hkv, 8, page, 16), generator=g).bfloat16().to(DEV) if kind == "level" else vc.clone()
    wk, wv = kc.clone(), vc.clone()
    atflash.append_paged_kv_cache(k, v, bidx, pos, (kc, vc), indices, indptr, kv_layout="HND" if kind == "HND" else "NHD",
                                  rope=(cos, sin), k_norm=(w, 1e-6), out_layout="sorted_pair")
    normed, _ = atflash.qk_norm_rope(k, None, w, None, cos, sin, positions=pos, out_layout="sorted_pair")
    on = ~bad.to(DEV)
    p = pos.long()[on]
    at, slot = indices.long()[indptr.long()[bidx.long()[on]] + p // page], p % page
    if kind == "level":
        wk.permute(0, 3, 1, 2, 4)[at, slot] = normed[on].view(-1, hkv, 8, 16)
    else:
        (wk.transpose(1, 2) if kind == "HND" else wk)[at, slot] = normed[on]
    (wv.transpose(1, 2) if kind == "HND" else wv)[at, slot] = v[on]
    assert torch.equal(kc, wk) and torch.equal(vc, wv)
    assert atflash.check_device_errors() == 2  # the padding is reported
