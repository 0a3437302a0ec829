"""The norms of q and k heads with their rotation on a B200, against a 64-bit
restatement: shapes, positions, strides, weights, outputs over their inputs, odd
values; and the appends' norm of K, bit for bit with the norm followed by an append."""
import numpy as np
import pytest
import torch

import _e4m3
import _norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tables(n, base=1e6):
    inv = 1.0 / (base ** (torch.arange(0, 128, 2).double() / 128))
    t = torch.arange(n).double()[:, None] * inv[None]
    return torch.cos(t).float(), torch.sin(t).float()


def _rows(shape, g):
    f = torch.exp2(torch.randint(-12, 13, (*shape[:-1], 1), generator=g).float())
    return (torch.randn(shape, generator=g) * f).bfloat16()


def _weight(g, dtype):
    return (1 + 0.3 * torch.randn(128, generator=g)).to(dtype)


def _check(got, x, w, pos, eps, order, n_pos=512):
    cos, sin = _tables(n_pos)
    pos = pos.reshape(-1).clamp(0, n_pos - 1).long()
    rows, size = _norm.norm_rope(x.float().reshape(-1, *x.shape[-2:]).double().numpy(), w.double().numpy(),
                                 cos[pos].double().numpy(), sin[pos].double().numpy(), eps, order)
    err = np.abs(got.cpu().double().reshape(rows.shape).numpy() - rows)
    assert (err <= _norm.bound(rows, size)).all(), (err - _norm.bound(rows, size)).max()


@pytest.mark.parametrize("order", ["rotate_half", "sorted_pair"])
@pytest.mark.parametrize("tokens,hq,hkv", [(1, 1, 1), (1, 28, 4), (3, 5, 1), (64, 24, 8), (777, 7, 3), (1500, 32, 8)])
def test_packed_tokens(tokens, hq, hkv, order):
    import atflash
    g = torch.Generator().manual_seed(tokens + hq)
    dt = torch.float32 if hq % 2 else torch.bfloat16
    q, k, qw, kw = _rows((tokens, hq, 128), g), _rows((tokens, hkv, 128), g), _weight(g, dt), _weight(g, dt)
    pos = torch.randint(0, 512, (tokens,), generator=g)
    cos, sin = (t.to(DEV) for t in _tables(512))
    for p in (pos.to(torch.int32), pos):
        oq, ok = atflash.qk_norm_rope(q.to(DEV), k.to(DEV), qw.to(DEV), kw.to(DEV), cos, sin, eps=1e-5,
                                      positions=p.to(DEV), out_layout=order)
        _check(oq, q, qw, pos, 1e-5, order)
        _check(ok, k, kw, pos, 1e-5, order)


@pytest.mark.parametrize("how", ["offset", "shared", "each"])
def test_batched_positions_and_clamping(how):
    import atflash
    g = torch.Generator().manual_seed(5)
    B, S = 3, 41
    q, k, w = _rows((B, S, 6, 128), g), _rows((B, S, 2, 128), g), _weight(g, torch.bfloat16)
    cos, sin = (t.to(DEV) for t in _tables(512))
    kw = {}
    if how == "offset":
        pos = (torch.arange(S) + 490)[None].expand(B, S)  # the last ones pass the tables' end
        kw["pos_offset"] = 490
    elif how == "shared":
        pos = torch.randint(-5, 600, (S,), generator=g)
        kw["positions"] = pos.to(DEV)
        pos = pos[None].expand(B, S)
    else:
        pos = torch.randint(-5, 600, (B, S), generator=g)
        wide = torch.full((B, 2 * S), -1, dtype=torch.int32)
        wide[:, ::2] = pos.to(torch.int32)
        kw["positions"] = wide.to(DEV)[:, ::2]  # any strides
    oq, ok = atflash.qk_norm_rope(q.to(DEV), k.to(DEV), w.to(DEV), w.to(DEV), cos, sin, **kw)
    _check(oq, q, w, pos, 1e-6, "rotate_half")
    _check(ok, k, w, pos, 1e-6, "rotate_half")


@pytest.mark.parametrize("order", ["rotate_half", "sorted_pair"])
@pytest.mark.parametrize("tokens", [2, 700])
def test_slices_of_one_projection_and_in_place(tokens, order):
    import atflash
    g = torch.Generator().manual_seed(tokens)
    hq, hkv = 6, 2
    qkv, w = _rows((tokens, hq + 2 * hkv, 128), g), _weight(g, torch.float32)
    pos = torch.randint(0, 512, (tokens,), generator=g)
    cos, sin = (t.to(DEV) for t in _tables(512))
    d = qkv.to(DEV)
    q, k = d[:, :hq], d[:, hq:hq + hkv]
    args = (w.to(DEV), w.to(DEV), cos, sin)
    want = atflash.qk_norm_rope(q, k, *args, positions=pos.to(DEV), out_layout=order)
    _check(want[0], qkv[:, :hq], w, pos, 1e-6, order)
    assert torch.equal(d.cpu(), qkv)
    got = atflash.qk_norm_rope(q, k, *args, positions=pos.to(DEV), out_layout=order, q_out=q, k_out=k)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(d[:, hq + hkv:].cpu(), qkv[:, hq + hkv:])  # v stays


def test_queries_alone_no_tokens_and_one_table_row():
    import atflash
    g = torch.Generator().manual_seed(3)
    q, w = _rows((9, 4, 128), g), _weight(g, torch.bfloat16)
    cos, sin = (t.to(DEV) for t in _tables(512))
    oq, ok = atflash.qk_norm_rope(q.to(DEV), None, w.to(DEV), None, cos, sin, pos_offset=7)
    assert ok is None
    _check(oq, q, w, torch.arange(9) + 7, 1e-6, "rotate_half")
    oq, ok = atflash.qk_norm_rope(q.to(DEV)[:0], q.to(DEV)[:0], w.to(DEV), w.to(DEV), cos, sin)
    assert oq.shape == ok.shape == (0, 4, 128)
    oq, _ = atflash.qk_norm_rope(q.to(DEV), None, w.to(DEV), None, cos[:1], sin[:1])
    _check(oq, q, w, torch.zeros(9, dtype=torch.long), 1e-6, "rotate_half", n_pos=1)


def test_zero_rows_and_rows_with_infinity_or_nan_keep_to_themselves():
    import atflash
    g = torch.Generator().manual_seed(4)
    q, w = _rows((40, 4, 128), g), _weight(g, torch.float32)
    q[3, 1] = 0
    bad = q.clone()
    bad[5, 2, 17], bad[6, 0, 3] = float("nan"), float("inf")
    cos, sin = (t.to(DEV) for t in _tables(512))
    a, _ = atflash.qk_norm_rope(q.to(DEV), None, w.to(DEV), None, cos, sin)
    b, _ = atflash.qk_norm_rope(bad.to(DEV), None, w.to(DEV), None, cos, sin)
    assert (a[3, 1] == 0).all() and a.isfinite().all()
    assert b[5, 2].isnan().all() and b[6, 0].isnan().any()
    keep = torch.ones(40, 4, dtype=torch.bool)
    keep[5, 2] = keep[6, 0] = False
    assert torch.equal(a.cpu()[keep], b.cpu()[keep])


def test_another_stream_and_a_replayed_graph():
    import atflash
    g = torch.Generator().manual_seed(8)
    q, k, w = _rows((33, 8, 128), g).to(DEV), _rows((33, 2, 128), g).to(DEV), _weight(g, torch.bfloat16).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(512))
    pos = torch.randint(0, 512, (33,), generator=g).to(DEV)
    want = atflash.qk_norm_rope(q, k, w, w, cos, sin, positions=pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = atflash.qk_norm_rope(q, k, w, w, cos, sin, positions=pos)
        oq, ok = torch.empty_like(q), torch.empty_like(k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            atflash.qk_norm_rope(q, k, w, w, cos, sin, positions=pos, q_out=oq, k_out=ok)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pos.copy_(pos.flip(0))
    graph.replay()
    want = atflash.qk_norm_rope(q, k, w, w, cos, sin, positions=pos)
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])


def test_no_gradient():
    import atflash
    q, w = torch.zeros((2, 1, 128), dtype=torch.bfloat16, device=DEV), torch.ones(128, device=DEV, requires_grad=True)
    cos, sin = (t.to(DEV) for t in _tables(4))
    with pytest.raises(RuntimeError, match="backward"):
        atflash.qk_norm_rope(q, None, w, None, cos, sin)
    with torch.no_grad():
        atflash.qk_norm_rope(q, None, w, None, cos, sin)


def test_refusals():
    import atflash
    q = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device=DEV)
    w = torch.ones(128, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(8))
    ok = dict(q=q, k=q.clone(), q_weight=w, k_weight=w, cos=cos, sin=sin)
    for bad in (dict(k=None), dict(k_weight=w.bfloat16()), dict(q_weight=w[:64]), dict(q_weight=w.half()), dict(eps=0.0),
                dict(eps=float("nan")), dict(eps=1e-60), dict(out_layout="pairs"), dict(q=q.float()), dict(q=q[..., :64]),
                dict(k=q[:3]), dict(k=q[None]), dict(cos=cos.half()), dict(cos=cos[:4]), dict(cos=cos[:, :32], sin=sin[:, :32]),
                dict(positions=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(positions=torch.zeros(4, device=DEV)), dict(positions=torch.zeros(4, dtype=torch.int32)),
                dict(q_out=torch.empty((4, 2, 128), device=DEV)), dict(q_out=q.transpose(0, 1)[:, :, :]),
                dict(q_out=torch.empty((1, 2, 128), dtype=torch.bfloat16, device=DEV).expand(4, 2, 128))):
        with pytest.raises(ValueError):
            atflash.qk_norm_rope(**{**ok, **bad})
    shifted = torch.zeros(4 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, 2, 128)
    with pytest.raises(atflash.AtfError, match="aligned"):
        atflash.qk_norm_rope(**{**ok, "q": shifted})
    atflash.qk_norm_rope(**ok)


# ------------------------------------------------------------------ appends

def _step(page, lens, app, g):
    npg = [-(-n // page) for n in lens]
    total = sum(npg) + 3
    indices = torch.randperm(total, generator=g).to(torch.int32)[:sum(npg)].contiguous()
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32)
    bidx = torch.tensor([b for b, a in enumerate(app) for _ in range(a)], dtype=torch.int32)
    pos = torch.tensor([p for n, a in zip(lens, app) for p in range(n - a, n)], dtype=torch.int32)
    return total, indptr, indices, bidx, pos


CASES = [(16, 8, [1], [1]), (16, 3, [37, 80, 5, 16], [1, 1, 1, 1]), (64, 2, [200, 64, 129], [130, 64, 1]),
         (32, 1, [300, 17], [300, 17]), (256, 2, [600, 255], [511, 254])]


@pytest.mark.parametrize("order", ["sorted_pair", "rotate_half"])
@pytest.mark.parametrize("kind", ["NHD", "HND", "level"])
@pytest.mark.parametrize("page,hkv,lens,app", CASES)
def test_append_norms_k_like_the_norm_itself(page, hkv, lens, app, kind, order):
    import atflash
    if kind == "level" and order != "sorted_pair":
        return
    g = torch.Generator().manual_seed(page + hkv)
    total, indptr, indices, bidx, pos = _step(page, lens, app, g)
    qkv = _rows((len(pos), 3 * hkv, 128), g).to(DEV)
    k, v, w = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:], _weight(g, torch.float32 if hkv == 2 else torch.bfloat16).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(700))
    shape = (total, page, hkv, 128) if kind != "HND" else (total, hkv, page, 128)
    vc = torch.randn(shape, generator=g).bfloat16().to(DEV)
    kc = torch.randn((total, hkv, 8, page, 16), generator=g).bfloat16().to(DEV) if kind == "level" else vc.clone()
    wk, wv = kc.clone(), vc.clone()
    idx = [t.to(DEV) for t in (bidx, pos, indptr, indices)]
    atflash.append_paged_kv_cache(k, v, idx[0], idx[1], (kc, vc), idx[3], idx[2], kv_layout="HND" if kind == "HND" else "NHD",
                                  rope=(cos, sin), k_norm=(w, 1e-5), out_layout=order)
    normed, _ = atflash.qk_norm_rope(k, None, w, None, cos, sin, eps=1e-5, positions=idx[1], out_layout=order)
    _check(normed, k.cpu(), w.cpu(), pos, 1e-5, order, n_pos=700)
    slot = pos.long() % page
    at = indices.long()[indptr.long()[bidx.long()] + pos.long() // page]
    if kind == "level":
        wk.permute(0, 3, 1, 2, 4)[at.to(DEV), slot.to(DEV)] = normed.view(-1, hkv, 8, 16)
    else:
        (wk.transpose(1, 2) if kind == "HND" else wk)[at.to(DEV), slot.to(DEV)] = normed
    (wv.transpose(1, 2) if kind == "HND" else wv)[at.to(DEV), slot.to(DEV)] = v
    assert torch.equal(kc, wk) and torch.equal(vc, wv)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("order", ["sorted_pair", "rotate_half"])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page,hkv,lens,app", CASES)
def test_e4m3_append_norms_k_like_the_norm_itself(page, hkv, lens, app, layout, order):
    import atflash
    g = torch.Generator().manual_seed(page + hkv)
    total, indptr, indices, bidx, pos = _step(page, lens, app, g)
    k, v, w = _rows((len(pos), hkv, 128), g), _rows((len(pos), hkv, 128), g), _weight(g, torch.bfloat16)
    cos, sin = (t.to(DEV) for t in _tables(700))
    cache = _e4m3.random_cache(total, page, hkv, layout, g)
    normed, _ = atflash.qk_norm_rope(k.to(DEV), None, w.to(DEV), None, cos, sin, positions=pos.to(DEV), out_layout=order)
    want = _e4m3.append(*cache, normed.cpu(), v, bidx, pos, indptr, indices, layout)
    d = [t.to(DEV) for t in cache]
    atflash.append_paged_kv_cache(k.to(DEV), v.to(DEV), bidx.to(DEV), pos.to(DEV), (d[0], d[2]), indices.to(DEV),
                                  indptr.to(DEV), kv_layout=layout, kv_scales=(d[1], d[3]), rope=(cos, sin),
                                  k_norm=(w.to(DEV), 1e-6), out_layout=order)
    for x, y in zip(d, want):
        assert np.array_equal(x.cpu().float().double().numpy(), y, equal_nan=True)
    assert atflash.check_device_errors() == 0


def test_append_norm_positions_padding_and_refusals():
    import atflash
    g = torch.Generator().manual_seed(1)
    k, w = _rows((3, 2, 128), g).to(DEV), _weight(g, torch.bfloat16).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(64))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache = torch.zeros((2, 16, 2, 128), dtype=torch.bfloat16, device=DEV)
    args = (k, k, i32(0, 7, 0), i32(0, 0, 17), (cache, cache.clone()), i32(1, 0), i32(0, 2))
    # token 1's request does not exist: left out and reported; angles from rope_positions
    rp = torch.tensor([5, 6, 900], device=DEV)
    atflash.append_paged_kv_cache(*args, rope=(cos, sin), rope_positions=rp, k_norm=(w, 1e-6))
    assert atflash.check_device_errors() == 2
    want, _ = atflash.qk_norm_rope(k, None, w, None, cos, sin, positions=rp, out_layout="sorted_pair")
    assert torch.equal(cache[1, 0], want[0]) and torch.equal(cache[0, 1], want[2])
    assert cache[1, 1:].abs().sum() == 0 and cache[0, 0].abs().sum() == 0
    for bad in (dict(k_norm=w), dict(k_norm=(w, 0.0)), dict(k_norm=(w[:64], 1e-6)), dict(k_norm=(w.half(), 1e-6)),
                dict(k_norm=(w.cpu(), 1e-6)), dict(k_norm=(w, 1e-6), rope=None)):
        with pytest.raises(ValueError):
            atflash.append_paged_kv_cache(*args, **{"rope": (cos, sin), **bad})
    with pytest.raises(RuntimeError, match="backward"):
        atflash.append_paged_kv_cache(*args, rope=(cos, sin), k_norm=(w.float().requires_grad_(), 1e-6))
    odd = torch.zeros(129, dtype=torch.bfloat16, device=DEV)[1:]
    with pytest.raises(atflash.AtfError, match="aligned"):
        atflash.append_paged_kv_cache(*args, rope=(cos, sin), k_norm=(odd, 1e-6))
