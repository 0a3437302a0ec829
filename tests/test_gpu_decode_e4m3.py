"""Decode over an e4m3 cache on a B200 against a 64-bit restatement: groups, page
sizes, layouts, lengths from 1, windows at their level boundaries, scales far
apart, special values past the ends, strides, streams, refusals.

Tolerances: the scores' products and sums are exact up to fp32 sums (128 terms,
relative 2^-17 of sum |q k|); P has 11 bits (relative 2^-12 each, independent), so
that out in fp32 is off by at most 2^-11 of sum p |v| plus 2^-20 of itself. The
bf16 output is the fp32 one, rounded. lse is off by the scores' error."""
import math

import numpy as np
import pytest
import torch

import _e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Z16 = [1 << 28, 777, 300, 150, 64, 33, 17, 0]


def _setup(lens, page, hkv, group, layout, seed, spread=2, qfac=1.0):
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // page) for n in lens]
    total = sum(npg) + 3
    indices = torch.randperm(total, generator=g).to(torch.int32)[:sum(npg)].contiguous()
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32)
    last = torch.tensor([(n - 1) % page + 1 if n else 0 for n in lens], dtype=torch.int32)
    q = (torch.randn((len(lens), hkv * group, 128), generator=g) * qfac).bfloat16()
    return _e4m3.random_cache(total, page, hkv, layout, g, spread), q, indptr, indices, last


def _exact(cache, q, indptr, indices, lens, layout, zhi=None, q_pos=None, pos0=None, scale=None):
    """(out, sum p |v|, lse, score error bound) in 64 bits."""
    k, ks, v, vs = (t.double().numpy() if t.dtype == torch.float32 else t.float().double().numpy() for t in cache)
    if layout == "HND":
        k, v = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
    B, hq, _ = q.shape
    hkv = k.shape[2]
    scale = 1 / math.sqrt(128) if scale is None else scale
    out, mag, lse, err = (np.zeros((B, hq, 128)), np.zeros((B, hq, 128)), np.full((B, hq), -np.inf), np.zeros((B, hq)))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = indices[int(indptr[b]):int(indptr[b + 1])].long().numpy()
        kb = (k[ids] * ks[ids][:, None, :, None]).reshape(-1, hkv, 128)[:n].copy()
        vb = (v[ids] * vs[ids][:, None, :, None]).reshape(-1, hkv, 128)[:n]
        if zhi is not None:
            z = (n - 1 if q_pos is None else q_pos[b]) - (0 if pos0 is None else pos0[b]) - np.arange(n)
            for i in range(1, 8):
                kb[z > zhi[i], :, 16 * i:16 * i + 16] = 0
        for h in range(hq):
            qq = q[b, h].double().numpy()
            kh, vh = kb[:, h * hkv // hq], vb[:, h * hkv // hq]
            s = kh @ qq * scale
            err[b, h] = (np.abs(kh) @ np.abs(qq) * scale).max() * 2.0 ** -17
            m = s.max()
            p = np.exp(s - m)
            lse[b, h] = m + np.log(p.sum())
            p /= p.sum()
            out[b, h], mag[b, h] = p @ vh, p @ np.abs(vh)
    return out, mag, lse, err


def _run(cache, q, indptr, indices, last, page, hkv, layout, run_kw=None, cache_arg=None, **plan_kw):
    import atflash
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(ws, layout)
    w.plan(indptr, indices, last, q.shape[1], hkv, 128, page, kv_data_type=torch.float8_e4m3fn, **plan_kw)
    d = [t.to(DEV) for t in cache] if cache_arg is None else cache_arg

    def run(dtype):
        return w.run(q.to(DEV), (d[0], d[2]), kv_scales=(d[1], d[3]), return_lse=True, out_dtype=dtype, **(run_kw or {}))
    out, lse = run(torch.float32)
    rounded, again = run(torch.bfloat16)
    nan = torch.isnan(out)
    assert torch.equal(rounded[~nan], out.bfloat16()[~nan]) and torch.equal(lse.isnan(), again.isnan())
    assert torch.isnan(rounded[nan]).all() and torch.equal(lse.nan_to_num(), again.nan_to_num())
    return out, lse


def _close(got, want, rounding=2.0 ** -20):
    out, lse = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    ref, mag, rl, err = want
    tol = (2.0 ** -11 + 2 * err[..., None]) * mag + rounding * np.abs(ref) + 1e-30
    assert np.all(np.abs(out - ref) <= tol), np.max(np.abs(out - ref) / tol)
    dead = np.isneginf(rl)
    assert np.array_equal(np.isneginf(lse), dead)
    assert np.all(np.abs(lse - rl)[~dead] <= (err + 2.0 ** -20 * (1 + np.abs(rl)))[~dead])


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page,hkv,group,lens", [
    (16, 8, 3, [1, 17, 300]),
    (16, 1, 1, [1]),
    (32, 2, 8, [31, 0, 1000, 64, 65]),
    (64, 4, 7, [63, 64, 129, 500]),
    (128, 2, 2, [127, 128, 385, 1025]),
    (256, 1, 4, [255, 700, 256]),
    (16, 2, 9, [40, 111]),                 # more than 8 heads: two tiles of heads
    (64, 1, 16, [1, 300, 2049]),
    (16, 3, 5, [127, 128, 129, 15, 16]),
])
def test_decode_e4m3_matches_the_definition(layout, page, hkv, group, lens):
    import atflash
    cache, q, indptr, indices, last = _setup(lens, page, hkv, group, layout, page + group)
    want = _exact(cache, q, indptr, indices, lens, layout)
    _close(_run(cache, q, indptr, indices, last, page, hkv, layout), want)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("page,hkv,group", [(16, 2, 3), (64, 1, 7), (256, 2, 12)])
@pytest.mark.parametrize("chunk", [0, 64, 320])
def test_decode_e4m3_window_and_splits(page, hkv, group, chunk):
    """Levels that end inside 16-key groups, slices and stages; many splits."""
    lens = [1500, 18, 850, 1]
    cache, q, indptr, indices, last = _setup(lens, page, hkv, group, "NHD", 7 + group)
    want = _exact(cache, q, indptr, indices, lens, "NHD", zhi=Z16)
    _close(_run(cache, q, indptr, indices, last, page, hkv, "NHD", window_table=Z16, max_chunk_keys=chunk), want)


@pytest.mark.parametrize("hkv,group", [(8, 1), (2, 8), (1, 11)])
def test_decode_e4m3_many_short_requests(hkv, group):
    """More rows than the split merge's blocks fill at once, empty requests among them."""
    g = np.random.default_rng(hkv)
    lens = [int(x) for x in g.integers(0, 90, 180)] + [0, 1500]
    cache, q, indptr, indices, last = _setup(lens, 16, hkv, group, "NHD", 5)
    _close(_run(cache, q, indptr, indices, last, 16, hkv, "NHD"), _exact(cache, q, indptr, indices, lens, "NHD"))


def test_decode_e4m3_positions_and_layouts():
    """Explicit positions move the window; without one the pair order is free."""
    lens = [600, 33]
    cache, q, indptr, indices, last = _setup(lens, 16, 2, 4, "NHD", 3)
    qp, p0 = [900, 40], [250, 3]
    want = _exact(cache, q, indptr, indices, lens, "NHD", zhi=Z16, q_pos=qp, pos0=p0)
    t = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
    _close(_run(cache, q, indptr, indices, last, 16, 2, "NHD", dict(q_pos=t(qp), kv_pos0=t(p0)), window_table=Z16), want)
    want = _exact(cache, q, indptr, indices, lens, "NHD", scale=0.3)
    _close(_run(cache, q, indptr, indices, last, 16, 2, "NHD", qk_layout="rotate_half", sm_scale=0.3), want)


@pytest.mark.parametrize("qfac", [2.0 ** -60, 1.0, 2.0 ** 40])
def test_decode_e4m3_scales_far_apart(qfac):
    """Pages whose scales differ by 2^60, an all-zero page with the least scale, a
    scale of zero, scales that are no powers of two; queries of any magnitude."""
    lens = [260, 70]
    cache, q, indptr, indices, last = _setup(lens, 16, 2, 3, "NHD", 21, qfac=qfac)
    g = torch.Generator().manual_seed(4)
    k, ks, v, vs = cache
    vs *= torch.exp2(torch.randint(-30, 31, vs.shape, generator=g).float()) * 1.37
    ks *= 1.21 * (0.02 / qfac)
    v[int(indices[2])] = 0
    vs[int(indices[2])] = 2.0 ** -126
    vs[int(indices[3]), 0] = 0
    ks[int(indices[4])] = 0
    want = _exact(cache, q, indptr, indices, lens, "NHD")
    _close(_run(cache, q, indptr, indices, last, 16, 2, "NHD"), want, rounding=2.0 ** -18)


def test_decode_e4m3_all_values_zero():
    lens = [50]
    cache, q, indptr, indices, last = _setup(lens, 16, 1, 2, "NHD", 22)
    cache[2].zero_()
    cache[3].zero_()
    out, lse = _run(cache, q, indptr, indices, last, 16, 1, "NHD")
    want = _exact(cache, q, indptr, indices, lens, "NHD")
    assert torch.count_nonzero(out) == 0
    _close((out, lse), want)


@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_e4m3_rows_past_the_end_are_not_read(page):
    """NaN in every slot past a request's last token, and in pages of nobody."""
    lens = [page + 1, 3, page - 1, 2 * page + 20]
    cache, q, indptr, indices, last = _setup(lens, page, 2, 3, "NHD", 23)
    want = _exact(cache, q, indptr, indices, lens, "NHD")
    mine = torch.zeros(cache[0].shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            mine[int(indices[int(indptr[b]) + j // page]), j % page] = True
    for t in (cache[0], cache[2]):
        t.view(torch.uint8)[~mine] = 0x7f
    _close(_run(cache, q, indptr, indices, last, page, 2, "NHD"), want)
    # a NaN of the request's own reaches its heads and no other
    cache[2].view(torch.uint8)[int(indices[0]), 0, 0, 5] = 0x7f
    out, _ = _run(cache, q, indptr, indices, last, page, 2, "NHD")
    assert torch.isnan(out[0, :3, 5]).all() and int(torch.isnan(out).sum()) == 3


def test_decode_e4m3_strides_stream_pdl_and_graph():
    import atflash
    lens = [300, 90, 411]
    cache, q, indptr, indices, last = _setup(lens, 16, 2, 4, "NHD", 24)
    want = _exact(cache, q, indptr, indices, lens, "NHD")
    base = _run(cache, q, indptr, indices, last, 16, 2, "NHD")
    _close(base, want)
    base = (base[0].bfloat16(), base[1])
    # K and V as halves of one tensor with room after each row; scales as columns
    P = cache[0].shape[0]
    wide = torch.zeros((P, 2, 16, 3, 160), dtype=torch.uint8, device=DEV)
    sc = torch.zeros((P, 3, 2), device=DEV)
    for i in (0, 1):
        wide[:, i, :, :2, :128] = cache[2 * i].view(torch.uint8).to(DEV)
        sc[:, :2, i] = cache[2 * i + 1].to(DEV)
    f8 = wide.view(torch.float8_e4m3fn)
    arg = [f8[:, 0, :, :2, :128], sc[:, :2, 0], f8[:, 1, :, :2, :128], sc[:, :2, 1]]
    qw = torch.zeros((3, 11, 136), dtype=torch.bfloat16, device=DEV)
    qw[:, 2:10, :128] = q.to(DEV)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(ws, "NHD", use_cuda_graph=True)
    w.plan(indptr, indices, last, 8, 2, 128, 16, kv_data_type=torch.float8_e4m3fn)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = torch.empty((3, 8, 128), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((3, 8), device=DEV)

    def run(**kw):
        return w.run(qw[:, 2:10, :128], (arg[0], arg[2]), kv_scales=(arg[1], arg[3]), out=out, lse=lse, return_lse=True,
                     **kw)
    with torch.cuda.stream(st):
        run()
    st.synchronize()
    assert torch.equal(out, base[0]) and torch.equal(lse, base[1])
    for _ in range(3):
        out.zero_()
        run(enable_pdl=True)
        torch.cuda.synchronize()
        assert torch.equal(out, base[0]) and torch.equal(lse, base[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, base[0]) and torch.equal(lse, base[1])
    assert atflash.check_device_errors() == 0


def test_decode_e4m3_cache_past_four_gigabytes():
    """Pages whose byte offsets pass 32 bits."""
    page, hkv = 256, 8
    P = (1 << 32) // (page * hkv * 128) + 40
    lens = [600]
    small, q, _, _, last = _setup(lens, page, hkv, 2, "NHD", 25)
    ids = torch.tensor([P - 1, P - 30, 1], dtype=torch.int32)
    d = []
    for i in (0, 2):
        t = torch.zeros((P, page, hkv, 128), dtype=torch.uint8, device=DEV)
        t[ids.long()] = small[i].view(torch.uint8)[:3].to(DEV)
        s = torch.ones((P, hkv), device=DEV)
        s[ids.long()] = small[i + 1][:3].to(DEV)
        d += [t.view(torch.float8_e4m3fn), s]
    indptr = torch.tensor([0, 3], dtype=torch.int32)
    want = _exact(small, q, indptr, torch.tensor([0, 1, 2], dtype=torch.int32), lens, "NHD")
    _close(_run(None, q, indptr, ids, last, page, hkv, "NHD", cache_arg=d), want)


def test_decode_e4m3_after_append_equals_the_written_values():
    """One serving step: tables from lengths, the append, the decode over them."""
    import atflash
    page, hkv, group, lens = 16, 2, 3, [70, 16, 200]
    g = torch.Generator().manual_seed(30)
    n_tok = sum(lens)
    k, v = (torch.randn((n_tok, hkv, 128), generator=g).bfloat16() for _ in range(2))
    q = torch.randn((3, hkv * group, 128), generator=g).bfloat16()
    cache = _e4m3.random_cache(40, page, hkv, "NHD", g)
    d = [t.to(DEV) for t in cache]
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    table = torch.full((3, 16), -1, dtype=torch.int32, device=DEV)
    npg = sum(-(-n // page) for n in lens)
    t = atflash.build_page_tables(ld, ld, table, page, num_tokens=n_tok, max_pages=npg,
                                  free_pages=torch.randperm(40, generator=g).to(torch.int32).to(DEV),
                                  free_head=torch.zeros(1, dtype=torch.int32, device=DEV))
    atflash.append_paged_kv_cache(k.to(DEV), v.to(DEV), t.batch_indices, t.positions, (d[0], d[2]), t.indices, t.indptr,
                                  kv_scales=(d[1], d[3]))
    got = _run(None, q, t.indptr, t.indices, t.last_page_len, page, hkv, "NHD", cache_arg=d)
    host = [x.cpu() for x in d]
    _close(got, _exact(host, q, t.indptr.cpu(), t.indices.cpu(), lens, "NHD"))
    # and the stored values are within half a step of e4m3 of what was appended
    val = host[0].float() * host[1][:, None, :, None]
    at = 0
    for b, n in enumerate(lens):
        ids = t.indices[int(t.indptr[b]):int(t.indptr[b + 1])].long().cpu()
        rows, s = val[ids].reshape(-1, hkv, 128)[:n], host[1][ids].repeat_interleave(page, 0)[:n, :, None]
        x = k[at:at + n].float()
        assert torch.all((rows - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10))
        at += n
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("window", [None, Z16])
def test_decode_e4m3_with_either_plan(window):
    """A plan of one item per CTA, and one of units that run through many requests."""
    lens = [1, 0, 90, 64, 5, 700, 33, 128, 2, 2, 2, 1300, 65] * 9
    cache, q, indptr, indices, last = _setup(lens, 32, 8, 2, "HND", 26)
    want = _exact(cache, q, indptr, indices, lens, "HND", zhi=window)
    import atflash
    d = [t.to(DEV) for t in cache]
    for dtype in ("bfloat16", torch.float8_e4m3fn):
        w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV), "HND")
        w.plan(indptr, indices, last, 16, 8, 128, 32, kv_data_type=dtype, window_table=window)
        _close(w.run(q.to(DEV), (d[0], d[2]), kv_scales=(d[1], d[3]), return_lse=True, out_dtype=torch.float32), want)
    # and the plan of units with a bf16 cache
    bf = [(d[i].float() * d[i + 1][:, :, None, None]).bfloat16() for i in (0, 2)]
    a = w.run(q.to(DEV), tuple(bf), out_dtype=torch.float32)
    w.plan(indptr, indices, last, 16, 8, 128, 32, window_table=window)
    b = w.run(q.to(DEV), tuple(bf), out_dtype=torch.float32)
    assert torch.all((a - b).abs() <= 2.0 ** -8 * torch.from_numpy(want[1]).to(DEV) + 1e-30)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("page,layout", [(16, "NHD"), (64, "HND")])
@pytest.mark.parametrize("window", [None, Z16])
def test_decode_e4m3_long_units(page, layout, window):
    """Units of over a hundred stages, so that the ring turns many times, and the same
    answer from every run."""
    lens = [9000, 13011, 77, 4032]
    cache, q, indptr, indices, last = _setup(lens, page, 2, 2, layout, 27)
    want = _exact(cache, q, indptr, indices, lens, layout, zhi=window)
    first = _run(cache, q, indptr, indices, last, page, 2, layout, window_table=window, min_chunk_keys=8192)
    _close(first, want)
    for _ in range(5):
        got = _run(cache, q, indptr, indices, last, page, 2, layout, window_table=window, min_chunk_keys=8192)
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])


def test_decode_e4m3_bad_pages_are_reported():
    import atflash
    cache, q, indptr, indices, last = _setup([100, 40], 16, 2, 3, "NHD", 31)
    for bad in (cache[0].shape[0], -1, 2 ** 31 - 1):
        ix = indices.clone()
        ix[3] = bad
        _run(cache, q, indptr, ix, last, 16, 2, "NHD")
        assert atflash.check_device_errors() == 2


def test_decode_e4m3_refusals():
    import atflash
    cache, q, indptr, indices, last = _setup([100, 40], 16, 2, 3, "NHD", 32)
    d = [t.to(DEV) for t in cache]
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)

    def call(q=q.to(DEV), kv=(d[0], d[2]), scales=(d[1], d[3]), page=16, plan={}, **kw):
        w = atflash.BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
        w.plan(torch.tensor([0, 1]), indices[:1], torch.tensor([page]) if page < 16 else last[:1], 6, 2, 128, page, **plan)
        return w.run(q[:1], kv, kv_scales=scales, **kw)
    call()
    bf = torch.zeros_like(d[0], dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        call(scales=None)
    with pytest.raises(TypeError):
        call(q=q.to(DEV).half())
    for kw in (dict(kv=(bf, bf)), dict(scales=(d[1], d[3][:-1])), dict(scales=(d[1].double(), d[3].double())),
               dict(scales=(d[1].cpu(), d[3].cpu())), dict(kv=(d[0], d[2][:-1])), dict(scales=d[1]),
               dict(kv=(d[0][..., :64], d[2][..., :64]))):
        with pytest.raises(ValueError):
            call(**kw)
    z8 = [1 << 20] * 16
    small = torch.zeros((4, 8, 2, 128), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    for kw in (dict(plan=dict(window_table=z8, window_mode="vec8")), dict(k_scale=1.0), dict(exchange=object()),
               dict(plan=dict(window_table=Z16, qk_layout="rotate_half")),
               dict(page=8, kv=(small, small), scales=(torch.ones(4, 2, device=DEV),) * 2)):
        with pytest.raises(NotImplementedError):
            call(**kw)
    odd = torch.zeros((30, 16, 2, 136), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[..., :128]
    with pytest.raises(atflash.AtfError):
        call(kv=(odd, odd), scales=(torch.ones(30, 2, device=DEV),) * 2)
    assert atflash.check_device_errors() == 0
