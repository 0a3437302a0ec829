"""The append into an e4m3 cache on a B200, byte for byte and scale for scale
against a 64-bit restatement (the arithmetic has one result: power-of-two scales,
one rounding): layouts, page sizes, ragged runs, scales that grow, RoPE at write,
strides, special values, refusals."""
import numpy as np
import pytest
import torch

import _e4m3
from _inputs import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _setup(layout, page, hkv, lens, app, seed, factor=8):
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // page) for n in lens]
    total = sum(npg) + 4
    indices = torch.randperm(total, generator=g).to(torch.int32)[:sum(npg)].contiguous()
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32)
    bidx = torch.tensor([b for b, a in enumerate(app) for _ in range(a)], dtype=torch.int32)
    pos = torch.tensor([p for n, a in zip(lens, app) for p in range(n - a, n)], dtype=torch.int32)
    nnz = len(pos)
    k, v = (torch.randn((nnz, hkv, 128), generator=g)
            * torch.exp2(torch.randint(-factor, factor + 1, (nnz, hkv, 1), generator=g).float()) for _ in range(2))
    return _e4m3.random_cache(total, page, hkv, layout, g), k.bfloat16(), v.bfloat16(), bidx, pos, indptr, indices


def _check(cache, want):
    for x, y in zip(cache, want):
        assert np.array_equal(x.cpu().float().double().numpy(), y, equal_nan=True)


def _append(cache, k, v, bidx, pos, indptr, indices, layout, **kw):
    import atflash
    d = [t.to(DEV) for t in cache]
    atflash.append_paged_kv_cache(k.to(DEV), v.to(DEV), bidx.to(DEV), pos.to(DEV), (d[0], d[2]), indices.to(DEV),
                                  indptr.to(DEV), kv_layout=layout, kv_scales=(d[1], d[3]), **kw)
    return d


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page,hkv,lens,app", [
    (16, 8, [1], [1]),
    (16, 4, [37, 80, 5, 16, 33], [1, 1, 1, 1, 1]),          # a decode step
    (16, 1, [37, 80, 5], [37, 33, 5]),                       # prompts and a chunk
    (64, 2, [200, 64, 0, 129], [130, 64, 0, 1]),             # runs over 16 rows, an empty request
    (256, 3, [600, 255], [511, 254]),
    (24, 2, [50, 7], [49, 3]),                               # any page size
    (1, 2, [9, 2], [4, 1]),
    (32, 8, [700], [700]),
])
def test_append_e4m3_matches_the_definition(layout, page, hkv, lens, app):
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup(layout, page, hkv, lens, app, page + hkv)
    want = _e4m3.append(*cache, k, v, bidx, pos, indptr, indices, layout)
    _check(_append(cache, k, v, bidx, pos, indptr, indices, layout), want)
    assert atflash.check_device_errors() == 0


def test_append_e4m3_many_tokens_then_steps():
    """A prompt, then tokens one by one whose magnitudes grow: scales are raised and
    the rows before are rounded again."""
    page, hkv, n = 16, 2, 1500
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", page, hkv, [n, n], [n, n], 5)
    import atflash
    d = [t.to(DEV) for t in cache]
    ref = list(cache)
    parts = [(0, n - 40)] + [(i, i + 1) for i in range(n - 40, n)]
    for lo, hi in parts:
        sel = torch.cat([torch.arange(lo, hi), torch.arange(n + lo, n + hi)])
        kk = k[sel] * (1.0 if hi - lo > 1 else 2.0 ** ((lo % 13) - 4))
        args = (kk, v[sel], bidx[sel], pos[sel], indptr, indices)
        out = _e4m3.append(*ref, *args, "NHD")
        ref = [torch.from_numpy(out[0]).to(torch.float8_e4m3fn), torch.from_numpy(out[1]).float(),
               torch.from_numpy(out[2]).to(torch.float8_e4m3fn), torch.from_numpy(out[3]).float()]
        atflash.append_paged_kv_cache(*(t.to(DEV) for t in args[:4]), (d[0], d[2]), indices.to(DEV), indptr.to(DEV),
                                      kv_scales=(d[1], d[3]))
    _check(d, out)


@pytest.mark.parametrize("out_layout", ["sorted_pair", "rotate_half"])
@pytest.mark.parametrize("rope_shift", [0, 11])
def test_append_e4m3_with_rope_equals_the_pack_then_the_append(out_layout, rope_shift):
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 3, [90, 21], [77, 1], 8, factor=2)
    cos, sin = rope_tables(128, 128, 1e4)
    rp = pos.long() + rope_shift
    packed = atflash.rope_pack(k.to(DEV)[None], cos.to(DEV), sin.to(DEV), positions=rp.to(DEV), out_layout=out_layout)
    want = _e4m3.append(*cache, packed[0].cpu(), v, bidx, pos, indptr, indices, "NHD")
    kw = dict(rope_positions=rp.to(DEV)) if rope_shift else {}
    _check(_append(cache, k, v, bidx, pos, indptr, indices, "NHD", rope=(cos.to(DEV), sin.to(DEV)),
                   out_layout=out_layout, **kw), want)


def test_append_e4m3_special_values():
    """Zeros, infinities, NaN, the smallest and the largest numbers."""
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 4, [16, 32, 48, 20, 7], [16, 16, 16, 4, 1], 9)
    k[:16] = 0
    v[:16, 1] = float("nan")
    k[16:32, 0, 5] = float("inf")
    k[16:32, 1, 7] = -float("inf")
    k[20, 2, 3] = float("nan")
    v[16:32] = torch.tensor(2.0 ** -133).bfloat16()
    v[20, 0, 0] = torch.finfo(torch.bfloat16).max
    k[32:48] = torch.where(torch.rand(16, 4, 128) < 0.5, 1.75 * 2.0 ** 3, 1.7578125 * 2.0 ** 3).bfloat16()
    k[48:52] = 0  # a run inside a page that keeps its scale
    v[48:52] = torch.finfo(torch.bfloat16).max
    want = _e4m3.append(*cache, k, v, bidx, pos, indptr, indices, "NHD")
    _check(_append(cache, k, v, bidx, pos, indptr, indices, "NHD"), want)


def test_append_e4m3_strided_inputs_and_one_tensor_cache():
    """Rows out of a fused projection; K and V pages as one tensor's halves; scales
    as columns of another tensor; a non-power-of-two scale set by the caller."""
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 2, [40, 23], [30, 2], 10)
    cache[1][:] *= 1.3
    want = _e4m3.append(*cache, k, v, bidx, pos, indptr, indices, "NHD")
    qkv = torch.zeros((len(pos), 9, 128), dtype=torch.bfloat16, device=DEV)
    qkv[:, 4:6], qkv[:, 7:9] = k.to(DEV), v.to(DEV)
    both = torch.stack([cache[0].view(torch.uint8), cache[2].view(torch.uint8)], dim=1).to(DEV).view(torch.float8_e4m3fn)
    sc = torch.stack([cache[1], cache[3]], dim=-1).to(DEV)
    atflash.append_paged_kv_cache(qkv[:, 4:6], qkv[:, 7:9], bidx.to(DEV), pos.to(DEV), both, indices.to(DEV),
                                  indptr.to(DEV), kv_scales=(sc[..., 0], sc[..., 1]))
    got = [both[:, 0], sc[..., 0], both[:, 1], sc[..., 1]]
    # 2.03125 / 1.3 is nearly a tie: the division must not round it into one
    _check(got, [want[0], want[1].astype(np.float32).astype(np.float64), want[2], want[3]])


def test_append_e4m3_padding_bad_pages_and_stream():
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 2, [40, 23], [30, 2], 11)
    st = torch.cuda.Stream()
    # padding entries are skipped without a report
    pb, pp = torch.cat([bidx, torch.full((5,), -1)]).to(torch.int32), torch.cat([pos, torch.full((5,), -1)]).to(torch.int32)
    pk, pv = (torch.cat([t, torch.full((5, 2, 128), 9.0, dtype=torch.bfloat16)]) for t in (k, v))
    want = _e4m3.append(*cache, k, v, bidx, pos, indptr, indices, "NHD")
    with torch.cuda.stream(st):
        got = _append(cache, pk, pv, pb, pp, indptr, indices, "NHD")
    st.synchronize()
    _check(got, want)
    assert atflash.check_device_errors() == 0
    # a position past the request's pages and a page id past the cache: skipped, reported
    for what in ("position", "page", "batch", "negative"):
        b2, p2, i2 = bidx.clone(), pos.clone(), indices.clone()
        if what == "position":
            p2[-2:] = torch.tensor([33, 34])
        elif what == "page":
            i2[-1] = 10 ** 6
        elif what == "batch":
            b2[-2:] = 2
        else:
            p2[-2:] = torch.tensor([-9, -8])
        want = _e4m3.append(*cache, k[:-2], v[:-2], b2[:-2], p2[:-2], indptr, i2, "NHD")
        _check(_append(cache, k, v, b2, p2, indptr, i2, "NHD"), want)
        assert atflash.check_device_errors() == 2, what


def test_append_e4m3_no_tokens_and_refusals():
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 2, [40], [3], 12)
    d = [t.to(DEV) for t in cache]
    e = torch.zeros(0, dtype=torch.int32, device=DEV)

    def call(k=k, v=v, cache=(d[0], d[2]), scales=(d[1], d[3]), b=bidx, p=pos, **kw):
        atflash.append_paged_kv_cache(k.to(DEV), v.to(DEV), b.to(DEV), p.to(DEV), cache, indices.to(DEV),
                                      indptr.to(DEV), kv_scales=scales, **kw)
    call(k[:0], v[:0], b=e, p=e)
    _check(d, [x.float().double().numpy() for x in cache])
    bf = torch.zeros_like(d[0], dtype=torch.bfloat16)
    bad = [dict(scales=None), dict(cache=(bf, bf)), dict(scales=(d[1], d[3][:-1])), dict(scales=(d[1].half(), d[3].half())),
           dict(scales=(d[1].cpu(), d[3].cpu())), dict(scales=d[1]), dict(scales=(d[1], d[3].t().contiguous().t())),
           dict(k=k.float()), dict(k=k[:, :1], v=v[:, :1]), dict(b=bidx[:1]), dict(kv_layout="DNH"),
           dict(cache=(d[0], d[2][:, :8])), dict(rope=(torch.zeros(64, 64), torch.zeros(64, 64))),
           dict(rope=(torch.zeros(64, 32, device=DEV), torch.zeros(64, 32, device=DEV))),
           dict(rope=(torch.zeros(64, 64, device=DEV),) * 2, rope_positions=torch.zeros(2, dtype=torch.int64))]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(KeyError):
        call(out_layout="interleaved")
    # rows of the cache that are not 16-byte aligned
    odd = torch.zeros((8, 16, 2, 136), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[..., :128]
    with pytest.raises(atflash.AtfError):
        call(cache=(odd, odd), scales=(torch.ones(8, 2, device=DEV),) * 2)
    assert atflash.check_device_errors() == 0
