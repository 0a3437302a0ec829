"""The append over ctypes writes what the compiled binding's writes, bit for bit, and
refuses the same calls."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:append_paged_kv_cache goes through ctypes")]
DEV = "cuda:0"


def _no_binding(monkeypatch):
    from atflash import _ffi

    def missing():
        raise ImportError("no binding")
    monkeypatch.setattr(_ffi, "binding", missing)


def _call(kind, ints=torch.int32, rope=True, **change):
    """Arguments of an append of 40 tokens of 2 requests, and its cache tensors"""
    g = torch.Generator().manual_seed(3)
    page, hkv, P = 16, 2, 6
    k, v = (torch.randn((40, hkv, 128), generator=g).bfloat16().to(DEV) for _ in range(2))
    pos = list(range(5, 30)) + list(range(15))
    layout = "HND" if kind.endswith("hnd") else "NHD"
    shape = (P, hkv, page, 128) if layout == "HND" else (P, page, hkv, 128)
    dtype = torch.float8_e4m3fn if kind.startswith("e4m3") else torch.bfloat16
    vc = torch.zeros(shape, device=DEV).to(dtype)
    kc = torch.zeros((P, hkv, 8, page, 16), device=DEV).to(dtype) if kind == "level" else torch.zeros_like(vc)
    scales = tuple(torch.ones((P, hkv), device=DEV) for _ in range(2)) if kind.startswith("e4m3") else None
    i = lambda x: torch.tensor(x, dtype=ints, device=DEV)
    a = dict(append_key=k, append_value=v, batch_indices=i([0] * 25 + [1] * 15), positions=i(pos), paged_kv_cache=(kc, vc),
             kv_indices=i([4, 1, 3]), kv_indptr=i([0, 2, 3]), kv_layout=layout, kv_scales=scales)
    if rope:
        t = torch.randn((64, 64), generator=g).to(DEV)
        a.update(rope=(t.cos(), t.sin()), rope_positions=i([p + 7 for p in pos]),
                 out_layout="rotate_half" if kind == "hnd" else "sorted_pair")
    a.update(change)
    return a, [kc, vc] + list(scales or ())


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("kind", ["nhd", "hnd", "level", "e4m3_nhd", "e4m3_hnd"])
def test_the_same_pages(monkeypatch, kind, rope, ints):
    import atflash
    a, want = _call(kind, ints, rope)
    atflash.append_paged_kv_cache(**a)
    b, got = _call(kind, ints, rope)
    _no_binding(monkeypatch)
    atflash.append_paged_kv_cache(**b)
    for x, y in zip(got, want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert want[1].float().abs().sum() > 0
    assert atflash.check_device_errors() == 0


def test_reports_and_empty_calls(monkeypatch):
    import atflash
    _no_binding(monkeypatch)
    for kind in ("nhd", "e4m3_nhd"):
        a, _ = _call(kind)
        a["kv_indices"] = a["kv_indices"].clone()
        a["kv_indices"][1] = 6  # outside the cache
        atflash.append_paged_kv_cache(**a)
        assert atflash.check_device_errors() == 2
        a, cache = _call(kind)
        for n in ("append_key", "append_value", "batch_indices", "positions", "rope_positions"):
            a[n] = a[n][:0]
        atflash.append_paged_kv_cache(**a)
        assert cache[1].float().abs().sum() == 0 and atflash.check_device_errors() == 0


@pytest.mark.parametrize("with_binding", [True, False])
def test_refusals(monkeypatch, with_binding):
    import atflash
    if not with_binding:
        _no_binding(monkeypatch)
    a, _ = _call("nhd")
    kc, vc = a["paged_kv_cache"]
    k, c = a["append_key"], a["rope"][0]
    e8 = kc.to(torch.float8_e4m3fn)
    for bad in (dict(append_value=a["append_value"][:3]), dict(append_key=k[:, :1], append_value=k[:, :1]),
                dict(append_key=k.float()), dict(paged_kv_cache=(kc, vc[:3])), dict(paged_kv_cache=(e8, e8)),
                dict(kv_layout="x"), dict(batch_indices=a["batch_indices"][:3]), dict(rope=(c, c[:3])), dict(rope=(c[:0], c[:0])),
                dict(rope=(c.double(), c.double())), dict(rope=(c, None)), dict(rope_positions=a["rope_positions"][:2]),
                dict(paged_kv_cache=(kc.cpu(), vc.cpu())), dict(append_key=k[0], append_value=k[0])):
        with pytest.raises(ValueError):
            atflash.append_paged_kv_cache(**{**a, **bad})
    with pytest.raises(KeyError):
        atflash.append_paged_kv_cache(**{**a, "out_layout": "x"})
    e, _ = _call("e4m3_nhd")
    s = e["kv_scales"][0]
    for bad in (dict(kv_scales=(s, s[:2])), dict(kv_scales=(s,)), dict(kv_scales=(s.double(), s.double())),
                dict(paged_kv_cache=(kc, vc)), dict(append_key=k.float()), dict(kv_layout="x")):
        with pytest.raises(ValueError):
            atflash.append_paged_kv_cache(**{**e, **bad})
    lv, _ = _call("level")
    lk, lvv = lv["paged_kv_cache"]
    for bad in (dict(paged_kv_cache=(lk[:, :, :4], lvv)), dict(paged_kv_cache=(lk[:, :1], lvv)), dict(out_layout="rotate_half")):
        with pytest.raises(ValueError):
            atflash.append_paged_kv_cache(**{**lv, **bad})
