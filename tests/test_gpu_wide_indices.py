"""64-bit index tensors: values that fit give the 32-bit call's results, values that do
not are reported, never taken modulo 2^32."""
import pytest
import torch

import _e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WIDE = 1 << 32


def _i64(*x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("wide", ["none", "kv_lens", "append_lens", "req_rows", "free_head", "free_pages"])
def test_tables_take_no_length_or_row_modulo_two_to_the_32(wide):
    import atflash
    a = dict(kv_lens=_i64(20, 5), append_lens=_i64(20, 5), req_rows=_i64(1, 0), free_pages=_i64(7, 8, 9), free_head=_i64(0))
    if wide != "none":
        a[wide] = a[wide] + WIDE * _i64(*([1] + [0] * (a[wide].numel() - 1)))
    table = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    r = atflash.build_page_tables(a["kv_lens"], a["append_lens"], table, 16, num_tokens=25, max_pages=3,
                                  req_rows=a["req_rows"], free_pages=a["free_pages"], free_head=a["free_head"])
    indices, code = r.indices.tolist(), atflash.check_device_errors()
    if wide == "none":
        assert code == 0 and indices == [7, 8, 9] and table.tolist() == [[9, -1], [7, 8]]
    elif wide == "free_pages":  # an id for the cache's own check
        assert indices == [2 ** 31 - 1, 8, 9]
    elif wide == "free_head":
        assert code == 2 and indices == [-1, -1, -1]
    else:  # that request counts as empty
        assert code == 2 and r.indptr.tolist() == [0, 0, 1]


@pytest.mark.parametrize("what", ["none", "batch", "position", "page"])
@pytest.mark.parametrize("e4m3", [True, False])
def test_append_writes_nothing_for_an_index_that_does_not_fit(what, e4m3):
    import atflash
    g = torch.Generator().manual_seed(1)
    k = torch.randn((1, 1, 128), generator=g).bfloat16().to(DEV)
    d = [t.to(DEV) for t in _e4m3.random_cache(3, 16, 1, "NHD", g)]
    if not e4m3:
        d = [t.float().bfloat16() if t.dim() == 4 else t for t in d]
    before = [t.clone() for t in d]
    a = dict(batch=_i64(0), position=_i64(3), page=_i64(1))
    if what != "none":
        a[what] = a[what] + WIDE
    atflash.append_paged_kv_cache(k, k, a["batch"], a["position"], (d[0], d[2]), a["page"], _i64(0, 1),
                                  **(dict(kv_scales=(d[1], d[3])) if e4m3 else {}))
    same = [torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(d, before)]
    if what == "none":
        assert atflash.check_device_errors() == 0 and not same[0] and not same[2]
    else:
        assert atflash.check_device_errors() == 2 and all(same)


def test_decode_reads_no_page_modulo_two_to_the_32():
    import atflash
    g = torch.Generator().manual_seed(2)
    d = [t.to(DEV) for t in _e4m3.random_cache(3, 16, 1, "NHD", g)]
    q = torch.randn((1, 2, 128), generator=g).bfloat16().to(DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.zeros(16 << 20, dtype=torch.uint8, device=DEV), "NHD")
    for pages, code in ((_i64(2, 0), 0), (_i64(2, WIDE), 2)):
        w.plan([0, 2], pages, [5], 2, 1, 128, 16, kv_data_type=torch.float8_e4m3fn)
        w.run(q, (d[0], d[2]), kv_scales=(d[1], d[3]))
        assert atflash.check_device_errors() == code
