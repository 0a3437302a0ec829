"""Items of over two hundred stages, so that the ring of the e4m3 decode turns many
times for one CTA, and the same answer from every run."""
import pytest
import torch

from test_gpu_decode_e4m3 import DEV, Z16, _close, _exact, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,layout", [(16, "NHD"), (64, "HND")])
@pytest.mark.parametrize("window", [None, Z16])
def test_decode_e4m3_items_of_two_hundred_stages(page, layout, window):
    import atflash
    lens = [9000, 13011, 77, 4032]
    cache, q, indptr, indices, last = _setup(lens, page, 2, 2, layout, 27)
    want = _exact(cache, q, indptr, indices, lens, layout, zhi=window)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV), layout)
    w.plan(indptr, indices, last, 4, 2, 128, page, kv_data_type=torch.float8_e4m3fn, window_table=window,
           min_chunk_keys=8192)
    items = w._plan["items"].cpu()
    assert int((items[:, 2] - items[:, 1]).max()) > 200 * 64
    d = [t.to(DEV) for t in cache]

    def run():
        return w.run(q.to(DEV), (d[0], d[2]), kv_scales=(d[1], d[3]), return_lse=True, out_dtype=torch.float32)
    first = run()
    _close(first, want)
    for _ in range(5):
        got = run()
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    assert atflash.check_device_errors() == 0
