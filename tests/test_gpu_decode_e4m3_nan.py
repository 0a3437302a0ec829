"""A NaN among a request's own scores reaches the outputs and the lse of its heads, and
nothing else; only a row without weight has an lse of -inf."""
import numpy as np
import pytest
import torch

import _e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("chunk", [0, 64])          # one item, and several to merge
@pytest.mark.parametrize("copies", [1, 70])         # the merge by blocks, and by warps
@pytest.mark.parametrize("where", ["q", "k", "k_scale", "q_inf"])
def test_decode_e4m3_nan_scores(where, copies, chunk):
    import atflash
    g = torch.Generator().manual_seed(3)
    page, hkv, group, lens = 16, 2, 9 if copies > 1 else 3, [200, 70] * copies
    npg = [-(-n // page) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(npg)])
    cache = [t.to(DEV) for t in _e4m3.random_cache(sum(npg), page, hkv, "NHD", g)]
    q = torch.randn((len(lens), hkv * group, 128), generator=g).bfloat16().to(DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.zeros(64 << 20, dtype=torch.uint8, device=DEV), "NHD")
    w.plan(indptr, torch.arange(sum(npg), dtype=torch.int32), [(n - 1) % page + 1 for n in lens], hkv * group, hkv, 128,
           page, kv_data_type=torch.float8_e4m3fn, max_chunk_keys=chunk)

    def run():
        return w.run(q, (cache[0], cache[2]), kv_scales=(cache[1], cache[3]), return_lse=True, out_dtype=torch.float32)
    out, lse = run()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    hit = torch.zeros(lse.shape, dtype=torch.bool, device=DEV)
    if where == "q":
        q[0, 1, 17] = float("nan")
        hit[0, 1] = True
    elif where == "q_inf":
        q[0, 1, 17] = float("inf")  # scores of both infinities
        hit[0, 1] = True
    elif where == "k":
        cache[0].view(torch.uint8)[1, 3, 1, 40] = 0x7f
        hit[0, group:] = True
    else:
        cache[1][1, 1] = float("nan")
        hit[0, group:] = True
    got, gl = run()
    assert torch.equal(gl.isnan(), hit)
    assert torch.equal(got.isnan(), hit[..., None].expand(got.shape))
    assert torch.equal(got[~hit], out[~hit]) and torch.equal(gl[~hit], lse[~hit])
    assert atflash.check_device_errors() == 0


def test_lse_merge_of_nan_and_of_no_weight():
    import atflash
    o = torch.ones((2, 1, 2, 128), device=DEV)
    lse = torch.tensor([[[1.0, -np.inf]], [[np.nan, -np.inf]]], device=DEV, dtype=torch.float32)
    out, l2 = atflash.lse_merge(o, lse, return_lse=True)
    assert torch.isnan(l2[0, 0]) and torch.isneginf(l2[0, 1])
    assert torch.isnan(out[0, 0]).all() and torch.count_nonzero(out[0, 1]) == 0
