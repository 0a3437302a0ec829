"""Pages whose V scale is far above the others' because of one channel: the other
channels keep their own accuracy, channel by channel.

Bound of a channel c, beside the scores' error (2 err, see test_gpu_decode_e4m3): P has
11 bits down to 2^-21 of the largest weight w_n = p_n vs_n, so 2^-11 of sum p |v_c|
with the sums' rounding; smaller weights are off by at most 2^-32 of the largest, each
times its stored |v_nc|."""
import math

import numpy as np
import pytest
import torch

from test_gpu_decode_e4m3 import DEV, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ratio", [0, 10, 16, 20, 24])
@pytest.mark.parametrize("group", [3, 12])
def test_decode_e4m3_one_channel_sets_some_pages_scale(ratio, group):
    import atflash
    lens, page, hkv = [700, 2000], 16, 2
    (k, ks, v, vs), q, indptr, indices, last = _setup(lens, page, hkv, group, "NHD", 40 + ratio, spread=0)
    ks *= 0.02  # scores of a few units
    for b in range(2):
        # the first 128 keys of each request: the state that its other keys go on with
        out = indices[int(indptr[b]):int(indptr[b]) + 8].long()
        v[out] = 0
        v[out, :, :, 5] = 448.0
        vs[out] *= 2.0 ** ratio
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV), "NHD")
    w.plan(indptr, indices, last, hkv * group, hkv, 128, page, kv_data_type=torch.float8_e4m3fn, min_chunk_keys=4096)
    got = w.run(q.to(DEV), (k.to(DEV), v.to(DEV)), kv_scales=(ks.to(DEV), vs.to(DEV)), out_dtype=torch.float32)
    got = got.double().cpu().numpy()
    kf, vf, ksd, vsd = k.float().double().numpy(), v.float().double().numpy(), ks.double().numpy(), vs.double().numpy()
    for b, n in enumerate(lens):
        ids = indices[int(indptr[b]):int(indptr[b + 1])].long().numpy()
        slot = np.arange(n) // page
        for h in range(hkv * group):
            hk = h // group
            kb = (kf[ids][:, :, hk] * ksd[ids, hk][:, None, None]).reshape(-1, 128)[:n]
            vb, sc = vf[ids][:, :, hk].reshape(-1, 128)[:n], vsd[ids, hk][slot]
            qq = q[b, h].double().numpy()
            s = kb @ qq / math.sqrt(128)
            err = (np.abs(kb) @ np.abs(qq) / math.sqrt(128)).max() * 2.0 ** -17
            p = np.exp(s - s.max())
            weight = p / p.sum() * sc
            ref, mag = weight @ vb, weight @ np.abs(vb)
            tol = (2.0 ** -11 + 2 * err) * mag + 2.0 ** -32 * weight.max() * np.abs(vb).sum(0) + 2.0 ** -20 * np.abs(ref)
            assert np.all(np.abs(got[b, h] - ref) <= tol), (np.abs(got[b, h] - ref) / tol).max()
    assert atflash.check_device_errors() == 0
