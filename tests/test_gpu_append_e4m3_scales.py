"""The e4m3 append under scales that another program set: the largest and the least
powers of two among them, byte for byte."""
import pytest
import torch

import _e4m3
from test_gpu_append_e4m3 import _append, _check, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent,factor", [(e, f) for e in (127, 126, 125, 121, -126) for f in (1.0, 1.5)] + [(-149, 1.0)])
def test_append_e4m3_under_extreme_scales(exponent, factor):
    cache, k, v, bidx, pos, indptr, indices = _setup("NHD", 16, 2, [40, 23], [30, 2], 10)
    k = (k.float().clamp(-1.9, 1.9) * 2.0 ** 126).bfloat16()
    v = v.float().bfloat16()
    for s in (cache[1], cache[3]):
        s.fill_(factor * 2.0 ** exponent)
    want = _e4m3.append(*cache, k, v, bidx, pos, indptr, indices, "NHD")
    _check(_append(cache, k, v, bidx, pos, indptr, indices, "NHD"), want)
