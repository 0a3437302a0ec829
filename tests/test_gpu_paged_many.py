"""Batches of more (request, kv head) pairs than are planned one by one: the long request
among them is cut, and every request is right."""
import pytest
import torch

from test_gpu_paged import ZHI, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("zhi", [None, ZHI])
@pytest.mark.parametrize("hq,hkv,reqs,look", [
    (16, 8, [(1, 300)] * 40 + [(2, 30001)] + [(1, 299)] * 60, (0, 39, 40, 41, 100)),
    (8, 8, [(1, 200 + i) for i in range(90)] + [(130, 40000)], (0, 50, 89, 90)),
    (16, 4, [(300, 700)] * 32 + [(1, 60000)] + [(3, 77)] * 8, (0, 31, 32, 33, 40)),
])
def test_a_long_request_among_many(hq, hkv, reqs, look, zhi):
    import atflash
    c = Case(16, "NHD", hq, hkv, reqs, seed=12)
    w = c.plan(zhi=zhi)
    assert w._plan.num_parts > 0 and (w._plan.num_items - w._plan.num_wide) * hkv + w._plan.num_wide * hq > 592
    out, lse = c.run(w)
    c.check(out, lse, zhi=zhi, requests=look)
    again = c.run(w)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert atflash.check_device_errors() == 0
