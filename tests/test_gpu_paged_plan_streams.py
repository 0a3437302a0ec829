"""Plans of the paged prefill and runs on other streams: what a plan converts is there
before a run on any stream reads it."""
import pytest
import torch

from test_gpu_paged import DEV, WS, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["int64", "strided"])
def test_indices_that_a_plan_converts_are_there_for_every_stream(kind):
    import atflash
    c = Case(16, "NHD", 8, 2, [(5, 900), (130, 700), (1, 33)], seed=4)
    want = c.run(c.plan())
    given = c.indices.to(DEV)
    if kind == "int64":
        given = given.long()
    else:
        wide = torch.zeros((given.numel(), 2), dtype=torch.int32, device=DEV)
        wide[:, 0] = given
        given = wide[:, 0]
    w = atflash.BatchPrefillWithPagedKVCacheWrapper(torch.empty(WS, dtype=torch.uint8, device=DEV), c.layout)
    other, late = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(late):
        torch.cuda._sleep(100_000_000)  # the stream of the plan is behind
        w.plan(c.cq, c.starts, given, c.last, c.hq, c.hkv, 128, c.page)
    with torch.cuda.stream(other):  # (which waits for nothing)
        got = c.run(w)
    other.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert atflash.check_device_errors() == 0
