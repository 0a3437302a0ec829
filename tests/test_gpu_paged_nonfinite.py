"""Keys and values that are not finite, in the attention of chunks over pages: what rows
that do not see them are, whether the keys are cut over SMs or not."""
import pytest
import torch

from test_gpu_paged import Case

pytestmark = pytest.mark.gpu


def _slot(c, b, key):
    return c.indices[c.starts[b] + key // c.page].long(), key % c.page


@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1)])
@pytest.mark.parametrize("reqs,cut", [([(4, 300), (130, 130)], False), ([(4, 20001)], True)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_masked_key_changes_no_row(hq, hkv, reqs, cut, value):
    """The last key of request 0 is the last row's alone; the others load its tile."""
    c = Case(16, "NHD", hq, hkv, reqs, seed=9)
    w = c.plan()
    assert (w._plan.num_parts > 0) == cut
    out, lse = c.run(w)
    c.check(out, lse)
    c.k[_slot(c, 0, reqs[0][1] - 1)] = value
    got, got_lse = c.run(w)
    last = c.cq[1] - 1
    keep = torch.arange(c.cq[-1]) != last
    assert torch.equal(got[keep], out[keep]) and torch.equal(got_lse[keep], lse[keep])
    if value != value:
        assert got[last].isnan().all() and got_lse[last].isnan().all()


@pytest.mark.parametrize("hq,hkv", [(2, 1), (4, 4)])
@pytest.mark.parametrize("where", [0, 4500, 8995])
def test_a_nan_key_reaches_every_row_over_cut_keys(hq, hkv, where):
    c = Case(16, "NHD", hq, hkv, [(5, 9000), (1, 20000)], seed=10)
    w = c.plan()
    assert w._plan.num_parts > 0
    out, lse = c.run(w)
    c.k[_slot(c, 0, where)] = float("nan")
    got, got_lse = c.run(w)
    assert got[:5].isnan().all() and got_lse[:5].isnan().all()
    assert torch.equal(got[5:], out[5:]) and torch.equal(got_lse[5:], lse[5:])


@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1)])
def test_an_infinite_value_stays_with_the_tiles_that_load_its_key_tile(hq, hkv):
    """Key 259 lies in key tile 2, which the rows before 256 do not load. The rows from 256 on
    do; the last one, which sees the key, is not finite, and what the others are is not said."""
    c = Case(16, "NHD", hq, hkv, [(260, 260), (6, 40)], seed=11)
    w = c.plan()
    out, lse = c.run(w)
    c.v[_slot(c, 0, 259)] = float("inf")
    got, got_lse = c.run(w)
    assert torch.equal(got[:256], out[:256]) and torch.equal(got[260:], out[260:])
    assert not torch.isfinite(got[259]).any()
    assert torch.equal(got_lse, lse)  # (no value enters it)
