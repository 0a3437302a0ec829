"""Page tables whose lists are cut by a capacity: the engine's rows, the free list and
the slots are those of the whole step, and the call repeated with room gives the whole
lists. A row that lacks a page is reported."""
import numpy as np
import pytest
import torch

from test_gpu_tables import DEV, _case, _plain, _same

pytestmark = pytest.mark.gpu


def _call(dl, da, t, page, free, head, tokens, pages):
    import atflash
    return atflash.build_page_tables(dl, da, t, page, num_tokens=tokens, max_pages=pages, free_pages=free, free_head=head)


@pytest.mark.parametrize("B,max_len,page", [(3, 100, 16), (40, 500, 16), (600, 900, 32)])
@pytest.mark.parametrize("part", [0.0, 0.4, 0.99])
def test_a_cut_list_loses_no_page(B, max_len, page, part):
    import atflash
    lens, app, table, rows, free, ct, cp = _case(B, max_len, page, B, zero=0.1, prompt=0.9)
    ref = table.copy()
    want = _plain(lens, app, ref, page, rows, free, 0, ct, cp)
    dl, da = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, app))
    t, fp, fh = torch.from_numpy(table.copy()).to(DEV), torch.from_numpy(free).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cut = int(part * cp)
    r = _call(dl, da, t, page, fp, fh, ct, cut)
    assert atflash.check_device_errors() == 2
    assert np.array_equal(t.cpu().numpy(), ref) and r.free_head.tolist() == want[7]
    assert r.indptr.tolist() == [min(x, cut) for x in want[0]] and r.indices.tolist() == want[1][:cut]
    assert [r.last_page_len.tolist(), r.append_indptr.tolist(), r.batch_indices.tolist(), r.positions.tolist(),
            r.slot_mapping.tolist()] == want[2:7]
    # fewer tokens listed than there are: the pages are the same
    t.copy_(torch.from_numpy(table))
    r = _call(dl, da, t, page, fp, fh, ct // 2, cp)
    assert atflash.check_device_errors() == 2
    assert np.array_equal(t.cpu().numpy(), ref) and r.free_head.tolist() == want[7] and r.indices.tolist() == want[1]
    assert r.slot_mapping.tolist() == want[6][:ct // 2]
    # again, over the rows as they are now and with room
    r = _call(dl, da, t, page, fp, fh, ct, cp)
    _same(r, t, want, ref)
    assert atflash.check_device_errors() == 0


def test_a_row_without_its_page_is_reported():
    import atflash
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    lens = torch.tensor([40, 33, 16], dtype=torch.int32, device=DEV)
    ones = torch.ones_like(lens)
    kw = dict(num_tokens=3, max_pages=7)
    atflash.build_page_tables(lens, ones, table, 16, **kw)
    assert atflash.check_device_errors() == 0
    table[1, 1] = -1
    r = atflash.build_page_tables(lens, ones, table, 16, **kw)
    assert atflash.check_device_errors() == 2
    assert r.indices.tolist() == [0, 1, 2, 4, -1, 6, 8]
