"""Page tables and slot maps on a B200, entry for entry against Python loops: odd
lengths, empty requests, new pages from the free list, rows in another order,
capacities, bad requests, another stream, a CUDA graph."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _plain(lens, app, table, page, rows, free, head, cap_tokens, cap_pages):
    """The definition, one entry at a time; table is changed in place."""
    indptr, indices, last, aptr, bi, pos, slots = [0], [], [], [0], [], [], []
    for b, (x, a) in enumerate(zip(lens, app)):
        n, have = -(-x // page), (-(-(x - a) // page) if free is not None else -(-x // page))
        for j in range(have, n):
            table[rows[b], j] = free[head]
            head += 1
        ids = table[rows[b], :n].tolist()
        indices += ids
        indptr.append(indptr[-1] + n)
        last.append(x - (n - 1) * page if n else 0)
        for p in range(x - a, x):
            bi.append(b)
            pos.append(p)
            slots.append(ids[p // page] * page + p % page)
        aptr.append(aptr[-1] + a)

    def pad(v, n):
        return v + [-1] * (n - len(v))
    return [indptr, pad(indices, cap_pages), last, aptr, pad(bi, cap_tokens), pad(pos, cap_tokens),
            pad(slots, cap_tokens), [head]]


def _case(B, max_len, page, seed, extra_cap=0, with_free=True, shuffled=False, zero=0.2, prompt=0.3):
    g = np.random.default_rng(seed)
    lens = [0 if g.random() < zero else int(g.integers(1, max_len + 1)) for _ in range(B)]
    app = [int(g.integers(0, x + 1)) if g.random() < prompt else min(x, 1) for x in lens]
    width = -(-max_len // page) + 3
    R = B + (5 if shuffled else 0)
    rows = g.permutation(R)[:B] if shuffled else np.arange(B)
    need = sum(-(-x // page) for x in lens)
    ids = g.permutation(need + 50)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for b in range(B):
        have = -(-(lens[b] - app[b]) // page) if with_free else -(-lens[b] // page)
        table[rows[b], :have] = ids[at:at + have]
        at += have
    free = ids[at:].astype(np.int32) if with_free else None
    return lens, app, table, rows, free, sum(app) + extra_cap, need + extra_cap


def _run(lens, app, table, page, rows, free, head, cap_tokens, cap_pages, use_rows=True):
    import atflash
    t = torch.from_numpy(table.copy()).to(DEV)
    kw = dict(num_tokens=cap_tokens, max_pages=cap_pages)
    if free is not None:
        kw.update(free_pages=torch.from_numpy(free).to(DEV), free_head=torch.tensor([head], dtype=torch.int32, device=DEV))
    if use_rows:
        kw.update(req_rows=torch.tensor(np.asarray(rows), device=DEV))
    r = atflash.build_page_tables(torch.tensor(lens, dtype=torch.int32, device=DEV),
                                  torch.tensor(app, dtype=torch.int32, device=DEV), t, page, **kw)
    return r, t


def _same(r, t, want, table):
    got = [r.indptr, r.indices, r.last_page_len, r.append_indptr, r.batch_indices, r.positions, r.slot_mapping]
    for x, y in zip(got, want):
        assert x.tolist() == y
    if r.free_head is not None:
        assert r.free_head.tolist() == want[7]
    assert np.array_equal(t.cpu().numpy(), table)


@pytest.mark.parametrize("B,max_len,page", [(1, 1, 16), (1, 40, 16), (3, 300, 16), (31, 77, 1), (33, 1000, 64),
                                            (257, 513, 24), (513, 2000, 16), (1025, 100, 256), (8192, 40, 16)])
@pytest.mark.parametrize("variant", ["free", "rows_padded", "table_only"])
def test_tables_match_the_definition(B, max_len, page, variant):
    import atflash
    with_free, shuffled, extra = variant != "table_only", variant == "rows_padded", 37 if variant == "rows_padded" else 0
    lens, app, table, rows, free, ct, cp = _case(B, max_len, page, B + max_len, extra, with_free, shuffled)
    head = 3 if with_free else 0
    if with_free:
        free = np.concatenate([np.full(head, 10 ** 6, np.int32), free])
    ref = table.copy()
    want = _plain(lens, app, ref, page, rows, free, head, ct, cp)
    r, t = _run(lens, app, table, page, rows, free, head, ct, cp, use_rows=shuffled)
    _same(r, t, want, ref)
    assert atflash.check_device_errors() == 0


def test_tables_all_empty_and_first_token():
    import atflash
    table = np.full((4, 0), -1, np.int32)
    r, _ = _run([0] * 4, [0] * 4, table, 16, range(4), None, 0, 0, 0, use_rows=False)
    assert r.indptr.tolist() == [0] * 5 and r.last_page_len.tolist() == [0] * 4 and r.append_indptr.tolist() == [0] * 5
    # lengths on each side of a page's end
    lens = [15, 16, 17, 32, 33, 1]
    table = np.full((6, 4), -1, np.int32)
    free = np.arange(100, 120, dtype=np.int32)
    for b, x in enumerate(lens):
        table[b, :-(-(x - 1) // 16)] = np.arange(-(-(x - 1) // 16)) + 10 * b
    ref = table.copy()
    want = _plain(lens, [1] * 6, ref, 16, range(6), free, 0, 6, 12)
    r, t = _run(lens, [1] * 6, table, 16, range(6), free, 0, 6, 12, use_rows=False)
    _same(r, t, want, ref)
    assert atflash.check_device_errors() == 0


def test_tables_report_bad_requests_and_capacities():
    import atflash
    free = np.arange(50, 90, dtype=np.int32)
    ok = dict(lens=[20, 33, 5], app=[20, 1, 5])
    table = np.tile(np.arange(4, dtype=np.int32), (3, 1)) + 4 * np.arange(3, dtype=np.int32)[:, None]

    def flagged(lens, app, free=free, head=0, ct=26, cp=6, rows=range(3)):
        r, _ = _run(lens, app, table, 16, rows, free, head, ct, cp)
        assert atflash.check_device_errors() == 2
        assert r.indptr.tolist() == sorted(r.indptr.tolist()) and r.indptr[-1] <= cp
        assert r.append_indptr[-1] <= ct
        return r

    for lens, app, rows in (([20, -1, 5], [20, 0, 5], range(3)), ([20, 5, 5], [20, 6, 5], range(3)),
                            ([20, 5, 5], [20, -1, 5], range(3)), ([20, 65, 5], [20, 1, 5], range(3)),
                            ([20, 33, 5], [20, 1, 5], [0, 3, 2]), ([20, 33, 5], [20, 1, 5], [0, -1, 2])):
        r = flagged(lens, app, rows=rows)  # the bad one counts as empty
        assert r.indptr.tolist() == [0, 2, 2, 3] and r.last_page_len.tolist() == [4, 0, 5]
        assert r.append_indptr.tolist() == [0, 20, 20, 25]
    # the free list ends: its pages come first, then -1, and their slots too
    r = flagged(**ok, head=39)
    assert r.indices.tolist()[0] == 89 and r.indices.tolist()[1] == -1 and r.free_head.tolist() == [40]
    assert r.slot_mapping.tolist()[:17] == [89 * 16 + i for i in range(16)] + [-1]
    flagged(**ok, head=-1)
    r = flagged(**ok, cp=4)
    assert r.indptr.tolist() == [0, 2, 4, 4]
    r = flagged(**ok, ct=21)
    assert r.append_indptr.tolist() == [0, 20, 21, 21]


def test_tables_refusals():
    import atflash
    a = dict(num_tokens=4, max_pages=4)
    lens = torch.tensor([4, 4], dtype=torch.int32, device=DEV)
    table = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens[:1], table, 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens.float(), lens, table, 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table[:1], 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table.long(), 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table[:, ::2], 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table[:1].expand(2, 3), 16, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table, 0, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table, 16, num_tokens=-1, max_pages=4)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table, 16, free_pages=lens, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens, lens, table, 16, free_pages=lens, free_head=lens, **a)
    with pytest.raises(ValueError):
        atflash.build_page_tables(lens.cpu(), lens, table, 16, **a)
    big = torch.zeros(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        atflash.build_page_tables(big, big, torch.zeros((8193, 1), dtype=torch.int32, device=DEV), 16, **a)


def test_tables_on_another_stream_and_in_a_graph():
    import atflash
    lens, app, table, rows, free, ct, cp = _case(65, 500, 16, 3)
    ref = table.copy()
    want = _plain(lens, app, ref, 16, rows, free, 0, ct, cp)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        r, t = _run(lens, app, table, 16, rows, free, 0, ct, cp, use_rows=False)
    st.synchronize()
    _same(r, t, want, ref)
    # a captured step follows the lengths in its buffers
    dl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    da = torch.tensor(app, dtype=torch.int32, device=DEV)
    t2, fp = torch.from_numpy(table.copy()).to(DEV), torch.from_numpy(free).to(DEV)
    fh = torch.zeros(1, dtype=torch.int32, device=DEV)
    kw = dict(num_tokens=ct, max_pages=cp, free_pages=fp, free_head=fh)
    atflash.build_page_tables(dl, da, t2.clone(), 16, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = atflash.build_page_tables(dl, da, t2, 16, **kw)
    for step in range(2):
        t2.copy_(torch.from_numpy(table))
        if step:
            app = [min(a, 1) for a in app]
            da.copy_(torch.tensor(app, dtype=torch.int32))
            ref = table.copy()
            for b in range(len(lens)):  # pages that only this step needs are in the table now
                ref[b, :-(-(lens[b] - app[b]) // 16)] = np.arange(-(-(lens[b] - app[b]) // 16)) + 7000
            t2.copy_(torch.from_numpy(ref))
            want = _plain(lens, app, ref, 16, rows, free, 0, ct, cp)
        graph.replay()
        torch.cuda.synchronize()
        _same(r, t2, want, ref)
    assert atflash.check_device_errors() == 0
