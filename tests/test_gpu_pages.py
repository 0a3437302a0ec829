"""Shared pages on a B200: fork, free and compact against a step-by-step model, entry
for entry; copies of pages in every kind of cache tensor; reports, streams, graphs; and
a run of them with the page tables, the append and the decode."""
import random

import pytest
import torch

from _pages import Pool, pages_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Mirror:
    """A pool and its tensors, with the calls made on both."""

    def __init__(self, num_pages, rows, width, page, seed=0):
        order = list(range(num_pages))
        random.Random(seed).shuffle(order)
        self.m, self.page = Pool(num_pages, rows, width, order), page
        self.table, self.shared, self.free, self.head = _i32(self.m.rows), _i32(self.m.shared), _i32(order), _i32([0])

    def upload(self):
        self.table, self.shared, self.free, self.head = (_i32(self.m.rows), _i32(self.m.shared), _i32(self.m.free),
                                                         _i32([self.m.head]))

    def fork(self, parents, children, lens):
        import atflash
        want = self.m.fork(parents, children, lens, self.page)
        f = atflash.fork_requests(_i32(parents), _i32(children), _i32(lens), self.table, self.page, free_pages=self.free,
                                  free_head=self.head, shared=self.shared)
        assert (f.src.tolist(), f.dst.tolist()) == (want[0], want[1])
        self.head = f.free_head
        return f

    def give_back(self, rows, lens, with_shared=True):
        import atflash
        self.m.give_back(rows, lens, self.page)
        self.head = atflash.free_requests(_i32(rows), _i32(lens), self.table, self.page, free_pages=self.free,
                                          free_head=self.head, shared=self.shared if with_shared else None)

    def compact(self, rows, lens, max_moves):
        import atflash
        want = self.m.compact(rows, lens, self.page, max_moves)
        c = atflash.compact_pages(_i32(lens), self.table, self.page, len(self.m.shared), max_moves=max_moves,
                                  free_pages=self.free, req_rows=_i32(rows), shared=self.shared)
        assert (c.src.tolist(), c.dst.tolist()) == (want[0], want[1])
        self.head = c.free_head
        return c

    def same(self, errors=0):
        import atflash
        assert self.table.tolist() == self.m.rows
        assert self.shared.tolist() == self.m.shared
        assert self.free.tolist() == self.m.free
        assert self.head.tolist() == [self.m.head]
        assert atflash.check_device_errors() == errors


@pytest.mark.parametrize("page,rows,width,seed", [(16, 12, 9, 0), (1, 5, 40, 1), (64, 40, 70, 2), (24, 300, 33, 3)])
def test_a_life_of_forks_frees_and_compactions(page, rows, width, seed):
    rng = random.Random(seed)
    x = Mirror(rows * width // 2 + 5, rows, width, page, seed)
    lens = {}  # requests in the rows
    for step in range(12):
        idle = [r for r in range(rows) if r not in lens]
        for r in rng.sample(idle, min(len(idle), rng.randint(0, 3))):  # new prompts
            n = rng.randint(0, page * width)
            if x.m.head + pages_of(n, page) <= len(x.m.free):
                x.m.take(r, pages_of(n, page))
                lens[r] = n
        x.upload()
        idle = [r for r in range(rows) if r not in lens]
        if lens and idle:
            kids = rng.sample(idle, rng.randint(1, min(len(idle), 20)))
            parents = [rng.choice(list(lens)) for _ in kids]
            take = [rng.choice([lens[p], rng.randint(0, lens[p])]) for p in parents]
            if x.m.head + len(kids) <= len(x.m.free):
                x.fork(parents, kids, take)
                lens.update(zip(kids, take))
                x.same()
        if lens and rng.random() < 0.7:
            gone = rng.sample(list(lens), rng.randint(1, len(lens)))
            x.give_back(gone, [lens[r] for r in gone])
            for r in gone:
                del lens[r]
            x.same()
        if lens and rng.random() < 0.6:
            order = rng.sample(list(lens), len(lens))
            x.compact(order, [lens[r] for r in order], rng.choice([1, 3, len(x.m.shared)]))
            x.same()


def test_one_parent_of_many_and_pages_freed_together():
    x = Mirror(64, 30, 8, 16)
    x.m.take(0, 8)
    x.upload()
    x.fork([0] * 25, list(range(1, 26)), [128 - (i % 3) * 5 for i in range(25)])
    x.same()
    x.give_back([0] + list(range(2, 26)), [128] + [128 - (i % 3) * 5 for i in range(1, 25)])  # all but one
    x.same()
    x.give_back([1], [128])  # the last holder
    x.same()
    assert x.m.shared == [0] * 64 and sorted(x.m.free) == list(range(64)) and x.m.head == 0


@pytest.mark.parametrize("rows,kids", [(10900, 50), (10200, 700), (11900, 60)])
def test_tables_whose_lists_fill_48_kb_of_shared_memory(rows, kids):
    # R + 2 N words, of which 48 KB need no leave
    x = Mirror(kids + 200, rows, 3, 8, 6)
    for r in range(40):
        x.m.take(r, 3)
    x.upload()
    children = list(range(rows - kids, rows))
    take = [24 - i % 25 for i in range(kids)]
    x.fork([i % 40 for i in range(kids)], children, take)
    x.same()
    x.give_back(children, take)
    x.same()


def test_the_largest_tables():
    rows, width = 8192, 20
    x = Mirror(rows * width // 2, rows, width, 16, 5)
    rng = random.Random(5)
    lens = {r: rng.randint(0, 16 * 7) for r in range(4096)}
    for r, n in lens.items():
        x.m.take(r, pages_of(n, 16))
    x.upload()
    kids = list(range(4096, 8192))
    take = [rng.randint(0, lens[k - 4096]) for k in kids]
    x.fork([k - 4096 for k in kids], kids, take)
    x.same()
    lens.update(zip(kids, take))
    gone = rng.sample(list(lens), 5000)
    x.give_back(gone, [lens.pop(r) for r in gone])
    x.same()
    x.compact(list(lens), list(lens.values()), 30000)
    x.same()


def test_compaction_of_a_million_pages():
    import atflash
    num, width = atflash._ffi.ATF_COMPACT_MAX_PAGES, 700
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(num, generator=g).to(torch.int32)[:900 * width].view(900, width).to(DEV)
    lens = torch.full((900,), width * 16, dtype=torch.int32, device=DEV)
    free = torch.zeros(num + 9, dtype=torch.int32, device=DEV)
    before = table.clone()
    c = atflash.compact_pages(lens, table, 16, num, max_moves=num, free_pages=free)
    live = 900 * width
    to = torch.arange(num, device=DEV)
    n = int((c.src >= 0).sum())
    to[c.src[:n].long()] = c.dst[:n].long()
    assert torch.equal(to[before.long()], table.long())
    assert torch.equal(table.view(-1).sort().values.long(), torch.arange(live, device=DEV))
    assert c.free_head.tolist() == [live + 9] and torch.equal(free[live + 9:].long(), torch.arange(live, num, device=DEV))
    assert (c.src[:n] >= live).all() and (c.dst[:n] < live).all() and (c.src[n:] == -1).all() and (c.dst[n:] == -1).all()
    assert (c.src[:n].diff() < 0).all() and (c.dst[:n].diff() > 0).all()
    assert atflash.check_device_errors() == 0


def test_without_counts_and_with_rows_in_order():
    x = Mirror(40, 6, 6, 16)
    for r in range(6):
        x.m.take(r, r + 1)
    x.upload()
    import atflash
    lens = [16 * (r + 1) - 3 for r in range(6)]
    x.m.give_back([0, 1, 2], lens[:3], 16)
    x.head = atflash.free_requests(None, _i32(lens[:3]), x.table, 16, free_pages=x.free, free_head=x.head)
    x.same()


def test_what_a_fork_leaves_out_is_reported():
    x = Mirror(40, 8, 4, 16)
    x.m.take(0, 3)
    x.upload()
    # a child twice (the first counts), a child that is a parent, a row and lengths out of range
    x.fork([0, 0, 2, 0, 0, 9, 0], [2, 2, 3, 1, 4, 5, 8], [40, 20, 16, 65, -1, 16, 16])
    x.same(errors=2)
    assert x.m.rows[3] == [-1] * 4 and x.m.rows[4] == [-1] * 4 and x.m.rows[1] == [-1] * 4


def test_a_fork_with_too_short_a_free_list():
    import atflash
    x = Mirror(8, 6, 4, 16)
    x.m.take(0, 3)
    x.m.free, x.m.head = x.m.free[:5], 3
    x.upload()
    f = x.fork([0, 0, 0], [1, 2, 3], [40, 41, 42])
    assert f.dst.tolist()[2] == -1 and f.src.tolist()[2] == -1 and f.free_head.tolist() == [5]
    x.same(errors=2)
    # pages that a row should hold but does not, and ids outside the cache
    table = _i32([[3, -1, 99, -1], [-1] * 4])
    shared = _i32([0] * 8)
    atflash.fork_requests(_i32([0]), _i32([1]), _i32([48]), table, 16, free_pages=x.free, free_head=_i32([0]), shared=shared)
    assert atflash.check_device_errors() == 2
    assert table.tolist()[1] == [3, -1, 99, -1] and shared.tolist() == [0, 0, 0, 1, 0, 0, 0, 0]


def test_what_a_free_leaves_out_is_reported():
    import atflash
    x = Mirror(40, 8, 4, 16)
    for r in range(3):
        x.m.take(r, 3)
    x.upload()
    x.give_back([1, 1, 9, -1, 2], [48, 48, 16, 16, 65])
    x.same(errors=2)
    # a page in two rows without a count for it: freed once
    table, free, shared = _i32([[5, 6], [6, 7]]), _i32([0] * 10), _i32([0] * 10)
    head = atflash.free_requests(None, _i32([32, 32]), table, 16, free_pages=free, free_head=_i32([4]), shared=shared)
    assert atflash.check_device_errors() == 2
    assert head.tolist() == [1] and free.tolist() == [0, 5, 6, 7, 0, 0, 0, 0, 0, 0] and shared.tolist() == [0] * 10
    # ids outside the cache, and a list without room
    table = _i32([[5, -1], [77, 7]])
    head = atflash.free_requests(None, _i32([32, 32]), table, 16, free_pages=free, free_head=_i32([1]), shared=shared)
    assert atflash.check_device_errors() == 2
    assert head.tolist() == [0] and free.tolist()[0] == 7 and shared.tolist() == [0] * 10


def test_what_a_compaction_leaves_out_is_reported():
    import atflash
    table = _i32([[9, 8], [-1, 40], [3, 2]])
    free = _i32([0] * 10)
    c = atflash.compact_pages(_i32([32, 32, 40]), table, 16, 10, max_moves=10, free_pages=free)
    assert atflash.check_device_errors() == 2
    assert table.tolist() == [[0, 1], [-1, 40], [3, 2]]
    assert c.src.tolist() == [9, 8] + [-1] * 8 and c.dst.tolist() == [0, 1] + [-1] * 8
    assert c.free_head.tolist() == [2] and free.tolist() == [0, 0] + list(range(2, 10))


def test_rows_of_a_wider_table_and_nothing_to_do():
    import atflash
    wide = torch.full((6, 10), -7, dtype=torch.int32, device=DEV)
    table = wide[:, :4]
    table[0] = _i32([3, 1, 2, 0])
    shared, free = _i32([0] * 8), _i32(list(range(8)))
    f = atflash.fork_requests(_i32([0, 0]), _i32([2, 5]), _i32([64, 0]), table, 16, free_pages=free, free_head=_i32([4]),
                              shared=shared)
    assert f.src.tolist() == [-1, -1] and f.free_head.tolist() == [4]
    assert wide[2].tolist() == [3, 1, 2, 0] + [-7] * 6 and (wide[5] == -7).all() and shared.tolist() == [1] * 4 + [0] * 4
    h = atflash.free_requests(_i32([2]), _i32([64]), table, 16, free_pages=free, free_head=f.free_head, shared=shared)
    assert h.tolist() == [4] and wide[2].tolist() == [-1] * 4 + [-7] * 6 and shared.tolist() == [0] * 8
    c = atflash.compact_pages(_i32([64]), table, 16, 8, max_moves=0, free_pages=free, shared=shared)
    assert c.src.numel() == 0 and c.free_head.tolist() == [4] and free.tolist()[4:] == [4, 5, 6, 7]
    assert atflash.check_device_errors() == 0


# ------------------------------------------------------------------ copies

def _fill(shape, dtype, g):
    if dtype == torch.float8_e4m3fn:
        return torch.randint(0, 256, shape, generator=g, dtype=torch.int32).to(torch.uint8).to(DEV).view(dtype)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("pairs", [1, 9, 300])
@pytest.mark.parametrize("page,hkv", [(16, 4), (64, 1), (1, 1), (24, 3)])
def test_copies_in_every_kind_of_tensor(page, hkv, pairs):
    import atflash
    g = torch.Generator().manual_seed(page)
    P = 2 * pairs + 5
    odd = torch.zeros(P * 77 + 1, dtype=torch.uint8, device=DEV)
    caches = [_fill((P, page, hkv, 128), torch.bfloat16, g), _fill((P, hkv, 8, page, 16), torch.bfloat16, g),
              _fill((P, hkv, page, 128), torch.float8_e4m3fn, g), _fill((P, hkv), torch.float32, g),
              _fill((P, 2, page, hkv, 128), torch.bfloat16, g)[:, 1],                     # the V half of pages
              _fill((P, page, hkv, 128), torch.bfloat16, g).transpose(1, 2),             # axes in another order
              _fill((P, 3), torch.float32, g).t().contiguous().t()[:, :1],               # one element a page
              odd[1:].view(P, 77),                                                       # bytes without alignment
              _fill((P,), torch.float32, g)]
    odd[1:].copy_(torch.randint(0, 256, (P * 77,), generator=g, dtype=torch.int32).to(torch.uint8))
    whole = [c._base if c._base is not None else c for c in caches]
    before = [_bits(c).clone() for c in caches]
    base_before = [_bits(c).clone() for c in whole]
    perm = torch.randperm(P, generator=g).to(torch.int32)
    src, dst = perm[:pairs].clone(), perm[pairs:2 * pairs].clone()
    if pairs > 2:
        src[1] = src[0]        # one page to two places
        src[2] = dst[2] = -1   # no copy
        dst[3] = src[3]        # onto itself
    copier = atflash.PageCopier(caches)
    copier.copy(src.to(DEV), dst.to(DEV))
    for c, b in zip(caches, before):
        want = b.clone()
        for s, d in zip(src.tolist(), dst.tolist()):
            if s >= 0:
                want[d] = b[s]
        assert torch.equal(_bits(c), want)
    # nothing else of the allocations changed
    half = whole[4]
    assert torch.equal(half.view(P, 2, page, hkv, 128)[:, 0], base_before[4].view(P, 2, page, hkv, 128)[:, 0])
    assert odd[0] == 0
    assert atflash.check_device_errors() == 0


def test_copies_of_many_tensors_and_large_pages():
    import atflash
    g = torch.Generator().manual_seed(2)
    caches = [_fill((6, 5 + i % 3, 32), torch.bfloat16, g) for i in range(600)]  # three launches
    caches.append(_fill((6, 300001), torch.uint8, g))                           # pages of several pieces, odd size
    before = [c.clone() for c in caches]
    atflash.copy_pages(caches, torch.tensor([5, 0], device=DEV), torch.tensor([2, 3], device=DEV))
    for c, b in zip(caches, before):
        b[2], b[3] = b[5], b[0]
        assert torch.equal(c, b)


def test_copies_past_two_gigabytes():
    import atflash
    P, page = 1100, 1 << 22  # 4.6 GB: byte offsets over 32 bits
    cache = torch.empty((P, page), dtype=torch.uint8, device=DEV)
    cache[0], cache[1099], cache[1050] = 7, 9, 0
    atflash.copy_pages([cache], _i32([1099, 0]), _i32([600, 1050]))
    assert (cache[600] == 9).all() and (cache[1050] == 7).all()


def test_copy_reports_ids_outside_the_cache():
    import atflash
    c = torch.arange(8, dtype=torch.float32, device=DEV).view(4, 2).clone()
    atflash.copy_pages([c], _i32([0, 4, -1, 1, -1]), _i32([2, 1, 3, -2, -1]))
    assert atflash.check_device_errors() == 2
    assert c.tolist() == [[0, 1], [2, 3], [0, 1], [6, 7]]
    atflash.copy_pages([c], _i32([]), _i32([]))
    assert atflash.check_device_errors() == 0


def test_refusals():
    import atflash
    i, t = _i32([0]), _i32([[0, 1]])
    s, f = _i32([0] * 4), _i32([0] * 4)
    fork = dict(parents=i, children=i, kv_lens=i, req_pages=t, page_size=16, free_pages=f, free_head=i, shared=s)
    for bad in (dict(children=_i32([0, 1])), dict(kv_lens=i.float()), dict(req_pages=t[0]), dict(req_pages=t.long()),
                dict(req_pages=_i32([[0, 1], [2, 3]]).t()), dict(req_pages=t.expand(3, 2)), dict(page_size=0), dict(free_head=f),
                dict(shared=s.long()), dict(shared=s[::2]), dict(parents=i[:0], children=i[:0], kv_lens=i[:0]),
                dict(req_pages=t[:, :0]), dict(parents=i.cpu())):
        with pytest.raises(ValueError):
            atflash.fork_requests(**{**fork, **bad})
    free = dict(req_rows=i, kv_lens=i, req_pages=t, page_size=16, free_pages=f, free_head=i, shared=s)
    for bad in (dict(free_pages=f.long()), dict(free_pages=f[::2]), dict(req_rows=None, kv_lens=_i32([1, 1])),
                dict(req_rows=_i32([0, 0])), dict(shared=s.cpu()), dict(shared=s.view(2, 2))):
        with pytest.raises(ValueError):
            atflash.free_requests(**{**free, **bad})
    comp = dict(kv_lens=i, req_pages=t, page_size=16, num_pages=4, max_moves=2, free_pages=f)
    for bad in (dict(num_pages=0), dict(num_pages=5), dict(max_moves=-1), dict(max_moves=5), dict(shared=s[:2]),
                dict(num_pages=(1 << 20) + 1, free_pages=torch.zeros((1 << 20) + 1, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            atflash.compact_pages(**{**comp, **bad})
    c = torch.zeros((4, 2, 2), device=DEV)
    for bad in ([], [c, c[:3]], [c[:, :, :1]], [c[:, :1].expand(4, 2, 2)], [c[:1].expand(4, 2, 2)], [c[:0]], [c[0, 0, 0]],
                [c, c.cpu()]):
        with pytest.raises(ValueError):
            atflash.PageCopier(bad)
    with pytest.raises(ValueError):
        atflash.PageCopier([c]).copy(i, _i32([0, 1]))


def test_replayed_graph_follows_its_tensors_on_another_stream():
    import atflash
    x = Mirror(40, 8, 6, 16)
    for r in range(3):
        x.m.take(r, 5)
    x.upload()
    cache = torch.randn((40, 16, 2, 128), device=DEV).bfloat16()
    copier = atflash.PageCopier([cache])
    parents, kids, lens = _i32([0, 1]), _i32([4, 5]), _i32([70, 64])
    head = x.head
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    atflash.check_device_errors()
    with torch.cuda.graph(graph, stream=s):
        f = atflash.fork_requests(parents, kids, lens, x.table, 16, free_pages=x.free, free_head=head, shared=x.shared)
        copier.copy(f.src, f.dst)
        back = atflash.free_requests(kids, lens, x.table, 16, free_pages=x.free, free_head=f.free_head, shared=x.shared)
    for p, n in (([0, 1], [70, 64]), ([2, 2], [33, 80]), ([1, 0], [0, 1])):
        parents.copy_(_i32(p))
        lens.copy_(_i32(n))
        was = cache.clone()
        graph.replay()
        src, dst = x.m.fork(p, [4, 5], n, 16)
        assert (f.src.tolist(), f.dst.tolist()) == (src, dst)
        for a, b in zip(src, dst):
            if a >= 0:
                was[b] = was[a]
        assert torch.equal(cache, was)
        x.m.give_back([4, 5], n, 16)
        assert back.tolist() == [x.m.head]
        assert x.table.tolist() == x.m.rows and x.shared.tolist() == x.m.shared and x.free.tolist() == x.m.free
    assert atflash.check_device_errors() == 0
