"""Attention of chunks over pages on a B200 against a 64-bit restatement: single tokens,
drafts and chunks, ragged and empty requests, page sizes and layouts, heads side by side,
keys shared out over SMs, windows, what lies behind the last key, plans, streams, graphs."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WS = 64 << 20
# level limits that drop terms within these lengths
ZHI = (1 << 30, 1500, 900, 500, 260, 130, 60, 20)


class Case:
    def __init__(self, page, layout, hq, hkv, reqs, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.page, self.layout, self.hq, self.hkv, self.reqs = page, layout, hq, hkv, reqs
        npg = [-(-nk // page) for _, nk in reqs]
        total = sum(npg) + spare
        perm = torch.randperm(total, generator=g).to(torch.int32)
        self.cq = [0] + np.cumsum([nq for nq, _ in reqs]).tolist()
        self.starts = [0] + np.cumsum(npg).tolist()
        self.indices = perm[:sum(npg)].contiguous()
        self.last = [(nk - 1) % page + 1 if nk else 0 for _, nk in reqs]
        shape = (total, page, hkv, 128) if layout == "NHD" else (total, hkv, page, 128)
        # what no request holds is NaN: rows behind the last key and pages of nobody
        self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.q = torch.randn((self.cq[-1], hq, 128), generator=g).bfloat16().to(DEV)
        self.rows = []
        for b, (_, nk) in enumerate(reqs):
            ids = self.indices[self.starts[b]:self.starts[b + 1]].long().to(DEV)
            kv = []
            for c in (self.k, self.v):
                x = torch.randn((nk, hkv, 128), generator=g).bfloat16().to(DEV)
                pos = torch.arange(nk, device=DEV)
                view = c if layout == "NHD" else c.transpose(1, 2)
                view[ids[pos // page], pos % page] = x
                kv.append(x)
            self.rows.append(kv)

    def plan(self, causal=True, zhi=None, ws=WS, **kw):
        import atflash
        w = atflash.BatchPrefillWithPagedKVCacheWrapper(torch.empty(ws, dtype=torch.uint8, device=DEV), self.layout)
        w.plan(self.cq, self.starts, self.indices.to(DEV), self.last, self.hq, self.hkv, 128, self.page, causal=causal,
               window_table=zhi, **kw)
        return w

    def check(self, out, lse, causal=True, zhi=None, scale=1 / math.sqrt(128), requests=None):
        """P has bf16's half step (2^-8) and the result another; scores are sums of 128 fp32
        products, so off by at most 128 x 2^-24 of the terms' sizes (under 180 here), which is
        2^-13 after the scale, in P and in the lse alike."""
        g = self.hq // self.hkv
        for b, (nq, nk) in enumerate(self.reqs):
            if requests is not None and b not in requests:
                continue
            o, s_lse = out[self.cq[b]:self.cq[b + 1]].double(), lse[self.cq[b]:self.cq[b + 1]].double()
            if nk == 0:
                assert (o == 0).all() and (s_lse == -math.inf).all()
                continue
            k, v = (x.double() for x in self.rows[b])
            row, col = torch.arange(nq, device=DEV)[:, None], torch.arange(nk, device=DEV)[None]
            near = nk - nq + row // 128 * 128 - (col // 128 * 128 + 127)
            for h in range(self.hq):
                q, kh, vh = self.q[self.cq[b]:self.cq[b + 1], h].double(), k[:, h // g], v[:, h // g]
                score = q[:, :16] @ kh[:, :16].T if zhi else q @ kh.T
                for i in range(1, 8 if zhi else 1):
                    d = slice(16 * i, 16 * i + 16)
                    score += (q[:, d] @ kh[:, d].T) * (near <= zhi[i])
                score *= scale
                if causal:
                    score.masked_fill_(col > row + nk - nq, -math.inf)
                want_lse = torch.logsumexp(score, -1)
                p = torch.exp(score - torch.where(want_lse == -math.inf, 0.0, want_lse)[:, None])
                want, size = p @ vh, p @ vh.abs()
                tol = size * (2.0 ** -8 + 2.0 ** -12) + want.abs() * 2.0 ** -8 + 1e-6
                err = (o[:, h] - want).abs()
                assert (err <= tol).all(), (b, h, (err - tol).max().item())
                dead = want_lse == -math.inf
                assert torch.equal(s_lse[:, h] == -math.inf, dead)
                assert ((s_lse[:, h] - want_lse).abs()[~dead] <= 2e-4).all()

    def run(self, w, **kw):
        return w.run(self.q, (self.k, self.v), return_lse=True, **kw)


CASES = [
    # page, layout, hq, hkv, (new tokens, keys) of each request
    (16, "NHD", 1, 1, [(1, 1)]),
    (16, "NHD", 7, 1, [(1, 17), (5, 5), (2, 300)]),
    (16, "NHD", 28, 4, [(1, 700), (4, 129), (18, 400), (19, 40)]),
    (64, "HND", 24, 8, [(130, 130), (1, 513), (300, 1100), (42, 42), (43, 1000)]),
    (32, "NHD", 12, 1, [(10, 2000), (11, 2001)]),
    (128, "HND", 16, 1, [(8, 128), (9, 129), (128, 256)]),
    (256, "NHD", 4, 2, [(64, 600), (65, 255), (257, 257), (1, 1)]),
    (16, "HND", 3, 3, [(128, 128), (129, 300), (256, 256), (384, 500)]),          # a group of one
    (16, "NHD", 8, 1, [(0, 50), (3, 0), (0, 0), (7, 1), (20, 12), (1, 2)]),       # empty; more tokens than keys
    (64, "NHD", 140, 1, [(2, 100), (130, 400)]),                                  # a group that no tile holds
    (16, "NHD", 6, 2, [(700, 1900), (40, 40)]),
]


@pytest.mark.parametrize("zhi", [None, ZHI])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,layout,hq,hkv,reqs", CASES)
def test_matches_the_definition(page, layout, hq, hkv, reqs, causal, zhi):
    import atflash
    c = Case(page, layout, hq, hkv, reqs, seed=page + hq)
    out, lse = c.run(c.plan(causal, zhi))
    c.check(out, lse, causal, zhi)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("page,hq,hkv,reqs", [
    (16, 7, 1, [(1, 40011)]),
    (16, 28, 4, [(5, 16001), (1, 9000), (3, 12345)]),
    (64, 3, 3, [(256, 9000)]),
    (16, 4, 4, [(200, 9000), (1, 7)]),
    (128, 16, 2, [(100, 20000)]),
])
def test_keys_shared_out_over_the_sms(page, hq, hkv, reqs):
    import atflash
    c = Case(page, "NHD", hq, hkv, reqs, seed=page)
    w = c.plan()
    assert w._plan.num_parts > 0
    out, lse = c.run(w)
    c.check(out, lse)
    again, lse2 = c.run(w)  # in one order of sums
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert atflash.check_device_errors() == 0


def test_whole_blocks_equal_the_packed_prefill_bit_for_bit():
    import atflash
    for zhi in (None, ZHI):
        c = Case(16, "NHD", 32, 16, [(512, 1100), (512, 512), (768, 901), (256, 2000)], seed=9)
        w = c.plan(zhi=zhi)
        assert w._plan.num_parts == 0 and w._plan.num_wide == w._plan.num_items
        out, lse = c.run(w)
        k, v = (torch.cat([r[i] for r in c.rows]) for i in range(2))
        r = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
        r.plan(c.cq, [0] + np.cumsum([nk for _, nk in c.reqs]).tolist(), 32, 16, causal=True, window_table=zhi)
        want, want_lse = r.run(c.q, k, v, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_equals_the_decode_within_its_rounding():
    import atflash
    c = Case(16, "NHD", 24, 8, [(1, n) for n in (1, 100, 3000, 777)], seed=4)
    out, lse = c.run(c.plan())
    d = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(WS, dtype=torch.uint8, device=DEV), "NHD")
    d.plan(c.starts, c.indices.to(DEV), c.last, 24, 8, 128, 16)
    k, v = (torch.nan_to_num(x) for x in (c.k, c.v))
    want, want_lse = d.run(c.q, (k, v), return_lse=True)
    c.check(want, want_lse)
    assert (lse - want_lse).abs().max() < 4e-4


def test_strides_scale_outputs_and_one_cache_tensor():
    import atflash
    c = Case(16, "NHD", 6, 2, [(3, 100), (140, 333)], seed=2)
    both = torch.stack([c.k, c.v], dim=1)  # (P, 2, page, Hkv, 128)
    wide = torch.zeros((c.cq[-1], 10, 128), dtype=torch.bfloat16, device=DEV)
    wide[:, 2:8] = c.q
    buf = torch.full((c.cq[-1] + 4, 9, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((c.cq[-1], 6), device=DEV)
    w = c.plan(sm_scale=0.2)
    got = w.run(wide[:, 2:8], both, out=buf[2:-2, 1:7], lse=lse)
    assert got.data_ptr() == buf[2:-2, 1:7].data_ptr()
    c.check(got, lse, scale=0.2)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[2:-2, 1:7] = False
    assert (buf[keep] == 5.0).all()
    assert atflash.check_device_errors() == 0


def test_rotate_half_order_without_a_window():
    c = Case(16, "NHD", 4, 2, [(3, 100)], seed=2)
    out, lse = c.run(c.plan(qk_layout="rotate_half"))
    c.check(out, lse)


def test_a_bad_page_costs_its_own_request_only():
    import atflash
    c = Case(16, "NHD", 8, 2, [(4, 500), (4, 500), (200, 300), (4, 90)], seed=6)
    c.indices = c.indices.clone()
    c.indices[c.starts[1] + 3] = c.k.shape[0]
    c.indices[c.starts[2] + 1] = -7
    out, lse = c.run(c.plan())
    assert atflash.check_device_errors() == 2
    c.check(out, lse, requests=(0, 3))
    assert atflash.check_device_errors() == 0


def test_nan_and_infinity_of_a_key_stay_with_the_rows_that_see_it():
    c = Case(16, "NHD", 2, 2, [(130, 130), (4, 300)], seed=8)
    c.check(*c.run(c.plan()))
    ids = c.indices[c.starts[1]:c.starts[2]].long()
    c.v[ids[299 // 16], 299 % 16] = float("inf")  # key 299: the last row's alone, in a tile that all rows load
    out, lse = c.run(c.plan())
    c.check(out, lse, requests=(0,))
    assert torch.isfinite(lse).all() and not torch.isfinite(out[c.cq[2] - 1]).any()


@pytest.mark.parametrize("reqs", [[(1, 1)], [(2, 2), (1, 129)], [(128, 128)], [(256, 256)]])
def test_a_nan_key_reaches_every_row_that_sees_it(reqs):
    """Each request's first key is NaN: no row may pass it over, the one that sees nothing
    else included."""
    c = Case(16, "NHD", 2, 1, reqs, seed=8)
    for b in range(len(reqs)):
        c.k[c.indices[c.starts[b]].long(), 0] = float("nan")
    out, lse = c.run(c.plan())
    assert out.isnan().all() and lse.isnan().all()


def test_plans_kept_dropped_and_small_workspaces():
    import atflash
    c = Case(16, "NHD", 28, 4, [(5, 16001)], seed=1)
    w = c.plan()
    need = 4 * 128 * w._plan.num_parts * 28
    with pytest.raises(ValueError, match="workspace too small"):
        c.plan(ws=need)
    first = c.run(w)
    # a plan dropped while its run is pending on another stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)
        got = c.run(w)
    w.plan([0, 1], [0, 1], [0], [1], 28, 4, 128, 16)
    torch.empty(1 << 20, dtype=torch.int32, device=DEV).fill_(-1)
    torch.cuda.synchronize()
    assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    assert atflash.check_device_errors() == 0


def test_captured_and_replayed():
    c = Case(16, "NHD", 28, 4, [(5, 9001), (300, 900)], seed=3)
    w = c.plan()
    want = c.run(w)
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(c.q, (c.k, c.v), out=out, lse=lse)
    graph.replay()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    c.q.mul_(0.5)
    want = c.run(w)
    graph.replay()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_cache_past_two_gigabytes():
    import atflash
    page, hkv = 16, 8
    pages = 150_000  # 4.9 GB of K
    k = torch.zeros((pages, page, hkv, 128), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    c = Case(page, "NHD", 16, hkv, [(3, 100), (130, 700)], seed=5)
    far = torch.arange(pages - 1, pages - 1 - c.k.shape[0], -1, device=DEV)
    k[far], v[far] = c.k, c.v
    w = c.plan()
    w.plan(c.cq, c.starts, far[c.indices.long().to(DEV)], c.last, 16, hkv, 128, page)
    out, lse = w.run(c.q, (k, v), return_lse=True)
    c.check(out, lse)
    assert atflash.check_device_errors() == 0


def test_refusals():
    import atflash
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):
        atflash.BatchPrefillWithPagedKVCacheWrapper(torch.empty(16), "NHD")
    with pytest.raises(ValueError):
        atflash.BatchPrefillWithPagedKVCacheWrapper(ws, "PHD")
    w = atflash.BatchPrefillWithPagedKVCacheWrapper(ws)
    with pytest.raises(RuntimeError, match="plan"):
        w.run(ws, (ws, ws))
    ok = dict(qo_indptr=[0, 2], paged_kv_indptr=[0, 2], paged_kv_indices=[1, 0], paged_kv_last_page_len=[5], num_qo_heads=4,
              num_kv_heads=2, head_dim=128, page_size=16)
    for bad in (dict(head_dim=64), dict(page_size=24), dict(window_table=ZHI, qk_layout="rotate_half")):
        with pytest.raises(NotImplementedError):
            w.plan(**{**ok, **bad})
    for bad in (dict(num_qo_heads=3), dict(qk_layout="x"), dict(qo_indptr=[0, 2, 3]), dict(qo_indptr=[1, 2]),
                dict(paged_kv_indptr=[0, -1]), dict(paged_kv_last_page_len=[17]), dict(paged_kv_last_page_len=[0]),
                dict(paged_kv_last_page_len=[5, 5]), dict(paged_kv_indices=[1]), dict(paged_kv_indices=torch.zeros(2, 1)),
                dict(sm_scale=0.0), dict(sm_scale=float("inf")), dict(window_table=(5,) * 7), dict(window_table=(9, 1, 2, 0, 0, 0, 0, 0))):
        with pytest.raises(ValueError):
            w.plan(**{**ok, **bad})
    w.plan(**ok)
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV)
    c = torch.zeros((3, 16, 2, 128), dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=q[:1]), dict(q=q[:, :2]), dict(cache=(c, c[:2])), dict(cache=(c[:, :8], c[:, :8])),
                dict(cache=(c[:0], c[:0])), dict(cache=(c.transpose(1, 2), c.transpose(1, 2))), dict(out=q.float()),
                dict(lse=torch.zeros((2, 4))), dict(cache=(c.cpu(), c.cpu())), dict(lse=torch.zeros((4, 2), device=DEV).t())):
        with pytest.raises(ValueError):
            w.run(bad.get("q", q), bad.get("cache", (c, c)), out=bad.get("out"), lse=bad.get("lse"))
    for bad in (dict(q=q.float()), dict(cache=(c, c.float())), dict(cache=(c.to(torch.float8_e4m3fn),) * 2)):
        with pytest.raises(TypeError):
            w.run(bad.get("q", q), bad.get("cache", (c, c)))
    odd = torch.zeros(2 * 4 * 128 + 4, dtype=torch.bfloat16, device=DEV)[4:].view(2, 4, 128)
    with pytest.raises(atflash.AtfError, match="aligned"):
        w.run(odd, (c, c))
    w.run(q, (c, c))


def test_an_expanded_output_is_refused():
    import atflash
    w = atflash.BatchPrefillWithPagedKVCacheWrapper(torch.empty(1 << 20, dtype=torch.uint8, device=DEV))
    w.plan([0, 2], [0, 1], [0], [5], 4, 2, 128, 16)
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV)
    c = torch.zeros((1, 16, 2, 128), dtype=torch.bfloat16, device=DEV)
    for out in (q[:1].expand(2, 4, 128), q[:, :1].expand(2, 4, 128)):
        with pytest.raises(ValueError, match="expanded"):
            w.run(q, (c, c), out=out)
