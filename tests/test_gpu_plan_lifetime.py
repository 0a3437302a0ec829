"""A plan on one stream, a run on another that is still busy, a new plan at once: the
old plan's tensors stay until the run has read them. And a schedule that names a
request outside the batch is reported, not followed."""
import numpy as np
import pytest
import torch

import _e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _late(run, replan, held):
    """run() behind a long wait on a stream of its own, then replan() at once and new
    tensors of the old plan's sizes: none may take the old ones' memory."""
    old = [(t.data_ptr(), t.numel(), t.dtype) for t in held()]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(1_000_000_000)
        got = run()
    replan()
    new = [torch.full((n,), 1 << 20, dtype=dt, device=DEV) for _, n, dt in old for _ in range(64)]
    taken = {t.data_ptr() for t in new} & {p for p, _, _ in old}
    assert not st.query()  # the run had not begun when the new tensors were made
    st.synchronize()
    assert not taken
    return got


def test_packed_prefill_replanned_while_a_run_is_pending():
    import atflash
    g = torch.Generator(device=DEV).manual_seed(1)
    nq = [200, 33, 129, 300]
    q = torch.randn((sum(nq), 4, 128), generator=g, device=DEV).bfloat16()
    k, v = (torch.randn((sum(nq), 2, 128), generator=g, device=DEV).bfloat16() for _ in range(2))
    cq = np.concatenate([[0], np.cumsum(nq)])
    w = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
    w.plan(cq, cq, 4, 2, 128)
    want, out = w.run(q, k, v), torch.zeros_like(q)
    other = np.concatenate([[0], np.cumsum(nq[::-1])])
    w.plan(cq, cq, 4, 2, 128)
    _late(lambda: w.run(q, k, v, out=out), lambda: w.plan(other, other, 4, 2, 128), lambda: [w._items])
    assert torch.equal(out, want)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("e4m3", [True, False])
def test_decode_replanned_while_a_run_is_pending(e4m3):
    import atflash
    g = torch.Generator().manual_seed(2)
    page, hkv, lens = 16, 2, [300, 90, 411, 700]
    npg = [-(-n // page) for n in lens]
    indices = torch.randperm(sum(npg) + 3, generator=g).to(torch.int32)[:sum(npg)].contiguous()
    indptr = torch.tensor([0] + list(np.cumsum(npg)), dtype=torch.int32)
    last = torch.tensor([(n - 1) % page + 1 for n in lens], dtype=torch.int32)
    cache = [t.to(DEV) for t in _e4m3.random_cache(sum(npg) + 3, page, hkv, "NHD", g)]
    q = torch.randn((4, 6, 128), generator=g).bfloat16().to(DEV)
    kv, kw = (cache[0], cache[2]), dict(kv_scales=(cache[1], cache[3]))
    if not e4m3:
        kv, kw = tuple((cache[i].float() * cache[i + 1][:, None, :, None]).bfloat16() for i in (0, 2)), {}
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV), "NHD")

    def plan(flip=False):
        w.plan(indptr, indices.flip(0) if flip else indices, last, 6, hkv, 128, page,
               kv_data_type=torch.float8_e4m3fn if e4m3 else None)
    plan()
    want, out = w.run(q, kv, **kw), torch.zeros_like(q)
    plan()
    names = ("items", "item_indptr", "indptr", "indices", "last_page_len")
    _late(lambda: w.run(q, kv, out=out, **kw), lambda: plan(True), lambda: [w._plan[n] for n in names])
    assert torch.equal(out, want)
    assert atflash.check_device_errors() == 0


@pytest.mark.parametrize("request_index", [4, -1, 2 ** 31 - 1, -2 ** 31])
def test_decode_e4m3_schedule_of_another_batch_is_reported(request_index):
    import atflash
    g = torch.Generator().manual_seed(3)
    cache = [t.to(DEV) for t in _e4m3.random_cache(8, 16, 1, "NHD", g)]
    q = torch.randn((4, 2, 128), generator=g).bfloat16().to(DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(16 << 20, dtype=torch.uint8, device=DEV), "NHD")
    one = torch.ones(4, dtype=torch.int32)
    w.plan(torch.arange(5, dtype=torch.int32), torch.arange(4, dtype=torch.int32), one * 16, 2, 1, 128, 16,
           kv_data_type=torch.float8_e4m3fn)
    w._plan["items"][1, 0] = request_index
    w.run(q, (cache[0], cache[2]), kv_scales=(cache[1], cache[3]))
    assert atflash.check_device_errors() == 2
