"""Index reports (a free list that ran out, lengths that do not fit, bad pages) are read
at the caller's leisure: attention runs on meanwhile. A wait that expired does stop it."""
import numpy as np
import pytest
import torch

import _e4m3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls():
    """name -> call(out) of every attention entry point, with its output's shape."""
    import atflash
    g = torch.Generator().manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=g).bfloat16().to(DEV)
    q, k, v = rand(1, 300, 4, 128), rand(1, 300, 2, 128), rand(1, 300, 2, 128)
    packed = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
    packed.plan([0, 100, 300], [0, 100, 300], 4, 2, 128)
    lens, page = [70, 200, 16], 16
    npg = [-(-n // page) for n in lens]
    cache = [t.to(DEV) for t in _e4m3.random_cache(sum(npg), page, 2, "NHD", g)]
    bf = [(cache[i].float() * cache[i + 1][:, None, :, None]).bfloat16() for i in (0, 2)]
    qd = rand(3, 6, 128)
    calls = {"prefill": (lambda out: atflash.prefill_fwd(q, k, v, out=out), q.shape),
             "packed": (lambda out: packed.run(q[0], k[0], v[0], out=out), q.shape[1:])}
    for name, dtype in (("decode", None), ("decode_e4m3", torch.float8_e4m3fn)):
        w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.zeros(16 << 20, dtype=torch.uint8, device=DEV), "NHD")
        w.plan(np.concatenate([[0], np.cumsum(npg)]), torch.arange(sum(npg), dtype=torch.int32),
               [(n - 1) % page + 1 for n in lens], 6, 2, 128, page, kv_data_type=dtype)
        kw = dict(kv_scales=(cache[1], cache[3])) if dtype else {}
        calls[name] = (lambda out, w=w, kv=(cache[0], cache[2]) if dtype else tuple(bf), kw=kw: w.run(qd, kv, out=out, **kw),
                       qd.shape)
    return calls


def _run(calls):
    outs = {}
    for name, (call, shape) in calls.items():
        outs[name] = torch.full(shape, 7.0, dtype=torch.bfloat16, device=DEV)
        call(outs[name])
    torch.cuda.synchronize()
    return outs


def _exhausted_free_list():
    import atflash
    i32 = dict(dtype=torch.int32, device=DEV)
    r = atflash.build_page_tables(torch.full((2,), 40, **i32), torch.full((2,), 40, **i32), torch.full((2, 3), -1, **i32), 16,
                                  num_tokens=80, max_pages=6, free_pages=torch.arange(4, **i32), free_head=torch.zeros(1, **i32))
    assert r.indices.tolist() == [0, 1, 2, 3, -1, -1]


def _append_to_a_bad_page():
    import atflash
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = torch.zeros((1, 1, 128), dtype=torch.bfloat16, device=DEV)
    c = torch.zeros((2, 16, 1, 128), dtype=torch.bfloat16, device=DEV)
    atflash.append_paged_kv_cache(k, k, z, z, (c, c.clone()), z + 9, torch.tensor([0, 1], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("report", [_exhausted_free_list, _append_to_a_bad_page])
def test_attention_runs_on_after_an_index_report(report):
    import atflash
    calls = _calls()
    want = _run(calls)
    assert atflash.check_device_errors() == 0
    report()
    got = _run(calls)
    assert atflash.check_device_errors() == 2
    for name in calls:
        assert torch.equal(got[name], want[name]), name


def test_decode_e4m3_with_a_bad_page_keeps_the_other_requests():
    import atflash
    g = torch.Generator().manual_seed(6)
    lens, page = [100, 500, 64, 300], 16
    npg = [-(-n // page) for n in lens]
    cache = [t.to(DEV) for t in _e4m3.random_cache(sum(npg), page, 2, "NHD", g)]
    q = torch.randn((4, 6, 128), generator=g).bfloat16().to(DEV)
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.zeros(16 << 20, dtype=torch.uint8, device=DEV), "NHD")
    indptr, ids = np.concatenate([[0], np.cumsum(npg)]), torch.arange(sum(npg), dtype=torch.int32)

    def run():
        w.plan(indptr, ids, [(n - 1) % page + 1 for n in lens], 6, 2, 128, page, kv_data_type=torch.float8_e4m3fn)
        return w.run(q, (cache[0], cache[2]), kv_scales=(cache[1], cache[3]))
    want = run()
    assert atflash.check_device_errors() == 0
    ids[int(indptr[1]) + 3] = -1
    got = run()
    assert atflash.check_device_errors() == 2
    for b in (0, 2, 3):
        assert torch.equal(got[b], want[b])


def test_an_expired_wait_stops_attention_until_it_is_read():
    import atflash
    from atflash import _runtime
    calls = _calls()
    want = _run(calls)
    flag = _runtime.error_flag(torch.device(DEV))
    flag.fill_(1)
    got = _run({n: c for n, c in calls.items() if n in ("prefill", "packed")})
    assert all(torch.all(x == 7) for x in got.values())
    assert atflash.check_device_errors() == 1
    flag.fill_(2)  # an index report, then a wait that expires: the wait is what is read
    assert _runtime.selftest_wait_timeout(torch.device(DEV)) == 1
    got = _run(calls)
    assert atflash.check_device_errors() == 0 and all(torch.equal(got[n], want[n]) for n in calls)


def test_a_new_flag_is_clear_for_every_stream(monkeypatch):
    """The flag's first value is there before a kernel on another stream can read it."""
    from atflash import _runtime
    monkeypatch.setattr(_runtime, "_flags", {})
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)
    flag = _runtime.error_flag(torch.device(DEV))
    assert torch.cuda.current_stream().query()  # the fill has run, not only been queued
    assert flag.item() == 0
