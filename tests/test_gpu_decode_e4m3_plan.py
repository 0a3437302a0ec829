"""A plan for an e4m3 cache refuses what its run would refuse."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Z16 = [1 << 28, 777, 300, 150, 64, 33, 17, 0]


@pytest.mark.parametrize("kw", [dict(page_size=24), dict(page_size=8), dict(page_size=512),
                                dict(window_table=[1 << 20] * 16, window_mode="vec8"),
                                dict(window_table=Z16, qk_layout="rotate_half")])
def test_a_plan_refuses_what_its_run_cannot_read(kw):
    import atflash
    w = atflash.BatchDecodeWithPagedKVCacheWrapper(torch.empty(16 << 20, dtype=torch.uint8, device=DEV), "NHD")
    a = dict(indptr=[0, 1], indices=[0], last_page_len=[5], num_qo_heads=4, num_kv_heads=2, head_dim=128, page_size=16)
    for dtype in (torch.float8_e4m3fn, "float8_e4m3fn"):
        w.plan(**a, kv_data_type=dtype)
        with pytest.raises(NotImplementedError):
            w.plan(**{**a, **kw}, kv_data_type=dtype)
    w.plan(**{**a, **kw})  # a bf16 cache takes them all
