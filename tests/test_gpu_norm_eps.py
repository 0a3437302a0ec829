"""An eps that fp32 does not hold is refused by the Python calls of the norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("eps", [0.0, -1e-6, 1e39, float("inf"), float("nan"), 1e-50])
def test_refused(eps):
    import atflash
    x, w, c = torch.ones((1, 1, 128), dtype=torch.bfloat16, device=DEV), torch.ones(128, device=DEV), torch.ones((1, 64), device=DEV)
    i, pages = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros((1, 16, 1, 128), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="eps"):
        atflash.qk_norm_rope(x, None, w, None, c, c, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        atflash.append_paged_kv_cache(x, x, i, i, (pages, pages), i, torch.arange(2, dtype=torch.int32, device=DEV),
                                      rope=(c, c), k_norm=(w, eps))
