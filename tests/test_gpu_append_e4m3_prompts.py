"""The e4m3 append with RoPE at prompt sizes, byte for byte: windows of 32 tokens per CTA
whose angles are staged once for all heads, runs that go on past a window, several warps
to a page, either layout and pair order."""
import numpy as np
import pytest
import torch

import _e4m3
from _inputs import rope_tables
from test_gpu_append_e4m3 import DEV, _append, _check, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,hkv,lens,app", [
    (16, 2, [2500, 37, 2477, 500], [2500, 1, 2470, 31]),
    (64, 3, [3001, 1999, 130], [3001, 1990, 3]),     # four warps to a page, runs past a window
    (256, 1, [2600, 2400], [2590, 2399]),            # eight warps, rows read twice
    (24, 2, [5000], [4999]),                         # pages that end inside a window
])
@pytest.mark.parametrize("layout,out_layout", [("NHD", "rotate_half"), ("HND", "sorted_pair"), ("HND", "rotate_half"),
                                               ("NHD", "sorted_pair")])
def test_append_e4m3_prompts_with_rope(page, hkv, lens, app, layout, out_layout):
    import atflash
    assert sum(app) > 148 * 32  # a window of 32 tokens for each CTA
    cache, k, v, bidx, pos, indptr, indices = _setup(layout, page, hkv, lens, app, page, factor=2)
    cos, sin = rope_tables(max(lens) + 5, 128, 1e6)
    rope = (cos.to(DEV), sin.to(DEV))
    packed = atflash.rope_pack(k.to(DEV)[None], *rope, positions=pos.long().to(DEV), out_layout=out_layout)
    want = _e4m3.append(*cache, packed[0].cpu(), v, bidx, pos, indptr, indices, layout)
    _check(_append(cache, k, v, bidx, pos, indptr, indices, layout, rope=rope, out_layout=out_layout), want)
    assert atflash.check_device_errors() == 0


def test_append_e4m3_prompts_with_other_rope_positions():
    """Positions of their own, past the tables' end too (the last row counts there)."""
    import atflash
    cache, k, v, bidx, pos, indptr, indices = _setup("HND", 32, 2, [5000], [4990], 3, factor=2)
    cos, sin = rope_tables(4096, 128, 1e4)
    rope = (cos.to(DEV), sin.to(DEV))
    rp = torch.from_numpy(np.random.default_rng(1).permutation(len(pos)) - 3)
    packed = atflash.rope_pack(k.to(DEV)[None], *rope, positions=rp.clamp(0, 4095).to(DEV), out_layout="sorted_pair")
    want = _e4m3.append(*cache, packed[0].cpu(), v, bidx, pos, indptr, indices, "HND")
    _check(_append(cache, k, v, bidx, pos, indptr, indices, "HND", rope=rope, rope_positions=rp.to(DEV)), want)
    assert atflash.check_device_errors() == 0
