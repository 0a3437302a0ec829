"""The example's serving loop on a B200 against plain attention in 64 bits: prompts,
then steps whose keys and values are those that the cache holds."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rope_sorted(x, cos, sin):
    """HF halves rotated at the rows' positions, widest pair first, bf16."""
    a, b = x.float().split(64, dim=-1)
    c, s = cos[:, None], sin[:, None]
    r = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flip(-2)
    return r.reshape(x.shape).bfloat16()


@pytest.mark.parametrize("lens,steps", [([1], 3), ([40, 17, 300, 16, 1], 20)])
def test_serving_loop(lens, steps):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import serving_step as ex
    import atflash
    hq, hkv, page = 12, 4, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    prompts = [torch.randn((n, 256), generator=g, device="cuda").bfloat16() for n in lens]
    prompt_out, outs, st = ex.serve(prompts, steps, hq=hq, hkv=hkv, page=page)
    assert atflash.check_device_errors() == 0
    layer, cos, sin = st["layer"], st["cos"], st["sin"]
    t = st["tables"]
    ids, ptr = t.indices.long(), t.indptr.tolist()
    assert st["kv_lens"].tolist() == [n + steps for n in lens]
    assert sorted(ids.tolist()) == sorted(set(ids.tolist()))  # no page twice
    at = 0
    for b, n in enumerate(lens):
        q, k, v = (z for z in layer.qkv(prompts[b]))
        qr, kr = _rope_sorted(q, cos[:n], sin[:n]).double(), _rope_sorted(k, cos[:n], sin[:n]).double()
        s = torch.einsum("qhd,khd->hqk", qr, kr.repeat_interleave(hq // hkv, 1)) / math.sqrt(128)
        p = torch.softmax(s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf), -1)
        vv = v.double().repeat_interleave(hq // hkv, 1)
        ref, mag = torch.einsum("hqk,khd->qhd", p, vv), torch.einsum("hqk,khd->qhd", p, vv.abs())
        # P and the output in bf16: 2^-8 each; scores in fp32; the batched projection may
        # round q, k, v by another ulp (2^-8 of them) than one per prompt
        err = (prompt_out[at:at + n].double() - ref).abs()
        assert torch.all(err <= 2.0 ** -4 * mag + 2.0 ** -7 * ref.abs() + 1e-6)
        at += n
        # the last step, over what the cache holds
        pages = ids[ptr[b]:ptr[b + 1]]
        total = n + steps
        kc, vc = ((c[pages].float() * sc[pages][:, None, :, None]).reshape(-1, hkv, 128)[:total].double()
                  for c, sc in zip(st["cache"], st["scales"]))
        q = layer.qkv(st["inputs"][-1])[0][b:b + 1]
        qr = _rope_sorted(q, cos[total - 1:total], sin[total - 1:total])[0].double()
        s = torch.einsum("hd,khd->hk", qr, kc.repeat_interleave(hq // hkv, 1)) / math.sqrt(128)
        p = torch.softmax(s, -1)
        vv = vc.repeat_interleave(hq // hkv, 1)
        ref, mag = torch.einsum("hk,khd->hd", p, vv), torch.einsum("hk,khd->hd", p, vv.abs())
        err = (outs[-1][b].double() - ref).abs()
        assert torch.all(err <= 2.0 ** -8 * mag + 2.0 ** -8 * ref.abs() + 1e-6)
        # and what the cache holds is the prompt's keys, to e4m3's half step (plus the projections' ulp)
        x = kr.float()
        assert torch.all((kc[:n].float() - x).abs() <= x.abs() * (2.0 ** -4 + 2.0 ** -6) +
                         st["scales"][0][pages].repeat_interleave(page, 0)[:n, :, None] * 2.0 ** -8)
