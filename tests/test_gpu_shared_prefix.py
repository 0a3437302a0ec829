"""The shared-prefix loop on a B200, every output against plain attention in 64 bits over
the tokens that its request has been given, its own and those of the requests it was
forked from: chunks, forks (at a prefix, of forks), frees, compactions, windows."""
import math
import os
import random
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ZHI = (1 << 30, 300, 200, 100, 60, 40, 20, 10)


def _check(ex, e, out):
    import atflash
    for r, per_layer in out.items():
        for i, (layer, o) in enumerate(zip(e.layers, per_layer)):
            q, k, v = (torch.cat([x[j] for x in e.history[r][i]]) for j in range(3))
            nk, nq = k.shape[0], o.shape[0]
            assert nk == e.lens[r]
            qr, kr = (x.double() for x in atflash.qk_norm_rope(q, k, layer.qw, layer.kw, e.cos, e.sin, eps=e.eps,
                                                               out_layout="sorted_pair"))
            qr, v = qr[nk - nq:], v.double()
            row, col = torch.arange(nq, device=e.dev)[:, None], torch.arange(nk, device=e.dev)[None]
            near = nk - nq + row // 128 * 128 - (col // 128 * 128 + 127)
            g = e.hq // e.hkv
            for h in range(e.hq):
                kh, vh = kr[:, h // g], v[:, h // g]
                if e.window is None:
                    s = qr[:, h] @ kh.T
                else:
                    s = sum((qr[:, h, 16 * n:16 * n + 16] @ kh[:, 16 * n:16 * n + 16].T) * (near <= e.window[n] if n else 1)
                            for n in range(8))
                s = (s / math.sqrt(128)).masked_fill(col > row + nk - nq, -math.inf)
                p = torch.softmax(s, -1)
                want, size = p @ vh, p @ vh.abs()
                # P and the output in bf16, 2^-8 each, and fp32 scores
                tol = size * (2.0 ** -8 + 2.0 ** -12) + want.abs() * 2.0 ** -8 + 1e-6
                assert ((o[:, h].double() - want).abs() <= tol).all(), (r, i, h)


@pytest.mark.parametrize("page,hq,hkv,window", [(16, 12, 4, None), (64, 4, 4, None), (32, 14, 2, ZHI)])
def test_every_output_of_a_life(page, hq, hkv, window):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import shared_prefix as ex
    import atflash
    rng = random.Random(page)
    e = ex.Engine(hq=hq, hkv=hkv, page=page, pages=1400 // page * 4, rows=40, window=window)
    g = torch.Generator(device="cuda").manual_seed(page)
    rand = lambda n: torch.randn((n, 256), generator=g, device="cuda").bfloat16()
    _check(ex, e, e.step({0: rand(130), 1: rand(33), 2: rand(1)}))
    _check(ex, e, e.step({0: rand(157), 1: rand(1), 2: rand(63)}))  # a chunk, a decode, another chunk
    kids = list(range(3, 15))
    e.fork([r % 3 for r in kids], kids, [rng.choice([e.lens[r % 3], rng.randint(1, e.lens[r % 3])]) for r in kids])
    _check(ex, e, e.step({r: rand(rng.randint(1, 5)) for r in (0, *kids)}))
    e.free([1, 2, *kids[::3]])
    e.compact(5)
    _check(ex, e, e.step({r: rand(rng.randint(1, 3)) for r in e.lens}))
    more = list(range(20, 30))
    e.fork([rng.choice(list(e.lens)) for _ in more], more)  # forks of forks
    _check(ex, e, e.step({r: rand(rng.choice([1, 1, 40])) for r in e.lens}))
    e.free([r for r in e.lens if r % 2])
    e.compact()
    used = e.pages_in_use()
    held = [e.req_pages[r, :-(-n // page)] for r, n in e.lens.items()]
    assert sorted(torch.cat(held).unique().tolist()) == list(range(used))
    _check(ex, e, e.step({r: rand(2) for r in e.lens}))
    e.free(list(e.lens))
    assert e.pages_in_use() == 0 and not e.shared.any() and sorted(e.free_pages.tolist()) == list(range(e.pages))
    assert atflash.check_device_errors() == 0


def test_the_example_runs():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "shared_prefix.py"), "--each", "3", "--steps", "2",
                          "--window"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "left after 2 steps" in out.stdout
