"""e4m3 paged cache in numpy, 64 bits: rounding, the scale rule and the append,
written from their definitions."""
import numpy as np
import torch

MAX = 448.0


def round_e4m3(x):
    """Nearest e4m3 value of float64 x, ties to even, saturating at 448; NaN stays."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), MAX)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(a > 0, a, 1.0)))
    step = np.exp2(np.maximum(e, -6) - 3)
    return np.where(np.isnan(x), np.nan, np.copysign(np.minimum(np.rint(a / step) * step, MAX), x))


def scale_for(amax):
    """The smallest power of two s in [2^-126, 2^120] with amax <= 448 s."""
    e = -126
    while e < 120 and amax > MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_f64(pages):
    return pages.cpu().float().double().numpy()


def append(kc, ks, vc, vs, k, v, bidx, pos, indptr, indices, layout):
    """The append on float64 copies of the pages (values as e4m3) and scales, one
    token list entry after another: runs of adjacent tokens in one page."""
    out = []
    page = kc.shape[1] if layout == "NHD" else kc.shape[2]
    for cache, scale, rows in ((kc, ks, k), (vc, vs, v)):
        c = to_f64(cache)
        if layout == "HND":
            c = c.transpose(0, 2, 1, 3)
        c, s, x = c.copy(), scale.cpu().double().numpy().copy(), rows.cpu().float().double().numpy()
        n, i = len(bidx), 0
        while i < n:
            b, p = int(bidx[i]), int(pos[i])
            m = 1
            while i + m < n and int(bidx[i + m]) == b and int(pos[i + m]) == p + m and (p + m) % page:
                m += 1
            if b >= 0:
                at = int(indptr[b]) + p // page
                if at < int(indptr[b + 1]) and 0 <= int(indices[at]) < c.shape[0]:
                    pg, slot = int(indices[at]), p % page
                    for h in range(x.shape[1]):
                        a = np.abs(x[i:i + m, h])
                        a = a[~np.isnan(a)]
                        want = scale_for(a.max() if a.size else 0.0)
                        new = max(s[pg, h], want) if slot else want
                        if slot and new != s[pg, h]:
                            c[pg, :slot, h] = round_e4m3(c[pg, :slot, h] * (s[pg, h] / new))
                        with np.errstate(invalid="ignore"):
                            c[pg, slot:slot + m, h] = round_e4m3(x[i:i + m, h] / new)
                        s[pg, h] = new
            i += m
        out += [c if layout == "NHD" else c.transpose(0, 2, 1, 3), s]
    return out


def random_cache(num_pages, page, hkv, layout, g, spread=2):
    """Random e4m3 pages with power-of-two scales that differ by page and head."""
    shape = (num_pages, page, hkv, 128) if layout == "NHD" else (num_pages, hkv, page, 128)
    out = []
    for _ in range(2):
        out.append((torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn))
        out.append(torch.exp2(torch.randint(-8 - spread, -7 + spread, (num_pages, hkv), generator=g).float()))
    return out  # k, k_scale, v, v_scale
