"""Cases of the serving-step operators, with a plain form of each.

    tables   page tables and slot maps of a step, from the requests' lengths
    append   K/V rows of new tokens into an e4m3 paged cache with one scale for
             each page and kv head (RoPE of K at write)
    decode   one query token per request over that cache
    packed   causal attention over packed prompts of different lengths

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run`
computes one pass: in elementary torch operations where `own` is false, through
the package's entry points where it is true."""
import math
import os
import random
import sys

import torch

own = False

D = 128  # head_dim
E4M3_MAX = 448.0
E4M3 = torch.float8_e4m3fn
PEAK_LEVELS = D // 16


def _atflash():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atflash-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import atflash
    return atflash


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a serving engine's decode step: every running request grows by one token
        dict(name="tables_step_b256", op="tables", batch=256, max_len=8192, page=16, prompts=0, mix=1),
        # a step that mixes decodes with new prompts, an odd request count, larger pages
        dict(name="tables_mixed_b61", op="tables", batch=61, max_len=3001, page=64, prompts=9, mix=2),
        # a large server: thousands of requests, about a million table entries
        dict(name="tables_b4096", op="tables", batch=4096, max_len=8000, page=16, prompts=64, mix=3),
        # the write side of a decode step, 8 kv heads, RoPE at write
        dict(name="append_step_b64", op="append", batch=64, max_len=4096, page=16, hkv=8, prompts=0, layout="NHD",
             rope=True, mix=4),
        # prompts of odd lengths that begin inside a page, HND pages, K already rotated
        dict(name="append_ragged_b13", op="append", batch=13, max_len=3001, page=64, hkv=4, prompts=13, layout="HND",
             rope=False, mix=5),
        # four long prompts written at once (64K tokens, as the bf16 append's measured size)
        dict(name="append_prompt_64k", op="append", batch=4, max_len=16384, page=16, hkv=8, prompts=-1, layout="NHD",
             rope=True, mix=6),
        # a few short requests, where the call's latency counts
        dict(name="decode_short_b3", op="decode", batch=3, max_len=300, page=16, hkv=8, group=3, window=False,
             layout="NHD", even=False, mix=7),
        # a batch of ragged requests, one kv head for 7 query heads, HND pages of 64
        dict(name="decode_ragged_b37", op="decode", batch=37, max_len=20011, page=64, hkv=4, group=7, window=False,
             layout="HND", even=False, mix=8),
        # 128K tokens x 8 requests, 24 / 8 heads, the window on: the bf16 decode's large configuration
        dict(name="decode_128k_b8", op="decode", batch=8, max_len=131072, page=16, hkv=8, group=3, window=True,
             layout="NHD", even=True, mix=9),
        # a handful of short prompts of odd lengths
        dict(name="packed_short_b5", op="packed", batch=5, max_len=213, hkv=4, group=7, prefix=0, window=False,
             even=False, mix=10),
        # a prefill batch of ragged prompts, 24 / 8 heads
        dict(name="packed_ragged_b16", op="packed", batch=16, max_len=4096, hkv=8, group=3, prefix=0, window=False,
             even=False, mix=11),
        # long prompts, 28 / 4 heads, each a chunk behind a cached prefix, the window on
        dict(name="packed_long_b4", op="packed", batch=4, max_len=8192, hkv=4, group=7, prefix=2048, window=True,
             even=False, mix=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tables", "append", "decode", "packed"])
    mix = rng.randrange(100, 1000000)
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "tables":
        batch = _log_int(rng, 1, 4096)
        return dict(op=op, batch=batch, max_len=_log_int(rng, 1, 8000), page=page, prompts=rng.choice([0, min(batch, 9)]),
                    mix=mix)
    hkv = rng.choice([1, 2, 4, 8])
    if op == "append":
        batch = _log_int(rng, 1, 64)
        prompts = rng.choice([0, batch])
        max_len = _log_int(rng, 1, 4096 if not prompts else max(1, min(16384, 60000 // batch)))
        return dict(op=op, batch=batch, max_len=max_len, page=page, hkv=hkv, prompts=prompts,
                    layout=rng.choice(["NHD", "HND"]), rope=rng.random() < 0.5, mix=mix)
    group = rng.choice([1, 2, 3, 4, 7, 8, 12])
    if op == "decode":
        batch = _log_int(rng, 1, 64)
        max_len = _log_int(rng, 1, min(131072, 8 * 131072 // batch))
        return dict(op=op, batch=batch, max_len=max_len, page=page, hkv=hkv, group=group, window=rng.random() < 0.5,
                    layout=rng.choice(["NHD", "HND"]), even=rng.random() < 0.3, mix=mix)
    group = rng.choice([1, 2, 3, 4, 7])
    batch = _log_int(rng, 1, 48)
    prefix = rng.choice([0, 0, _log_int(rng, 1, 1500)])
    max_len = _log_int(rng, 1, max(1, min(8192, int(math.sqrt(7e9 / (batch * hkv * group))) - prefix)))
    return dict(op=op, batch=batch, max_len=max_len, hkv=hkv, group=group, prefix=prefix, window=rng.random() < 0.4,
                even=False, mix=mix)


def _lens(case):
    """Lengths of the requests after the step and the tokens that the step adds."""
    rng = random.Random(case["mix"])
    n, top = case["batch"], case["max_len"]
    if case.get("even"):
        lens = [top] * n
    else:
        lens = [_log_int(rng, 1, top) if rng.random() < 0.4 else rng.randint(1, top) for _ in range(n)]
        lens[rng.randrange(n)] = top
    if case["op"] == "packed":  # queries and keys of each sequence
        keys = [x + (rng.randint(0, case["prefix"]) if case["prefix"] else 0) for x in lens]
        return keys, lens
    prompts = case.get("prompts", 0)
    if prompts < 0:  # whole prompts, from their first token
        lens = [top] * n
        return lens, list(lens)
    first = set(rng.sample(range(n), prompts))
    return lens, [rng.randint(1, x) if b in first else 1 for b, x in enumerate(lens)]


def _zhi(base=1e6, k=2.0, cap=1 << 30):
    """Largest distance at which each 16-dim level of a head is read (pairs sorted
    by falling wavelength, width k wavelengths; the first level always)."""
    p = D // 2
    w = [k * 2.0 * math.pi * base ** (2.0 * (p - 1 - j) / D) for j in range(p)]
    return [cap] + [min(cap, int(w[8 * i])) for i in range(1, PEAK_LEVELS)]


# ------------------------------------------------------------------ inputs

def _indptr(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _i32(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _quantised(rows, page_axes, gen_factor):
    """e4m3 pages and their power-of-two scales for random rows (P, A, B, D)."""
    x = rows * gen_factor
    amax = x.abs().amax(dim=page_axes, keepdim=True).clamp_min(1e-20)
    s = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)))
    return (x / s).to(E4M3), s


def _cache(case, num_pages, gen):
    """A filled cache: pages in the case's layout and scales (P, Hkv) for K and V.
    Pages differ in magnitude, as the tokens of a text do."""
    page, hkv, nhd = case["page"], case["hkv"], case["layout"] == "NHD"
    shape = (num_pages, page, hkv, D) if nhd else (num_pages, hkv, page, D)
    fshape = (num_pages, 1, hkv, 1) if nhd else (num_pages, hkv, 1, 1)
    out = []
    for _ in range(2):
        rows = torch.randn(shape, device="cuda", generator=gen)
        f = torch.exp2(torch.randint(-2, 3, fshape, device="cuda", generator=gen).float())
        pages, s = _quantised(rows, (1, 3) if nhd else (2, 3), f)
        out += [pages, s.reshape(num_pages, hkv).contiguous()]
        del rows
    return out  # k, k_scale, v, v_scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    lens, extra = _lens(case)
    s = {"case": case, "op": op}
    if op in ("tables", "append", "decode"):
        page = case["page"]
        npg = [(x + page - 1) // page for x in lens]
        total = sum(npg)
        perm = torch.randperm(total + 7, generator=gen, device="cuda").to(torch.int32)
    if op == "tables":
        # each request's row of the engine's table holds the pages it has already;
        # new ones come from the free list
        have = [(x - a + page - 1) // page for x, a in zip(lens, extra)]
        width = (case["max_len"] + page - 1) // page
        counts, start = _i32(have).long(), _i32(_indptr(have)[:-1]).long()
        j = torch.arange(width, device="cuda")
        held = j[None] < counts[:, None]
        table = torch.where(held, perm.long()[(start[:, None] + j[None]).clamp(max=perm.numel() - 1)], -1)
        s.update(kv_lens=_i32(lens), append_lens=_i32(extra), req_pages=table.to(torch.int32).contiguous(), page=page,
                 free_pages=perm[sum(have):].contiguous(), free_head=_i32([0]), tokens=sum(extra), pages=total)
        return s
    if op == "append":
        hkv = case["hkv"]
        k, ks, v, vs = _cache(case, total + 7, gen)
        ap = _indptr(extra)
        rope = None
        if case["rope"]:
            inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").float() / D))
            t = torch.arange(case["max_len"], device="cuda").float()[:, None] * inv[None]
            rope = (torch.cos(t), torch.sin(t))
        new = [(torch.randn((ap[-1], hkv, D), device="cuda", generator=gen)
                * torch.exp2(torch.randint(-2, 3, (ap[-1], 1, 1), device="cuda", generator=gen).float())).bfloat16()
               for _ in range(2)]
        which = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _i32(extra).long(), output_size=ap[-1])
        pos = torch.arange(ap[-1], device="cuda") - _i32(ap[:-1]).long()[which] + (_i32(lens) - _i32(extra)).long()[which]
        s.update(key=new[0], value=new[1], k=k, ks=ks, v=v, vs=vs, batch_indices=which.to(torch.int32),
                 positions=pos.to(torch.int32), indptr=_i32(_indptr(npg)), indices=perm[:total].contiguous(), rope=rope)
        return s
    if op == "decode":
        hq = case["hkv"] * case["group"]
        k, ks, v, vs = _cache(case, total + 7, gen)
        q = torch.randn((len(lens), hq, D), device="cuda", generator=gen).bfloat16()
        last = [(x - 1) % page + 1 for x in lens]
        s.update(q=q, k=k, ks=ks, v=v, vs=vs, kv_lens=_i32(lens), indptr=_i32(_indptr(npg)),
                 indices=perm[:total].contiguous(), max_pages=max(npg), zhi=_zhi() if case["window"] else None)
        if own:  # a serving program plans a step once and keeps the wrapper for all layers
            w = _atflash().BatchDecodeWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"),
                                                              case["layout"])
            w.plan(_indptr(npg), s["indices"], last, hq, case["hkv"], D, page, kv_data_type=E4M3,
                   window_table=s["zhi"])
            s["wrapper"] = w
        return s
    hkv, hq = case["hkv"], case["hkv"] * case["group"]
    cq, ck = _indptr(extra), _indptr(lens)
    s.update(q=torch.randn((cq[-1], hq, D), device="cuda", generator=gen).bfloat16(),
             k=torch.randn((ck[-1], hkv, D), device="cuda", generator=gen).bfloat16(),
             v=torch.randn((ck[-1], hkv, D), device="cuda", generator=gen).bfloat16(),
             cu_q=_i32(cq), cu_k=_i32(ck), max_q=max(extra), max_k=max(lens), zhi=_zhi() if case["window"] else None)
    if own:
        w = _atflash().BatchPrefillWithRaggedKVCacheWrapper(torch.device("cuda"))
        w.plan(cq, ck, hq, hkv, D, causal=True, window_table=s["zhi"])
        s["wrapper"] = w
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    return {"tables": _tables, "append": _append, "decode": _decode, "packed": _packed}[state["op"]](state)


def _tables(s):
    if own:
        t = _atflash().build_page_tables(s["kv_lens"], s["append_lens"], s["req_pages"], s["page"],
                                         num_tokens=s["tokens"], max_pages=s["pages"], free_pages=s["free_pages"],
                                         free_head=s["free_head"])
        return [t.indptr, t.indices, t.last_page_len, t.append_indptr, t.batch_indices, t.positions, t.slot_mapping,
                t.free_head, s["req_pages"]]
    page, table = s["page"], s["req_pages"]
    lens, app = s["kv_lens"].long(), s["append_lens"].long()
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    n = (lens + page - 1) // page
    have = (lens - app + page - 1) // page
    indptr = torch.cat([zero, n.cumsum(0)])
    fresh = torch.cat([zero, (n - have).cumsum(0)])
    ap = torch.cat([zero, app.cumsum(0)])
    # pages: entry e belongs to request b, and is its page j
    e = torch.arange(s["pages"], device="cuda")
    b = torch.searchsorted(indptr, e, right=True) - 1
    j = e - indptr[b]
    new = j >= have[b]
    at = (s["free_head"].long() + fresh[b] + j - have[b]).clamp(0, s["free_pages"].numel() - 1)
    indices = torch.where(new, s["free_pages"][at], table[b, j])
    table[b, j] = indices
    # tokens: entry t belongs to request b at position pos
    t = torch.arange(s["tokens"], device="cuda")
    tb = torch.searchsorted(ap, t, right=True) - 1
    pos = lens[tb] - app[tb] + t - ap[tb]
    slot = table[tb, pos // page].long() * page + pos % page
    last = torch.where(n > 0, lens - (n - 1) * page, 0)
    i32 = torch.int32
    return [indptr.to(i32), indices, last.to(i32), ap.to(i32), tb.to(i32), pos.to(i32), slot,
            (s["free_head"] + fresh[-1:]).to(i32), table]


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, within [2^-126, 2^120]."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), -126).clamp(-126, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def _append(s):
    case = s["case"]
    if own:
        _atflash().append_paged_kv_cache(s["key"], s["value"], s["batch_indices"], s["positions"], (s["k"], s["v"]),
                                         s["indices"], s["indptr"], kv_layout=case["layout"],
                                         kv_scales=(s["ks"], s["vs"]), rope=s["rope"], out_layout="sorted_pair")
        return [s["k"], s["ks"], s["v"], s["vs"]]
    page, nhd = case["page"], case["layout"] == "NHD"
    pos, pages = s["positions"].long(), s["k"].shape[0]
    slot = pos % page
    target = s["indices"].long()[s["indptr"].long()[s["batch_indices"].long()] + pos // page]
    x = s["key"].float()
    if s["rope"] is not None:
        c, sn = s["rope"][0][pos][:, None], s["rope"][1][pos][:, None]
        lo, hi = x[..., :64], x[..., 64:]
        r = torch.stack([lo * c - hi * sn, hi * c + lo * sn], dim=-1).flip(-2)  # widest pair first
        x = r.reshape(x.shape).bfloat16().float()
    # first slot that the call writes in each page: before it, rows stay
    start = torch.full((pages,), page, dtype=torch.long, device="cuda").scatter_reduce(0, target, slot, "amin")
    touched = start < page
    for rows, cache, scale in ((x, s["k"], s["ks"]), (s["value"].float(), s["v"], s["vs"])):
        view = cache if nhd else cache.transpose(1, 2)  # (P, page, Hkv, D)
        amax = torch.zeros(scale.shape, device="cuda").index_reduce_(0, target, rows.abs().amax(-1), "amax")
        want = _scale_of(amax)
        new = torch.where(touched[:, None], torch.where(start[:, None] > 0, torch.maximum(scale, want), want), scale)
        # rows already there, under a scale that grows
        p, h = torch.nonzero(touched[:, None] & (start[:, None] > 0) & (new != scale), as_tuple=True)
        old = view[p, :, h].float() * (scale[p, h] / new[p, h])[:, None, None]
        keep = (torch.arange(page, device="cuda")[None] < start[p][:, None])[..., None]
        view[p, :, h] = torch.where(keep, old, view[p, :, h].float()).to(E4M3)
        view[target, slot] = (rows / new[target][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        scale.copy_(new)
    return [s["k"], s["ks"], s["v"], s["vs"]]


def _decode(s):
    case = s["case"]
    if own:
        out, lse = s["wrapper"].run(s["q"], (s["k"], s["v"]), kv_scales=(s["ks"], s["vs"]), return_lse=True)
        return [out, lse]
    page, hkv, g = case["page"], case["hkv"], case["group"]
    nhd, n = case["layout"] == "NHD", s["q"].shape[0]
    j = torch.arange(s["max_pages"], device="cuda")
    first = s["indptr"].long()
    ids = s["indices"].long()[(first[:-1, None] + j[None]).clamp(max=s["indices"].numel() - 1)]  # (B, pages)

    def rows(cache, scale):  # (B, Hkv, keys, D) in 32 bits
        x = cache[ids]
        x = x.permute(0, 3, 1, 2, 4) if nhd else x.permute(0, 2, 1, 3, 4)
        x = x.float() * scale[ids].permute(0, 2, 1)[..., None, None]
        return x.reshape(n, hkv, -1, D)
    key = torch.arange(s["max_pages"] * page, device="cuda")
    lens = s["kv_lens"].long()
    k = rows(s["k"], s["ks"])
    if s["zhi"] is not None:  # the levels of a key that its distance keeps
        dist = lens[:, None] - 1 - key[None]
        reach = torch.tensor(s["zhi"], device="cuda").repeat_interleave(16)
        k = k.mul_((dist[..., None] <= reach)[:, None])
    score = (s["q"].float().view(n, hkv, g, D) @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    del k
    score = score.masked_fill_((key[None] >= lens[:, None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    den = p.sum(-1, keepdim=True)
    out = (p @ rows(s["v"], s["vs"])) / den
    return [out.reshape(n, hkv * g, D).bfloat16(), (top + torch.log(den)).reshape(n, hkv * g)]


def _packed(s):
    case = s["case"]
    if own:
        out, lse = s["wrapper"].run(s["q"], s["k"], s["v"], return_lse=True)
        return [out, lse]
    hkv, g, n = case["hkv"], case["group"], case["batch"]
    lq, lk = s["max_q"], s["max_k"]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    nq, nk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    iq, ik = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    qi = (cq[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)  # rows of each sequence, padded to the longest
    ki = (ck[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"].float()[qi].view(n, lq, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * lq, D)
    k = s["k"].float()[ki].permute(0, 2, 3, 1)  # (B, Hkv, D, keys)
    v = s["v"].float()[ki].permute(0, 2, 1, 3)
    place = iq[None] + (nk - nq)[:, None]  # position of each query among its keys
    dead = (ik[None, None] > place[..., None]) | (ik[None, None] >= nk[:, None, None])  # (B, q, k)
    if s["zhi"] is None:
        score = q @ k
    else:  # a level counts in a tile of 128 x 128 where the tile's smallest distance keeps it
        near = (place - iq[None] % 128)[:, :, None] - (ik // 128 * 128 + 127)[None, None]
        score = q[..., :16] @ k[:, :, :16]
        for i in range(1, PEAK_LEVELS):
            part = (q[..., 16 * i:16 * i + 16] @ k[:, :, 16 * i:16 * i + 16]).view(n, hkv, g, lq, lk)
            score += part.mul_((near <= s["zhi"][i])[:, None, None]).view(score.shape)
            del part
    score = score.view(n, hkv, g, lq, lk).mul_(1.0 / math.sqrt(D)).masked_fill_(dead[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    score = score.sub_(top).exp_()
    den = score.sum(-1, keepdim=True)
    out = (score.view(n, hkv, g * lq, lk) @ v).view(n, hkv, g, lq, D)
    out = torch.where(den > 0, out / den, 0.0)
    lse = top + torch.log(den)
    seq, row = torch.nonzero(iq[None] < nq[:, None], as_tuple=True)  # the packed rows, in order
    out = out.permute(0, 3, 1, 2, 4)[seq, row].reshape(-1, hkv * g, D)
    return [out.bfloat16(), lse[..., 0].permute(0, 3, 1, 2)[seq, row].reshape(-1, hkv * g)]


# ------------------------------------------------------------------ work

def _pairs(nq, nk):
    """Query-key pairs of a causal block of nq queries at the end of nk keys."""
    return sum(max(0, nk - nq + 1 + i) for i in (0, nq - 1)) * nq / 2


def work(case):
    lens, extra = _lens(case)
    op = case["op"]
    if op == "tables":
        page = case["page"]
        pages = sum((x + page - 1) // page for x in lens)
        fresh = pages - sum((x - a + page - 1) // page for x, a in zip(lens, extra))
        n = len(lens)
        return {"bytes": 8 * n + 4 * (2 * (n + 1) + n) + 8 * pages + 4 * fresh + 16 * sum(extra), "flops": 0}
    if op == "append":
        rows = 2 * sum(extra) * case["hkv"]
        page = case["page"]
        runs = sum((x - 1) // page - (x - a) // page + 1 for x, a in zip(lens, extra))
        tables = 2 * 64 * 4 * sum(extra) if case["rope"] else 0
        return {"bytes": rows * D * 3 + runs * case["hkv"] * 8 + 8 * sum(extra) + tables,
                "flops": rows * D * (5 if case["rope"] else 2)}
    if op == "decode":
        hkv, hq, page = case["hkv"], case["hkv"] * case["group"], case["page"]
        keys = sum(lens)
        reach = _zhi() if case["window"] else [1 << 30] * PEAK_LEVELS
        kdims = sum(16 * min(x, z + 1) for x in lens for z in reach)
        pages = sum((x + page - 1) // page for x in lens)
        return {"bytes": hkv * (kdims + keys * D) + 4 * pages * (1 + 2 * hkv) + 4 * len(lens) * hq * (D + 1),
                "flops": 2 * hq * (kdims + keys * D)}
    hkv, hq = case["hkv"], case["hkv"] * case["group"]
    pairs = sum(_pairs(a, x) for x, a in zip(lens, extra))
    kpairs = pairs * D
    if case["window"]:
        reach = _zhi()
        kpairs = 0
        for x, a in zip(lens, extra):
            for t in range(0, a, 128):
                rows = min(128, a - t)
                q0 = x - a + t
                # keys seen by the rows of this query tile, level by level
                for z in reach:
                    lo = 0 if q0 - 127 - z <= 0 else (q0 - 127 - z + 127) // 128 * 128
                    kpairs += 16 * sum(max(0, q0 + i + 1 - lo) for i in (0, rows - 1)) * rows / 2
    io = 4 * hq * D * sum(extra) + 4 * hkv * D * sum(lens) + 4 * hq * sum(extra)
    return {"bytes": io, "flops": 2 * hq * (kpairs + pairs * D)}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    lens, extra = _lens(case)
    with torch.no_grad():
        return {"append": _exact_append, "decode": _exact_decode, "packed": _exact_packed}[case["op"]](case, s, lens,
                                                                                                        extra)


def _round_e4m3(x):
    """float64 values to the nearest e4m3 value (ties to even), saturating."""
    a = x.abs().clamp(max=E4M3_MAX)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 1).clamp(min=-6) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=E4M3_MAX)


def _exact_append(case, s, lens, extra):
    page, nhd = case["page"], case["layout"] == "NHD"
    indptr, ids = s["indptr"].tolist(), s["indices"].tolist()
    key = s["key"].double()
    if s["rope"] is not None:
        # the rotation is defined in 32 bits with separately rounded products, then bf16
        pos = s["positions"].long()
        c, sn = (t[pos][:, None] for t in s["rope"])
        a, b = s["key"].float().split(64, dim=-1)
        first, second = torch.sub(a * c, b * sn), torch.add(b * c, a * sn)
        key = torch.empty_like(s["key"])
        key[..., 0::2], key[..., 1::2] = first.flip(-1).bfloat16(), second.flip(-1).bfloat16()
        key = key.double()
    out = []
    for rows, cache, scale in ((key, s["k"], s["ks"]), (s["value"].double(), s["v"], s["vs"])):
        values = (cache if nhd else cache.transpose(1, 2)).double().contiguous()
        scales = scale.double()
        runs, at = [], 0
        for b, (x, a) in enumerate(zip(lens, extra)):
            pos = x - a
            while pos < x:
                m = min(page - pos % page, x - pos)
                runs.append((ids[indptr[b] + pos // page], pos % page, m, at))
                at, pos = at + m, pos + m
        if len(runs) > 6000:
            return None
        amax = torch.stack([rows[t:t + m].abs().amax(dim=(0, 2)) for _, _, m, t in runs])
        _, e = torch.frexp(amax / E4M3_MAX)
        exact_power = torch.ldexp(torch.ones_like(amax), e - 1) == amax / E4M3_MAX
        want = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e - exact_power.to(e.dtype), -126).clamp(-126, 120))
        for (pg, slot, m, t), w in zip(runs, want):
            new = torch.maximum(scales[pg], w) if slot else w
            if slot:
                values[pg, :slot] = torch.where((new == scales[pg])[:, None], values[pg, :slot],
                                                _round_e4m3(values[pg, :slot] * (scales[pg] / new)[:, None]))
            values[pg, slot:slot + m] = _round_e4m3(rows[t:t + m] / new[:, None])
            scales[pg] = new
        out += [(values if nhd else values.transpose(1, 2).contiguous()), scales]
    return out


def _exact_decode(case, s, lens, extra):
    page, hkv, g = case["page"], case["hkv"], case["group"]
    indptr = s["indptr"].tolist()
    out, lse = [], []
    for b, n in enumerate(lens):
        ids = s["indices"][indptr[b]:indptr[b + 1]].long()
        kv = []
        for cache, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = cache[ids].double()
            x = x if case["layout"] == "NHD" else x.transpose(1, 2)
            kv.append((x * scale[ids].double()[:, None, :, None]).reshape(-1, hkv, D)[:n].transpose(0, 1))
        if s["zhi"] is not None:
            dist = torch.arange(n - 1, -1, -1, device="cuda")
            for i in range(1, PEAK_LEVELS):
                kv[0][:, dist > s["zhi"][i], 16 * i:16 * i + 16] = 0
        score = torch.einsum("hgd,hnd->hgn", s["q"][b].double().view(hkv, g, D), kv[0]) / math.sqrt(D)
        lse.append(torch.logsumexp(score, -1).reshape(-1))
        out.append(torch.einsum("hgn,hnd->hgd", torch.softmax(score, -1), kv[1]).reshape(-1, D))
        del kv, score
    return [torch.stack(out), torch.stack(lse)]


def _exact_packed(case, s, lens, extra):
    hkv, g = case["hkv"], case["group"]
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    if sum(a * x for x, a in zip(lens, extra)) * hkv * g > 12e9:
        return None
    out, lse = [], []
    for b, (nk, nq) in enumerate(zip(lens, extra)):
        q = s["q"][cq[b]:cq[b + 1]].double()
        k, v = (t[ck[b]:ck[b + 1]].double() for t in (s["k"], s["v"]))
        row = torch.arange(nq, device="cuda")[:, None]
        col = torch.arange(nk, device="cuda")[None]
        o = torch.empty((nq, hkv * g, D), dtype=torch.float64, device="cuda")
        ls = torch.empty((nq, hkv * g), dtype=torch.float64, device="cuda")
        smallest = nk - nq + row // 128 * 128 - (col // 128 * 128 + 127)
        for h in range(hkv * g):
            levels = range(PEAK_LEVELS) if s["zhi"] is not None else [None]
            score = 0
            for i in levels:
                d = slice(0, D) if i is None else slice(16 * i, 16 * i + 16)
                part = q[:, h, d] @ k[:, h // g, d].T
                score = score + (part if not i else part * (smallest <= s["zhi"][i]))
            score = (score / math.sqrt(D)).masked_fill(col > row + nk - nq, -math.inf)
            ls[:, h] = torch.logsumexp(score, -1)
            o[:, h] = torch.softmax(score, -1) @ v[:, h // g]
        out.append(o)
        lse.append(ls)
    return [torch.cat(out), torch.cat(lse)]
