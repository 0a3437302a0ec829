"""Cases of the operators around a paged cache that requests share, with a plain form
of each.

    norm     RMS norms of the query and key heads with their rotation in one pass
    nappend  the same norm and rotation of K on its way into the cache's pages
             (bf16 pages, K level-major or as V; e4m3 pages with their scales)
    fork     requests freed, others forked from running ones: pages shared, the last
             partial page of each copied in every layer's cache
    compact  the pages in use moved to the low end of the pool, tables and free list
             with them
    chunk    attention of a chunk of new tokens (one to thousands of a request) over
             the cache's pages

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
LEVELS = D // 16
EPS = 1e-6


def _atflash():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atflash-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import atflash
    return atflash


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a decode step of 64 requests, 28 / 4 heads, each token at its own position
        dict(name="norm_step_t64", op="norm", tokens=64, hq=28, hkv=4, layout="sorted_pair", fused=True, w32=False, mix=1),
        # a prefill batch of an odd size, 24 / 8 heads, out of separate projections
        dict(name="norm_prompt_64k", op="norm", tokens=65521, hq=24, hkv=8, layout="rotate_half", fused=False, w32=True,
             mix=2),
        # the write side of a decode step into the decode's level-major K pages
        dict(name="nappend_step_b64", op="nappend", batch=64, max_len=4096, page=16, hkv=8, prompts=0, kind="level",
             mix=3),
        # prompts of odd lengths that begin inside a page, into e4m3 HND pages
        dict(name="nappend_e4m3_b13", op="nappend", batch=13, max_len=3001, page=64, hkv=4, prompts=13, kind="e4m3_hnd",
             mix=4),
        # four long prompts written at once (64K tokens), bf16 pages
        dict(name="nappend_prompt_64k", op="nappend", batch=4, max_len=16384, page=16, hkv=8, prompts=-1, kind="level",
             mix=5),
        # beam search or parallel sampling: four prompts, four continuations each, 28 layers
        dict(name="fork_p4x4", op="fork", parents=4, each=4, max_len=2000, page=16, hkv=4, layers=28, kind="bf16", mix=6),
        # many continuations of long prompts, e4m3 pages with scales
        dict(name="fork_p12x8", op="fork", parents=12, each=8, max_len=8192, page=64, hkv=8, layers=8, kind="e4m3", mix=7),
        # a small pool after some requests have left it
        dict(name="compact_b9", op="compact", batch=9, max_len=1500, page=16, hkv=8, layers=4, pool=2.0, mix=8),
        # a large pool, half of its pages free and scattered
        dict(name="compact_b200", op="compact", batch=200, max_len=4000, page=64, hkv=4, layers=2, pool=2.0, mix=9),
        # a few drafted tokens a request, verified at once over long contexts, 28 / 4 heads
        dict(name="chunk_verify_b24", op="chunk", batch=24, chunk=5, even=True, max_len=16001, page=16, hkv=4, group=7,
             window=False, layout="NHD", mix=10),
        # a step that mixes decodes with chunks of prompts, 24 / 8 heads, HND pages of 64
        dict(name="chunk_mixed_b9", op="chunk", batch=9, chunk=700, even=False, max_len=5003, page=64, hkv=8, group=3,
             window=False, layout="HND", mix=11),
        # chunked prefill of long prompts behind cached prefixes, 28 / 4 heads, the window on
        dict(name="chunk_long_b2", op="chunk", batch=2, chunk=8192, even=True, max_len=32768, page=16, hkv=4, group=7,
             window=True, layout="NHD", mix=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "nappend", "fork", "compact", "chunk"])
    mix = rng.randrange(100, 1000000)
    page = rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "norm":
        group = rng.choice([1, 2, 3, 4, 7, 8])
        return dict(op=op, tokens=_log_int(rng, 1, 65521 * 32 // (hkv * (group + 1)) if hkv * (group + 1) > 32 else 65521),
                    hq=hkv * group, hkv=hkv, layout=rng.choice(["sorted_pair", "rotate_half"]), fused=rng.random() < 0.5,
                    w32=rng.random() < 0.5, mix=mix)
    if op == "nappend":
        batch = _log_int(rng, 1, 64)
        prompts = rng.choice([0, batch])
        max_len = _log_int(rng, 1, 4096 if not prompts else max(1, min(16384, 60000 // batch)))
        return dict(op=op, batch=batch, max_len=max_len, page=page, hkv=hkv, prompts=prompts,
                    kind=rng.choice(["level", "nhd", "hnd", "e4m3_nhd", "e4m3_hnd"]), mix=mix)
    if op == "fork":
        parents, each = _log_int(rng, 1, 12), _log_int(rng, 1, 8)
        layers = _log_int(rng, 1, max(1, min(28, 900000 // (parents * each * page * hkv))))
        return dict(op=op, parents=parents, each=each, max_len=_log_int(rng, 1, 8192 // parents + 500), page=page,
                    hkv=hkv, layers=layers, kind=rng.choice(["bf16", "e4m3"]), mix=mix)
    if op == "compact":
        batch = _log_int(rng, 1, 200)
        return dict(op=op, batch=batch, max_len=_log_int(rng, 1, min(4000, 100000 // batch)), page=page,
                    hkv=min(hkv, 4), layers=rng.choice([1, 2, 3]), pool=rng.choice([1.1, 1.5, 2.0, 3.0]), mix=mix)
    group = rng.choice([1, 2, 3, 4, 7, 8])
    batch = _log_int(rng, 1, 24)
    max_len = _log_int(rng, 1, 32768)
    top = max(1, min(max_len, int(2e9 / (batch * hkv * group * max_len))))
    return dict(op=op, batch=batch, chunk=_log_int(rng, 1, top), even=rng.random() < 0.4, max_len=max_len, page=page,
                hkv=hkv, group=group, window=rng.random() < 0.4, layout=rng.choice(["NHD", "HND"]), mix=mix)


def _lens(case):
    """Lengths of the requests (with the new tokens) and how many tokens are new."""
    rng = random.Random(case["mix"])
    op, top = case["op"], case["max_len"]
    n = case["parents"] if op == "fork" else case["batch"]
    if op == "chunk" and case["even"]:
        lens = [max(case["chunk"], top - rng.randint(0, top // 8)) for _ in range(n)]
    else:
        lens = [_log_int(rng, 1, top) if rng.random() < 0.4 else rng.randint(1, top) for _ in range(n)]
    lens[rng.randrange(n)] = top
    if op == "chunk":
        return lens, [case["chunk"] if case["even"] else min(x, _log_int(rng, 1, case["chunk"])) for x in lens]
    if op in ("fork", "compact"):
        return lens, None
    prompts = case["prompts"]
    if prompts < 0:  # whole prompts, from their first token
        return [top] * n, [top] * n
    first = set(rng.sample(range(n), prompts))
    return lens, [rng.randint(1, x) if b in first else 1 for b, x in enumerate(lens)]


def _zhi(base=1e6, k=2.0, cap=1 << 30):
    """Largest distance at which each 16-dim level of a head is read (pairs sorted
    by falling wavelength, width k wavelengths; the first level always)."""
    p = D // 2
    w = [k * 2.0 * math.pi * base ** (2.0 * (p - 1 - j) / D) for j in range(p)]
    return [cap] + [min(cap, int(w[8 * i])) for i in range(1, LEVELS)]


# ------------------------------------------------------------------ inputs

def _indptr(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _rope_tables(n):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").double() / D))
    t = torch.arange(n, device="cuda").double()[:, None] * inv[None]
    return torch.cos(t).float(), torch.sin(t).float()


def _weight(gen, wide):
    """A norm's weights: around one, a few of them large, as training leaves them."""
    w = 1.0 + 0.25 * torch.randn(D, device="cuda", generator=gen)
    w = w * torch.exp2(torch.randint(-1, 3, (D,), device="cuda", generator=gen).float() * 0.5)
    return w if wide else w.bfloat16()


def _rows(shape, gen):
    """Projections before a norm: rows of different sizes."""
    f = torch.exp2(torch.randint(-3, 4, (*shape[:-1], 1), device="cuda", generator=gen).float())
    return (torch.randn(shape, device="cuda", generator=gen) * f).bfloat16()


def _pages(shape, gen, e4m3, head_axis):
    """Filled pages, and for e4m3 their power-of-two scales (pages, kv heads)."""
    if not e4m3:
        return torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16), None
    rows = torch.randn(shape, device="cuda", generator=gen)
    fshape = [shape[0], 1, 1, 1]
    fshape[head_axis] = shape[head_axis]
    rows *= torch.exp2(torch.randint(-2, 3, fshape, device="cuda", generator=gen).float())
    axes = tuple(a for a in (1, 2, 3) if a != head_axis)
    s = torch.exp2(torch.ceil(torch.log2(rows.abs().amax(dim=axes, keepdim=True).clamp_min(1e-20) / E4M3_MAX)))
    return (rows / s).to(E4M3), s.reshape(shape[0], shape[head_axis]).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case, "op": case["op"]}
    {"norm": _prepare_norm, "nappend": _prepare_nappend, "fork": _prepare_fork, "compact": _prepare_compact,
     "chunk": _prepare_chunk}[case["op"]](case, s, gen)
    return s


def _prepare_norm(case, s, gen):
    t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
    if case["fused"]:  # one projection for q, k and v
        qkv = _rows((t, hq + 2 * hkv, D), gen)
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv])
    else:
        s.update(q=_rows((t, hq, D), gen), k=_rows((t, hkv, D), gen))
    top = 131072
    s.update(qw=_weight(gen, case["w32"]), kw=_weight(gen, case["w32"]), rope=_rope_tables(top),
             positions=torch.randint(0, top, (t,), device="cuda", generator=gen).to(torch.int32))


def _page_lists(lens, page, gen, spare=7):
    npg = [(x + page - 1) // page for x in lens]
    perm = torch.randperm(sum(npg) + spare, generator=gen, device="cuda").to(torch.int32)
    return npg, perm


def _prepare_nappend(case, s, gen):
    lens, extra = _lens(case)
    page, hkv, kind = case["page"], case["hkv"], case["kind"]
    npg, perm = _page_lists(lens, page, gen)
    pages = perm.numel()
    e4m3, hnd = kind.startswith("e4m3"), kind.endswith("hnd")
    shape = (pages, hkv, page, D) if hnd else (pages, page, hkv, D)
    v, vs = _pages(shape, gen, e4m3, 1 if hnd else 2)
    if kind == "level":
        k, ks = torch.randn((pages, hkv, LEVELS, page, 16), device="cuda", generator=gen, dtype=torch.bfloat16), None
    else:
        k, ks = _pages(shape, gen, e4m3, 1 if hnd else 2)
    ap = _indptr(extra)
    which = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _i32(extra).long(), output_size=ap[-1])
    pos = torch.arange(ap[-1], device="cuda") - _i32(ap[:-1]).long()[which] + (_i32(lens) - _i32(extra)).long()[which]
    qkv = _rows((ap[-1], 4 * hkv, D), gen)  # k and v lie in one projection with two heads' worth of q
    s.update(key=qkv[:, 2 * hkv:3 * hkv], value=qkv[:, 3 * hkv:], k=k, ks=ks, v=v, vs=vs, kw=_weight(gen, False),
             rope=_rope_tables(case["max_len"]), batch_indices=which.to(torch.int32), positions=pos.to(torch.int32),
             indptr=_i32(_indptr(npg)), indices=perm[:sum(npg)].contiguous(), hnd=hnd)


def _layer_caches(case, pages, gen, e4m3):
    """K and V pages of every layer, with their scales: what an engine hands over to be
    copied page by page."""
    out = []
    for _ in range(2 * case["layers"]):
        x, sc = _pages((pages, case["page"], case["hkv"], D), gen, e4m3, 2)
        out.append(x)
        if e4m3:
            out.append(sc)
    return out


def _prepare_fork(case, s, gen):
    lens, _ = _lens(case)
    page, each, n = case["page"], case["each"], case["parents"]
    rng = random.Random(case["mix"] + 1)
    npg = [(x + page - 1) // page for x in lens]
    kids = [(p, min(lens[p], rng.choice([lens[p], rng.randint(1, lens[p])]))) for p in range(n) for _ in range(each)]
    fresh = sum(1 for _, x in kids if x % page)
    live = sum(npg) + fresh
    pages = live + 7
    perm = torch.randperm(pages, generator=gen, device="cuda").tolist()
    width = (case["max_len"] + page - 1) // page
    rows = [[-1] * width for _ in range(n + len(kids))]
    shared = [0] * pages
    start = _indptr(npg)
    for p in range(n):
        rows[p][:npg[p]] = perm[start[p]:start[p + 1]]
    at = sum(npg)
    for c, (p, x) in enumerate(kids):  # the continuations of the last step, which this one replaces
        full = x // page
        rows[n + c][:full] = rows[p][:full]
        for j in range(full):
            shared[rows[p][j]] += 1
        if x % page:
            rows[n + c][full] = perm[at]
            at += 1
    s.update(parents=_i32([p for p, _ in kids]), children=_i32([n + c for c in range(len(kids))]),
             lens=_i32([x for _, x in kids]), req_pages=_i32(rows), shared=_i32(shared), free_pages=_i32(perm),
             free_head=_i32([live]), page=page, caches=_layer_caches(case, pages, gen, case["kind"] == "e4m3"))
    if own:
        s["copier"] = _atflash().PageCopier(s["caches"])


def _prepare_compact(case, s, gen):
    lens, _ = _lens(case)
    page = case["page"]
    npg = [(x + page - 1) // page for x in lens]
    pages = int(sum(npg) * case["pool"]) + 3
    perm = torch.randperm(pages, generator=gen, device="cuda").tolist()
    width = (case["max_len"] + page - 1) // page
    rows = [[-1] * width for _ in lens]
    shared = [0] * pages
    at = 0
    for b, n in enumerate(npg):
        j = 0
        if b % 3 == 2:  # every third request shares the first pages of the one before
            j = min(n, npg[b - 1]) // 2
            rows[b][:j] = rows[b - 1][:j]
            for p in rows[b][:j]:
                shared[p] += 1
        rows[b][j:n] = perm[at:at + n - j]
        at += n - j
    s.update(lens=_i32(lens), req_pages=_i32(rows), shared=_i32(shared), req_pages0=_i32(rows), shared0=_i32(shared),
             free_pages=_i32(perm), num_pages=pages, max_moves=max(1, at), page=page,
             caches=_layer_caches(case, pages, gen, False))
    if own:
        s["copier"] = _atflash().PageCopier(s["caches"])


def _prepare_chunk(case, s, gen):
    lens, extra = _lens(case)
    page, hkv, hq = case["page"], case["hkv"], case["hkv"] * case["group"]
    npg, perm = _page_lists(lens, page, gen)
    nhd = case["layout"] == "NHD"
    shape = (perm.numel(), page, hkv, D) if nhd else (perm.numel(), hkv, page, D)
    cq, last = _indptr(extra), [(x - 1) % page + 1 for x in lens]
    s.update(q=torch.randn((cq[-1], hq, D), device="cuda", generator=gen).bfloat16(), cq=cq, lens=lens,
             k=_pages(shape, gen, False, 0)[0], v=_pages(shape, gen, False, 0)[0], starts=_indptr(npg),
             indices=perm[:sum(npg)].contiguous(), zhi=_zhi() if case["window"] else None)
    if own:  # a serving program plans a step once and keeps the wrapper for all layers
        w = _atflash().BatchPrefillWithPagedKVCacheWrapper(torch.empty(256 << 20, dtype=torch.uint8, device="cuda"),
                                                           case["layout"])
        w.plan(cq, s["starts"], s["indices"], last, hq, hkv, D, page, causal=True, window_table=s["zhi"])
        s["wrapper"] = w


# ------------------------------------------------------------------ one pass

def run(state):
    return {"norm": _norm, "nappend": _nappend, "fork": _fork, "compact": _compact, "chunk": _chunk}[state["op"]](state)


def _normed(x, w, rope, pos, layout):
    """Rows (T, H, D) normed over D, weighted and rotated, in 32 bits."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    c, sn = rope[0][pos][:, None], rope[1][pos][:, None]
    lo, hi = y[..., :64], y[..., 64:]
    a, b = lo * c - hi * sn, hi * c + lo * sn
    if layout == "rotate_half":
        return torch.cat([a, b], dim=-1)
    return torch.stack([a, b], dim=-1).flip(-2).reshape(x.shape)  # widest pair first


def _norm(s):
    case = s["case"]
    if own:
        return list(_atflash().qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], *s["rope"], eps=EPS,
                                            positions=s["positions"], out_layout=case["layout"]))
    pos = s["positions"].long()
    return [_normed(s[x], s[x + "w"], s["rope"], pos, case["layout"]).bfloat16() for x in ("q", "k")]


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, within [2^-126, 2^120]."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), -126).clamp(-126, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def _nappend(s):
    case, e4m3 = s["case"], s["ks"] is not None
    outputs = [s["k"], s["ks"], s["v"], s["vs"]] if e4m3 else [s["k"], s["v"]]
    if own:
        _atflash().append_paged_kv_cache(s["key"], s["value"], s["batch_indices"], s["positions"], (s["k"], s["v"]),
                                         s["indices"], s["indptr"], kv_layout="HND" if s["hnd"] else "NHD",
                                         rope=s["rope"], k_norm=(s["kw"], EPS), out_layout="sorted_pair",
                                         kv_scales=(s["ks"], s["vs"]) if e4m3 else None)
        return outputs
    page, pages = case["page"], s["v"].shape[0]
    pos = s["positions"].long()
    slot = pos % page
    target = s["indices"].long()[s["indptr"].long()[s["batch_indices"].long()] + pos // page]
    key = _normed(s["key"], s["kw"], s["rope"], pos, "sorted_pair").bfloat16()
    if not e4m3:
        if case["kind"] == "level":
            s["k"].permute(0, 3, 1, 2, 4)[target, slot] = key.view(-1, case["hkv"], LEVELS, 16)
        else:
            (s["k"].transpose(1, 2) if s["hnd"] else s["k"])[target, slot] = key
        (s["v"].transpose(1, 2) if s["hnd"] else s["v"])[target, slot] = s["value"]
        return outputs
    # first slot that the call writes in each page: before it, rows stay
    start = torch.full((pages,), page, dtype=torch.long, device="cuda").scatter_reduce(0, target, slot, "amin")
    touched = start < page
    for rows, cache, scale in ((key.float(), s["k"], s["ks"]), (s["value"].float(), s["v"], s["vs"])):
        view = cache.transpose(1, 2) if s["hnd"] else cache  # (P, page, Hkv, D)
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
    return outputs


def _copy_plain(caches, src, dst):
    to, of = dst[src >= 0].long(), src[src >= 0].long()
    for x in caches:
        x = x.view(torch.uint8) if x.dtype == E4M3 else x
        x.index_copy_(0, to, x[of])


def _fork(s):
    page, n = s["page"], s["lens"].numel()
    if own:
        at = _atflash()
        head = at.free_requests(s["children"], s["lens"], s["req_pages"], page, free_pages=s["free_pages"],
                                free_head=s["free_head"], shared=s["shared"])
        f = at.fork_requests(s["parents"], s["children"], s["lens"], s["req_pages"], page, free_pages=s["free_pages"],
                             free_head=head, shared=s["shared"])
        s["copier"].copy(f.src, f.dst)
        return [head, f.src, f.dst, f.free_head, s["req_pages"], s["shared"], s["free_pages"], *s["caches"]]
    lens, table, shared = s["lens"].long(), s["req_pages"], s["shared"]
    kids, parents = s["children"].long(), s["parents"].long()
    j = torch.arange(table.shape[1], device="cuda")
    held = j[None] < ((lens + page - 1) // page)[:, None]
    # the pages of the children that go: one holder less each, free where none is left
    e = torch.nonzero(held.view(-1)).view(-1)
    ids = table[kids].view(-1)[e].long()
    uses = torch.zeros_like(shared).index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    last = torch.full((shared.numel(),), -1, device="cuda").scatter_reduce(0, ids, e, "amax")
    gone = (uses[ids] > shared[ids]) & (last[ids] == e)
    freed = ids[gone]
    head = s["free_head"] - freed.numel()
    s["free_pages"].index_copy_(0, head.long() + torch.arange(freed.numel(), device="cuda"), freed.to(torch.int32))
    shared.copy_((shared - uses).clamp_min_(0))
    table[kids] = torch.where(held, -1, table[kids])
    # the new ones: full pages shared, a page of its own for a partial one
    full = lens // page
    part = lens % page > 0
    order = head.long() + part.long().cumsum(0) - part.long()
    fresh = s["free_pages"][order.clamp(max=s["free_pages"].numel() - 1)]
    src = torch.where(part, table[parents, full.clamp(max=table.shape[1] - 1)], -1)
    dst = torch.where(part, fresh, -1)
    row = torch.where(j[None] < full[:, None], table[parents], table[kids])
    row = torch.where((j[None] == full[:, None]) & part[:, None], dst[:, None], row)
    table[kids] = row
    mine = row[j[None] < full[:, None]].long()
    shared.index_add_(0, mine, torch.ones_like(mine, dtype=torch.int32))
    _copy_plain(s["caches"], src, dst)
    return [head, src, dst, head + part.sum(dtype=torch.int32), table, shared, s["free_pages"], *s["caches"]]


def _compact(s):
    # (a pass begins with the same tables as the last one, scattered again)
    s["req_pages"].copy_(s["req_pages0"])
    s["shared"].copy_(s["shared0"])
    page, table, shared, pages = s["page"], s["req_pages"], s["shared"], s["num_pages"]
    if own:
        m = _atflash().compact_pages(s["lens"], table, page, pages, max_moves=s["max_moves"],
                                     free_pages=s["free_pages"], shared=shared)
        s["copier"].copy(m.src, m.dst)
        return [m.src, m.dst, m.free_head, table, shared, s["free_pages"], *s["caches"]]
    j = torch.arange(table.shape[1], device="cuda")
    held = j[None] < ((s["lens"].long() + page - 1) // page)[:, None]
    live = torch.zeros(pages, dtype=torch.bool, device="cuda")
    live[table[held].long()] = True
    n = live.sum()
    i = torch.arange(pages, device="cuda")
    holes = torch.nonzero(~live & (i < n)).view(-1)  # rising
    movers = torch.nonzero(live & (i >= n)).view(-1).flip(0)  # falling
    src = torch.full((s["max_moves"],), -1, dtype=torch.int32, device="cuda")
    dst = src.clone()
    src[:movers.numel()], dst[:holes.numel()] = movers.to(torch.int32), holes.to(torch.int32)
    to = i.clone()
    to[movers] = holes
    table.copy_(torch.where(held, to[table.clamp_min(0).long()].to(torch.int32), table))
    moved = shared[movers]
    shared[movers] = 0
    shared[holes] = moved
    head = n.to(torch.int32).view(1)
    s["free_pages"].copy_(torch.where(i < n, s["free_pages"], i.to(torch.int32)))
    _copy_plain(s["caches"], src, dst)
    return [src, dst, head, table, shared, s["free_pages"], *s["caches"]]


def _chunk(s):
    if own:
        out, lse = s["wrapper"].run(s["q"], (s["k"], s["v"]), return_lse=True)
        return [out, lse]
    case = s["case"]
    hkv, g, page, nhd = case["hkv"], case["group"], case["page"], case["layout"] == "NHD"
    cq, starts, lens = s["cq"], s["starts"], s["lens"]
    out = torch.empty(s["q"].shape, device="cuda")
    lse = torch.empty(s["q"].shape[:2], device="cuda")
    for b, nk in enumerate(lens):
        nq = cq[b + 1] - cq[b]
        ids = s["indices"][starts[b]:starts[b + 1]].long()
        k, v = (x[ids] if nhd else x[ids].transpose(1, 2) for x in (s["k"], s["v"]))
        k, v = (x.reshape(-1, hkv, D)[:nk].float() for x in (k, v))
        q = s["q"][cq[b]:cq[b + 1]].float() * (1.0 / math.sqrt(D))
        row, col = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
        dead = col[None] > row[:, None] + (nk - nq)
        # smallest distance of a row's tile of 128 queries to a key's tile of 128 keys
        near = (nk - nq + row // 128 * 128)[:, None] - (col // 128 * 128 + 127)[None]
        for h in range(hkv):
            qh, kh = q[:, h * g:(h + 1) * g].transpose(0, 1), k[:, h].T
            if s["zhi"] is None:
                score = qh @ kh
            else:
                score = qh[..., :16] @ kh[:16]
                for i in range(1, LEVELS):
                    part = qh[..., 16 * i:16 * i + 16] @ kh[16 * i:16 * i + 16]
                    score += part.mul_(near <= s["zhi"][i])
            score.masked_fill_(dead, -math.inf)
            top = score.amax(-1, keepdim=True)
            score.sub_(top).exp_()
            den = score.sum(-1, keepdim=True)
            out[cq[b]:cq[b + 1], h * g:(h + 1) * g] = ((score @ v[:, h]) / den).transpose(0, 1)
            lse[cq[b]:cq[b + 1], h * g:(h + 1) * g] = (top + torch.log(den))[..., 0].T
    return [out.bfloat16(), lse]


# ------------------------------------------------------------------ work

def work(case):
    op = case["op"]
    if op == "norm":
        rows = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": 4 * D * rows + case["tokens"] * (4 + 4 * D), "flops": 7 * D * rows}
    lens, extra = _lens(case)
    page = case["page"]
    npg = [(x + page - 1) // page for x in lens]
    if op == "nappend":
        rows = sum(extra) * case["hkv"]
        out = 1 if case["kind"].startswith("e4m3") else 2
        return {"bytes": rows * D * 2 * (2 + out) + sum(extra) * (8 + 4 * D), "flops": rows * D * 8}
    if op in ("fork", "compact"):
        size = page * case["hkv"] * D * (2 if case.get("kind", "bf16") == "bf16" else 1) * 2 * case["layers"]
        if op == "fork":
            rng = random.Random(case["mix"] + 1)
            kids = [min(x, rng.choice([x, rng.randint(1, x)])) for x in lens for _ in range(case["each"])]
            entries, moves = sum((x + page - 1) // page for x in kids), sum(1 for x in kids if x % page)
        else:
            live = 0
            for b, n in enumerate(npg):
                live += n - (min(n, npg[b - 1]) // 2 if b % 3 == 2 else 0)
            pages = int(sum(npg) * case["pool"]) + 3
            entries, moves = sum(npg), int(live * (pages - live) / pages)
        return {"bytes": 2 * size * moves + 16 * entries, "flops": 0}
    hkv, hq = case["hkv"], case["hkv"] * case["group"]
    reach = _zhi() if case["window"] else [1 << 30] * LEVELS
    pairs = kdims = keys = 0
    for x, a in zip(lens, extra):
        keys += x
        pairs += a * (x - a) + a * (a + 1) // 2
        for t in range(0, a, 128):
            rows = min(128, a - t)
            q0 = x - a + t
            for z in reach:  # keys seen by the rows of this query tile, level by level
                lo = max(0, (q0 - 127 - z + 127) // 128 * 128)
                kdims += 16 * sum(max(0, q0 + i + 1 - lo) for i in (0, rows - 1)) * rows // 2
    io = 4 * hq * D * sum(extra) + 4 * hkv * D * keys + 4 * hq * sum(extra) + 4 * sum(npg)
    return {"bytes": io, "flops": 2 * hq * (kdims + D * pairs)}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "nappend": _exact_nappend, "chunk": _exact_chunk}[case["op"]](case, s)


def _exact_rows(x, w, rope, pos, order):
    x = x.double()
    size = torch.sqrt(torch.einsum("thd,thd->th", x, x) / D + EPS)
    y = x / size[..., None] * w.double()
    z = torch.complex(y[..., :64], y[..., 64:]) * torch.complex(rope[0][pos].double(), rope[1][pos].double())[:, None]
    out = torch.empty_like(x)
    if order == "rotate_half":
        out[..., :64], out[..., 64:] = z.real, z.imag
    else:
        for r in range(64):  # pair r of the sorted order is pair 63 - r of the other
            out[..., 2 * r], out[..., 2 * r + 1] = z.real[..., 63 - r], z.imag[..., 63 - r]
    return out


def _exact_norm(case, s):
    pos = s["positions"].long()
    return [_exact_rows(s["q"], s["qw"], s["rope"], pos, case["layout"]),
            _exact_rows(s["k"], s["kw"], s["rope"], pos, case["layout"])]


def _round_e4m3(x):
    """float64 values to the nearest e4m3 value (ties to even), saturating."""
    a = x.abs().clamp(max=E4M3_MAX)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 1).clamp(min=-6) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=E4M3_MAX)


def _exact_nappend(case, s):
    lens, extra = _lens(case)
    page, hkv = case["page"], case["hkv"]
    indptr, ids = s["indptr"].tolist(), s["indices"].tolist()
    key = _exact_rows(s["key"], s["kw"], s["rope"], s["positions"].long(), "sorted_pair")
    runs, at = [], 0  # page, first slot, rows, first token
    for b, (x, a) in enumerate(zip(lens, extra)):
        pos = x - a
        while pos < x:
            m = min(page - pos % page, x - pos)
            runs.append((ids[indptr[b] + pos // page], pos % page, m, at))
            at, pos = at + m, pos + m
    if len(runs) > 6000:
        return None
    out = []
    for rows, cache, scale in ((key, s["k"], s["ks"]), (s["value"].double(), s["v"], s["vs"])):
        values = cache.double()
        if cache.dim() == 5:  # (P, page, Hkv, D) from level-major pages
            values = values.permute(0, 3, 1, 2, 4).reshape(cache.shape[0], page, hkv, D)
        elif s["hnd"]:
            values = values.transpose(1, 2)
        values = values.contiguous()
        if scale is not None:
            rows = rows.bfloat16().double()  # e4m3 pages hold the rounding of what bf16 pages would hold
            scales = scale.double()
            amax = torch.stack([rows[t:t + m].abs().amax(dim=(0, 2)) for _, _, m, t in runs])
            _, e = torch.frexp(amax / E4M3_MAX)
            power = torch.ldexp(torch.ones_like(amax), e - 1) == amax / E4M3_MAX
            want = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e - power.to(e.dtype), -126).clamp(-126, 120))
        for i, (pg, slot, m, t) in enumerate(runs):
            if scale is None:
                values[pg, slot:slot + m] = rows[t:t + m]
                continue
            new = torch.maximum(scales[pg], want[i]) if slot else want[i]
            if slot:
                values[pg, :slot] = torch.where((new == scales[pg])[:, None], values[pg, :slot],
                                                _round_e4m3(values[pg, :slot] * (scales[pg] / new)[:, None]))
            values[pg, slot:slot + m] = _round_e4m3(rows[t:t + m] / new[:, None])
            scales[pg] = new
        if cache.dim() == 5:
            values = values.view(-1, page, hkv, LEVELS, 16).permute(0, 2, 3, 1, 4)
        elif s["hnd"]:
            values = values.transpose(1, 2)
        out += [values.contiguous()] + ([scales] if scale is not None else [])
    return out


def _exact_chunk(case, s):
    lens, extra = _lens(case)
    hkv, g = case["hkv"], case["group"]
    if sum(a * x for x, a in zip(lens, extra)) * hkv * g > 20e9:
        return None
    out, lse, at = [], [], 0
    for b, (nk, nq) in enumerate(zip(lens, extra)):
        q = s["q"][at:at + nq].double()
        at += nq
        ids = s["indices"][s["starts"][b]:s["starts"][b + 1]].long()
        kv = []
        for x in (s["k"], s["v"]):
            x = x.index_select(0, ids).double()
            if case["layout"] == "HND":
                x = x.transpose(1, 2)
            kv.append(x.reshape(-1, hkv, D)[:nk])
        row = torch.arange(nq, device="cuda")[:, None]
        col = torch.arange(nk, device="cuda")[None]
        smallest = nk - nq + row // 128 * 128 - (col // 128 * 128 + 127)
        o = torch.empty((nq, hkv * g, D), dtype=torch.float64, device="cuda")
        ls = torch.empty((nq, hkv * g), dtype=torch.float64, device="cuda")
        for h in range(hkv * g):
            levels = range(LEVELS) if s["zhi"] is not None else [None]
            score = 0
            for i in levels:
                d = slice(0, D) if i is None else slice(16 * i, 16 * i + 16)
                part = q[:, h, d] @ kv[0][:, h // g, d].T
                score = score + (part if not i else part * (smallest <= s["zhi"][i]))
            score = (score / math.sqrt(D)).masked_fill(col > row + nk - nq, -math.inf)
            ls[:, h] = torch.logsumexp(score, -1)
            o[:, h] = torch.softmax(score, -1) @ kv[1][:, h // g]
        out.append(o)
        lse.append(ls)
    return [torch.cat(out), torch.cat(lse)]
