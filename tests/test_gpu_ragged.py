"""Prefill over packed sequences on a B200: each sequence's rows are bit for bit
those of a prefill of that sequence alone, and within derived bounds of 64-bit
attention; rows without keys, empty sequences, NaN in the neighbours, strides,
streams, graphs, refusals.

Bounds against 64 bits: scores have exact products and fp32 sums (2^-17 of sum
|q k|); P is rounded to bf16 with 8 significant bits, relative 2^-8 at most, V and
the sums are exact, the output has a half ulp of at most 2^-8 of itself."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Z16 = [1 << 28, 900, 400, 257, 130, 64, 20, 0]


def _packed(nq, nk, hq, hkv, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn((sum(nq), hq, 128), generator=g, device=DEV).bfloat16()
    k, v = (torch.randn((sum(nk), hkv, 128), generator=g, device=DEV).bfloat16() for _ in range(2))
    return q, k, v, np.concatenate([[0], np.cumsum(nq)]), np.concatenate([[0], np.cumsum(nk)])


def _run(q, k, v, cq, ck, run_kw=None, **kw):
    import atflash
    w = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
    w.plan(cq, ck, q.shape[1], k.shape[1], 128, **kw)
    return w.run(q, k, v, return_lse=True, **(run_kw or {}))


def _same_as_alone(got, q, k, v, cq, ck, **kw):
    import atflash
    for b in range(len(cq) - 1):
        sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        if cq[b + 1] == cq[b]:
            continue
        o, lse = atflash.prefill_fwd(q[None, sq], k[None, sk], v[None, sk], return_lse=True, **kw)
        assert torch.equal(got[0][sq], o[0]), b
        assert torch.equal(got[1][sq], lse[0].t()), b


def _exact(q, k, v, zhi=None, causal=True):
    """(out, sum p |v|, lse, bound of the score error), one sequence, 64 bits."""
    nq, hq, _ = q.shape
    nk, hkv, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    row, col = torch.arange(nq, device=DEV)[:, None], torch.arange(nk, device=DEV)[None]
    near = (nk - nq + row // 128 * 128) - (col // 128 * 128 + 127)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    lse, err = torch.zeros((nq, hq), device=DEV).double(), torch.zeros((nq, hq), device=DEV).double()
    for h in range(hq):
        s, a = 0, 0
        for i in range(8):
            d = slice(16 * i, 16 * i + 16)
            on = 1.0 if zhi is None or i == 0 else (near <= zhi[i]).double()
            s = s + q[:, h, d] @ k[:, h * hkv // hq, d].T * on
            a = a + q[:, h, d].abs() @ k[:, h * hkv // hq, d].T.abs() * on
        s = s / math.sqrt(128)
        if causal:
            s = s.masked_fill(col > row + nk - nq, -math.inf)
        lse[:, h] = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1)
        p = torch.where(torch.isneginf(lse[:, h:h + 1]), 0.0, p)
        out[:, h], mag[:, h] = p @ v[:, h * hkv // hq], p @ v[:, h * hkv // hq].abs()
        err[:, h] = a.max(-1).values / math.sqrt(128) * 2.0 ** -17
    return out, mag, lse, err


def _close(out, lse, want):
    ref, mag, rl, err = want
    tol = (2.0 ** -8 + 2 * err[..., None]) * mag + 2.0 ** -8 * ref.abs() + 1e-30
    assert torch.all((out.double() - ref).abs() <= tol), float(((out.double() - ref).abs() / tol).max())
    dead = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse), dead)
    assert torch.all(((lse.double() - rl).abs() <= err + 2.0 ** -18 * (1 + rl.abs()))[~dead])


CASES = [
    (4, 4, [1], [1]),
    (7, 1, [5, 0, 130, 1, 128, 127, 256, 257], None),
    (6, 2, [300, 77, 1, 600], [300, 400, 512, 645]),        # chunks behind cached prefixes
    (24, 8, [129, 1000, 31], None),
    (8, 8, [384, 2], [1025, 4096]),
]


@pytest.mark.parametrize("hq,hkv,nq,nk", CASES)
@pytest.mark.parametrize("window", [None, Z16])
@pytest.mark.parametrize("layout", ["sorted_pair", "rotate_half"])
def test_ragged_rows_are_those_of_the_sequence_alone(hq, hkv, nq, nk, window, layout):
    import atflash
    q, k, v, cq, ck = _packed(nq, nk or nq, hq, hkv, len(nq) + hq)
    got = _run(q, k, v, cq, ck, window_table=window, qk_layout=layout)
    _same_as_alone(got, q, k, v, cq, ck, causal=True, window_table=window, qk_layout=layout)
    if layout == "sorted_pair":
        for b in range(len(nq)):
            if nq[b]:
                sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
                _close(got[0][sq], got[1][sq], _exact(q[sq], k[sk], v[sk], window))
    assert atflash.check_device_errors() == 0


def test_ragged_not_causal_and_scale():
    nq, nk = [40, 300, 1], [200, 77, 513]
    q, k, v, cq, ck = _packed(nq, nk, 6, 3, 2)
    got = _run(q, k, v, cq, ck, causal=False)
    for b in range(3):
        sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        _close(got[0][sq], got[1][sq], _exact(q[sq], k[sk], v[sk], causal=False))
    import atflash
    got = _run(q, k, v, cq, ck, causal=False, sm_scale=0.2)
    for b in (0, 2):  # the dense entry takes no more queries than keys
        sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        o = atflash.prefill_fwd(q[None, sq], k[None, sk], v[None, sk], causal=False, softmax_scale=0.2)
        assert torch.equal(got[0][sq], o[0])


def test_ragged_rows_without_keys():
    """More queries than keys: the first rows see none; sequences without keys."""
    nq, nk = [300, 5, 600, 140, 2], [77, 0, 130, 139, 300]
    q, k, v, cq, ck = _packed(nq, nk, 4, 2, 3)
    for x in (v, k):  # whatever is near, a row without keys is 0
        x[ck[4]:ck[4] + 3] = float("nan")
    out, lse = _run(q, k, v, cq, ck)
    for b in range(4):
        sq, sk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        empty = max(0, nq[b] - nk[b])
        assert torch.count_nonzero(out[sq][:empty]) == 0 and torch.isneginf(lse[sq][:empty]).all()
        if nk[b]:
            _close(out[sq], lse[sq], _exact(q[sq], k[sk], v[sk]))
    # nothing but sequences without keys, and nothing at all
    none = k[:0]
    out, lse = _run(q[:7], none, none, [0, 5, 7], [0, 0, 0])
    assert torch.count_nonzero(out) == 0 and torch.isneginf(lse).all()
    out, lse = _run(q[:0], k[:9], v[:9], [0, 0], [0, 9])
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_ragged_neighbours_do_not_reach_a_sequence(bad):
    nq = [130, 60, 300, 1, 128, 40]
    q, k, v, cq, ck = _packed(nq, nq, 6, 2, 4)
    base = _run(q, k, v, cq, ck)
    for b in (1, 3, 5):
        for x, c in ((q, cq), (k, ck), (v, ck)):
            x[c[b]:c[b + 1]] = bad
    got = _run(q, k, v, cq, ck)
    for b in (0, 2, 4):
        s = slice(cq[b], cq[b + 1])
        assert torch.equal(got[0][s], base[0][s]) and torch.equal(got[1][s], base[1][s])


def test_ragged_many_short_sequences():
    g = np.random.default_rng(5)
    nq = [int(x) for x in g.integers(0, 40, 300)]
    q, k, v, cq, ck = _packed(nq, nq, 8, 2, 5)
    out, lse = _run(q, k, v, cq, ck)
    for b in list(range(0, 300, 37)) + [299]:
        s = slice(cq[b], cq[b + 1])
        if nq[b]:
            _close(out[s], lse[s], _exact(q[s], k[s], v[s]))


def test_ragged_strides_out_stream_graph():
    nq, nk = [200, 33, 129], [200, 50, 300]
    q, k, v, cq, ck = _packed(nq, nk, 4, 2, 6)
    base = _run(q, k, v, cq, ck)
    kv = torch.zeros((sum(nk), 7, 136), dtype=torch.bfloat16, device=DEV)
    kv[:, 1:3, :128], kv[:, 4:6, :128] = k, v
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)  # head-major rows
    out = torch.full((sum(nq), 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((sum(nq), 4), device=DEV)
    import atflash
    w = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
    w.plan(torch.tensor(cq, device=DEV), torch.tensor(ck, device=DEV), 4, 2, 128)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        w.run(qt, kv[:, 1:3, :128], kv[:, 4:6, :128], out=out[:, 1:5], lse=lse)
    st.synchronize()
    assert torch.equal(out[:, 1:5], base[0]) and torch.equal(lse, base[1])
    assert torch.all(out[:, 0] == 7) and torch.all(out[:, 5] == 7)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(qt, kv[:, 1:3, :128], kv[:, 4:6, :128], out=out[:, 1:5], lse=lse)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:, 1:5], base[0])
    o, l2, _ = atflash.flash_attn_varlen_func(q, k, v, torch.tensor(cq), torch.tensor(ck), 200, 300, causal=True,
                                              return_attn_probs=True)
    assert torch.equal(o, base[0]) and torch.equal(l2, base[1].t())


def test_ragged_refusals():
    import atflash
    q, k, v, cq, ck = _packed([20, 30], [20, 30], 4, 2, 7)
    w = atflash.BatchPrefillWithRaggedKVCacheWrapper(DEV)
    with pytest.raises(RuntimeError):
        w.run(q, k, v)
    for bad in (([0, 30, 20], ck), ([1, 20, 50], ck), ([0, 50], ck), ([[0, 20, 50]], ck), ([0.0, 20.0, 50.0], ck), ([0], [0])):
        with pytest.raises(ValueError):
            w.plan(*bad, 4, 2, 128)
    with pytest.raises(ValueError):
        w.plan(cq, ck, 4, 3, 128)
    with pytest.raises(ValueError):
        w.plan(cq, ck, 4, 2, 128, qk_layout="x")
    with pytest.raises(ValueError):
        w.plan(cq, ck, 4, 2, 128, window_table=[4, 5] + [0] * 6)
    with pytest.raises(ValueError):
        w.plan(cq, ck, 4, 2, 128, window_table=[4] * 7 + [-1])
    with pytest.raises(NotImplementedError):
        w.plan(cq, ck, 4, 2, 64)
    w.plan(cq, ck, 4, 2, 128)
    for a in ((q[:-1], k, v), (q, k[:-1], v[:-1]), (q, k, v[:, :1]), (q[:, :2], k, v), (q.cpu(), k, v)):
        with pytest.raises(ValueError):
            w.run(*a)
    with pytest.raises(TypeError):
        w.run(q.float(), k, v)
    with pytest.raises(ValueError):
        w.run(q, k, v, out=torch.empty_like(q).float())
    with pytest.raises(ValueError):
        w.run(q, k, v, lse=torch.empty((4, 50), device=DEV).t())
    odd = torch.zeros((50, 2, 132), dtype=torch.bfloat16, device=DEV)[..., :128]
    with pytest.raises(atflash.AtfError):
        w.run(q, odd, odd)
    with pytest.raises(ValueError):
        atflash.BatchPrefillWithRaggedKVCacheWrapper("cpu")
    for kw in (dict(dropout_p=0.1), dict(window_size=(5, 0)), dict(softcap=1.0), dict(block_table=q)):
        with pytest.raises(NotImplementedError):
            atflash.flash_attn_varlen_func(q, k, v, cq, ck, **kw)
    assert atflash.check_device_errors() == 0
