#!/usr/bin/env python
"""A small serving loop over an e4m3 paged cache: packed prompts, page tables and slot
maps built on the GPU, the append and the decode, as an engine would call them for
one attention layer.

    python examples/serving_step.py [--steps 8] [--window]

The layer's projections are random matrices; what the loop shows is which call feeds
which. `serve` returns every step's attention output, so that a test can compare
them with a plain implementation."""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atflash-kernel_b200"))
import atflash  # noqa: E402

HEAD_DIM = 128


class Layer:
    """One attention layer: q, k, v projections of a hidden state."""

    def __init__(self, hidden, hq, hkv, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.hq, self.hkv = hq, hkv
        self.w = torch.randn((hidden, (hq + 2 * hkv) * HEAD_DIM), generator=g, device=device).bfloat16() / math.sqrt(hidden)

    def qkv(self, x):
        y = (x @ self.w).view(x.shape[0], self.hq + 2 * self.hkv, HEAD_DIM)
        return y[:, :self.hq], y[:, self.hq:self.hq + self.hkv], y[:, self.hq + self.hkv:]


def serve(prompts, steps, *, hq=12, hkv=4, page=16, window=None, rope_base=1e6, device="cuda", seed=0):
    """prompts: a list of (tokens, hidden) bf16 tensors. Returns (prompt output
    (total tokens, hq, 128), [output (B, hq, 128) of each step], state)."""
    dev = torch.device(device)
    B, lens = len(prompts), [p.shape[0] for p in prompts]
    layer = Layer(prompts[0].shape[1], hq, hkv, dev, seed)
    longest = max(lens) + steps
    cos, sin = atflash.cos_sin_table(longest, HEAD_DIM, rope_base, device=dev)

    # the cache: pages, their scales, the engine's table and its free list
    pages = sum(-(-(n + steps) // page) for n in lens)
    cache = [torch.zeros((pages, page, hkv, HEAD_DIM), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.zeros((pages, hkv), device=dev) for _ in range(2)]
    req_pages = torch.full((B, -(-longest // page)), -1, dtype=torch.int32, device=dev)
    free_pages = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(dev)
    free_head = torch.zeros(1, dtype=torch.int32, device=dev)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device=dev)

    def grow(append_lens, new_tokens):
        nonlocal free_head
        max_pages = sum(-(-n // page) for n in lens)
        t = atflash.build_page_tables(kv_lens, append_lens, req_pages, page, num_tokens=new_tokens, max_pages=max_pages,
                                      free_pages=free_pages, free_head=free_head)
        free_head = t.free_head
        return t

    def append(k, v, t):
        atflash.append_paged_kv_cache(k, v, t.batch_indices, t.positions, tuple(cache), t.indices, t.indptr,
                                      kv_scales=tuple(scales), rope=(cos, sin), out_layout="sorted_pair")

    # ---- the prompts: one packed batch
    q, k, v = layer.qkv(torch.cat(prompts))
    t = grow(kv_lens, sum(lens))
    append(k, v, t)
    positions = t.positions.long()
    qr, kr = (atflash.rope_pack(x[None], cos, sin, positions=positions, out_layout="sorted_pair")[0] for x in (q, k))
    prefill = atflash.BatchPrefillWithRaggedKVCacheWrapper(dev)
    prefill.plan(t.append_indptr, t.append_indptr, hq, hkv, HEAD_DIM, causal=True, window_table=window)
    prompt_out = prefill.run(qr, kr, v)

    # ---- decode: every request grows by a token a step
    ones = torch.ones(B, dtype=torch.int32, device=dev)
    decode = atflash.BatchDecodeWithPagedKVCacheWrapper(workspace, "NHD")
    last = torch.tensor([sum(lens[:b + 1]) - 1 for b in range(B)], device=dev)
    x = prompt_out[last].reshape(B, -1)[:, :prompts[0].shape[1]].contiguous()
    outs, inputs = [], []
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        kv_lens = kv_lens + 1
        inputs.append(x)
        q, k, v = layer.qkv(x)
        t = grow(ones, B)
        append(k, v, t)
        qr = atflash.rope_pack(q[None], cos, sin, positions=t.positions.long(), out_layout="sorted_pair")[0]
        # (a step's tables are on the GPU; the decode's schedule is built on the host)
        decode.plan(t.indptr, t.indices, t.last_page_len, hq, hkv, HEAD_DIM, page, kv_data_type=torch.float8_e4m3fn,
                    window_table=window)
        out = decode.run(qr, tuple(cache), kv_scales=tuple(scales))
        outs.append(out)
        x = out.reshape(B, -1)[:, :x.shape[1]].contiguous()
    state = dict(layer=layer, cos=cos, sin=sin, cache=cache, scales=scales, tables=t, kv_lens=kv_lens, inputs=inputs)
    return prompt_out, outs, state


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--window", action="store_true", help="windows of 2 wavelengths (rope base 1e6)")
    a = ap.parse_args()
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [700, 33, 1, 2048, 129]
    prompts = [torch.randn((n, 512), generator=g, device="cuda").bfloat16() for n in lens]
    window = atflash.WindowTable(HEAD_DIM, 1e6, 2.0) if a.window else None
    prompt_out, outs, state = serve(prompts, a.steps, window=window)
    assert atflash.check_device_errors() == 0
    used = sum(c.numel() for c in state["cache"]) + sum(4 * s.numel() for s in state["scales"])
    print(f"{len(lens)} prompts, {sum(lens)} tokens: output {tuple(prompt_out.shape)}; {a.steps} steps of {tuple(outs[0].shape)}; "
          f"cache {used / 1e6:.1f} MB (bf16: {2 * used / 1e6:.1f} MB)")


if __name__ == "__main__":
    main()
