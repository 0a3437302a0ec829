#!/usr/bin/env python
"""Several continuations of each prompt over one paged cache: prompts prefilled in chunks
over the cache's pages, forked (pages shared, the last partial page copied in every
layer), grown a few tokens at a time, freed and compacted, as an engine would call
it for layers with norms of their q and k heads.

    python examples/shared_prefix.py [--each 4] [--steps 4] [--window]

With --window the scores depend a little on where chunks begin, as
BatchPrefillWithPagedKVCacheWrapper says.

The layers' projections are random matrices; what the loop shows is which call feeds
which. `Engine` keeps what each request's tokens were projected to, so that a test can
compare every output with a plain implementation."""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atflash-kernel_b200"))
import atflash  # noqa: E402

HEAD_DIM = 128


class Layer:
    """One attention layer: projections of a hidden state, norms of the q and k heads, and
    its pages of the cache."""

    def __init__(self, hidden, hq, hkv, pages, page, device, seed):
        g = torch.Generator(device=device).manual_seed(seed)
        self.hq, self.hkv = hq, hkv
        self.w = torch.randn((hidden, (hq + 2 * hkv) * HEAD_DIM), generator=g, device=device).bfloat16() / math.sqrt(hidden)
        self.qw, self.kw = (1 + 0.2 * torch.randn(HEAD_DIM, generator=g, device=device) for _ in range(2))
        self.k, self.v = (torch.zeros((pages, page, hkv, HEAD_DIM), dtype=torch.bfloat16, device=device) for _ in range(2))

    def qkv(self, x):
        y = (x @ self.w).view(x.shape[0], self.hq + 2 * self.hkv, HEAD_DIM)
        return y[:, :self.hq], y[:, self.hq:self.hq + self.hkv], y[:, self.hq + self.hkv:]


class Engine:
    """Requests in the rows of a page table. `lens` (host) is each row's tokens."""

    def __init__(self, hidden=256, hq=12, hkv=4, page=16, pages=256, rows=32, layers=2, longest=1024, eps=1e-6,
                 window=None, rope_base=1e6, device="cuda", seed=0):
        dev = self.dev = torch.device(device)
        self.hq, self.hkv, self.page, self.pages, self.eps, self.window = hq, hkv, page, pages, eps, window
        self.layers = [Layer(hidden, hq, hkv, pages, page, dev, seed + i) for i in range(layers)]
        self.copier = atflash.PageCopier([t for layer in self.layers for t in (layer.k, layer.v)])
        self.cos, self.sin = atflash.cos_sin_table(longest, HEAD_DIM, rope_base, device=dev)
        self.req_pages = torch.full((rows, -(-longest // page)), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(dev)
        self.free_head = torch.zeros(1, dtype=torch.int32, device=dev)
        self.shared = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.attention = atflash.BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=dev))
        self.lens, self.history = {}, {}

    def _i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def step(self, tokens):
        """tokens: {row: (n, hidden) bf16}, a decode (n = 1), a draft or a chunk of a prompt
        each. Returns {row: [output (n, hq, 128) of each layer]}."""
        rows, new = list(tokens), [t.shape[0] for t in tokens.values()]
        for r, n in zip(rows, new):
            self.lens[r] = self.lens.get(r, 0) + n
        lens = [self.lens[r] for r in rows]
        t = atflash.build_page_tables(self._i32(lens), self._i32(new), self.req_pages, self.page, num_tokens=sum(new),
                                      max_pages=sum(-(-n // self.page) for n in lens), req_rows=self._i32(rows),
                                      free_pages=self.free_pages, free_head=self.free_head)
        self.free_head = t.free_head
        # one plan for all layers
        self.attention.plan(t.append_indptr, t.indptr, t.indices, t.last_page_len, self.hq, self.hkv, HEAD_DIM, self.page,
                            causal=True, window_table=self.window)
        x = torch.cat(list(tokens.values()))
        at = [0]
        for n in new:
            at.append(at[-1] + n)
        out = {r: [] for r in rows}
        for i, layer in enumerate(self.layers):
            q, k, v = layer.qkv(x)
            atflash.append_paged_kv_cache(k, v, t.batch_indices, t.positions, (layer.k, layer.v), t.indices, t.indptr,
                                          rope=(self.cos, self.sin), k_norm=(layer.kw, self.eps))
            qr, _ = atflash.qk_norm_rope(q, None, layer.qw, None, self.cos, self.sin, eps=self.eps, positions=t.positions,
                                         out_layout="sorted_pair")
            o = self.attention.run(qr, (layer.k, layer.v))
            for j, r in enumerate(rows):
                part = slice(at[j], at[j + 1])
                out[r].append(o[part])
                self.history.setdefault(r, [[] for _ in self.layers])[i].append((q[part], k[part], v[part]))
        return out

    def fork(self, parents, children, lens=None):
        """Children of running requests, from their first lens[i] tokens (default all)."""
        lens = [self.lens[p] for p in parents] if lens is None else lens
        f = atflash.fork_requests(self._i32(parents), self._i32(children), self._i32(lens), self.req_pages, self.page,
                                  free_pages=self.free_pages, free_head=self.free_head, shared=self.shared)
        self.free_head = f.free_head
        self.copier.copy(f.src, f.dst)
        for p, c, n in zip(parents, children, lens):
            self.lens[c] = n
            self.history[c] = []
            for h in self.history[p]:
                q, k, v = (torch.cat([x[j] for x in h])[:n] for j in range(3))
                self.history[c].append([(q, k, v)])

    def free(self, rows):
        self.free_head = atflash.free_requests(self._i32(rows), self._i32([self.lens[r] for r in rows]), self.req_pages,
                                               self.page, free_pages=self.free_pages, free_head=self.free_head,
                                               shared=self.shared)
        for r in rows:
            del self.lens[r], self.history[r]

    def compact(self, max_moves=None):
        """Afterwards the pages in use are the cache's first."""
        rows = list(self.lens)
        m = atflash.compact_pages(self._i32([self.lens[r] for r in rows]), self.req_pages, self.page, self.pages,
                                  max_moves=self.pages if max_moves is None else max_moves, req_rows=self._i32(rows),
                                  free_pages=self.free_pages, shared=self.shared)
        self.free_head = m.free_head
        self.copier.copy(m.src, m.dst)

    def pages_in_use(self):
        return self.pages - int(self.free_pages.numel() - self.free_head)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--each", type=int, default=4, help="continuations of a prompt")
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--window", action="store_true", help="windows of 2 wavelengths (rope base 1e6)")
    a = ap.parse_args()
    e = Engine(rows=3 + 3 * a.each, window=atflash.WindowTable(HEAD_DIM, 1e6, 2.0) if a.window else None)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda n: torch.randn((n, 256), generator=g, device="cuda").bfloat16()
    prompts = {0: 333, 1: 96, 2: 50}
    for lo in range(0, 333, 128):  # chunks of up to 128 tokens
        e.step({r: rand(min(n - lo, 128)) for r, n in prompts.items() if n > lo})
    print(f"3 prompts: {e.pages - e.pages_in_use()} of {e.pages} pages free")
    parents = [r for r in prompts for _ in range(a.each)]
    children = list(range(3, 3 + len(parents)))
    e.fork(parents, children)
    e.free(list(prompts))
    print(f"{len(children)} continuations instead: {e.pages - e.pages_in_use()} free")
    for _ in range(a.steps):
        out = e.step({r: rand(1 + r % 3) for r in children})
    e.free(children[::2])
    e.compact()
    out = e.step({r: rand(1) for r in e.lens})
    assert atflash.check_device_errors() == 0
    print(f"{len(out)} left after {a.steps} steps: {e.pages - e.pages_in_use()} free; output {tuple(next(iter(out.values()))[0].shape)}")


if __name__ == "__main__":
    main()
