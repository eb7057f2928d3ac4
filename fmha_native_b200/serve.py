"""A small serving loop over the paged operators, as they are used together.

Requests under one shared system prompt: the prompt enters the cache once, the
requests' own prompts (text, or image patches with time/height/width positions)
follow packed, then every request decodes one token a step.  Each layer of the
stand-in model projects, appends its rotated K and V to the pages
(:func:`paged_append`) and attends (:func:`paged_fwd` for the system prompt,
:func:`prefix_fwd` for the requests).  Weights and inputs are random.

    python -m fmha_native_b200.serve --requests 16 --prefix 2000 --steps 32
"""
from __future__ import annotations

import argparse
import time

import torch

import fmha_native_b200 as fm

SECTIONS = (8, 12, 12)  # pairs turned by time, height and width


class PagedKV:
    """K/V pages of all layers and the sequences' page tables.

    Pages are handed out on the host; the device sees ``table`` ([slots,
    max_pages] int32) and ``lengths`` ([slots] int32).
    """

    def __init__(self, layers: int, pages: int, page: int, heads_k: int, slots: int, max_pages: int, device):
        shape = (layers, pages, page, heads_k, fm.HEAD_DIM)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.page, self.free = page, list(range(pages))
        self.host_table = torch.zeros(slots, max_pages, dtype=torch.int32)
        self.owned = [[] for _ in range(slots)]
        self.host_lengths = [0] * slots
        self.table = self.host_table.to(device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=device)

    def pages_for(self, tokens: int) -> list[int]:
        need = -(-tokens // self.page)
        if need > len(self.free):
            raise fm.FmhaError(fm.FMHA_ERR_ARG, f"the cache is out of pages ({need} wanted, {len(self.free)} free)")
        return [self.free.pop() for _ in range(need)]

    def extend(self, new: list[int]) -> None:
        """Makes room for new[i] tokens in slot i; lengths then include them.  All of it or none."""
        need = [-(-(self.host_lengths[i] + n) // self.page) for i, n in enumerate(new)]
        if max(need) > self.host_table.shape[1]:
            raise fm.FmhaError(fm.FMHA_ERR_ARG, f"a sequence of {max(need)} pages, {self.host_table.shape[1]} at most")
        pages = self.pages_for(self.page * sum(max(0, n - len(own)) for n, own in zip(need, self.owned)))
        for i, n in enumerate(new):
            while len(self.owned[i]) < need[i]:
                self.owned[i].append(pages.pop(0))
                self.host_table[i, len(self.owned[i]) - 1] = self.owned[i][-1]
            self.host_lengths[i] += n
        self.table.copy_(self.host_table, non_blocking=True)
        self.lengths.copy_(torch.tensor(self.host_lengths, dtype=torch.int32), non_blocking=True)

    def release(self, slot: int) -> None:
        self.free += self.owned[slot]
        self.owned[slot], self.host_lengths[slot] = [], 0


class Layer:
    def __init__(self, width: int, heads_q: int, heads_k: int, generator, device):
        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=generator, device=device) * rows ** -0.5).to(torch.bfloat16)

        self.heads_q, self.heads_k = heads_q, heads_k
        self.qkv = weight(width, (heads_q + 2 * heads_k) * fm.HEAD_DIM)
        self.out = weight(heads_q * fm.HEAD_DIM, width)

    def project(self, x):
        """Q, K, V as views of one projection (the operators take its strides)."""
        y = (x @ self.qkv).unflatten(-1, (-1, fm.HEAD_DIM))
        return y.split([self.heads_q, self.heads_k, self.heads_k], dim=-2)


class Server:
    """`slots` requests at once under one system prompt."""

    def __init__(self, *, layers=2, width=512, heads_q=8, heads_k=2, page=16, slots=16, max_len=4096, prefix_len=2000,
                 device="cuda", seed=0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.layers = [Layer(width, heads_q, heads_k, g, device) for _ in range(layers)]
        self.width, self.slots, self.prefix_len, self.device, self.generator = width, slots, prefix_len, device, g
        per_slot = -(-max_len // page)
        self.kv = PagedKV(layers, slots * per_slot + -(-prefix_len // page), page, heads_k, slots, per_slot, device)
        self.angles = fm.rope_table(prefix_len + max_len, device=device)
        self.prefix_pages = torch.tensor(self.kv.pages_for(prefix_len), dtype=torch.int32, device=device)
        self._enter_prefix()

    def embed(self, *tokens):
        return torch.randn(*tokens, self.width, generator=self.generator, device=self.device).to(torch.bfloat16)

    def _enter_prefix(self):
        """The system prompt, as one sequence whose page table is the prefix's."""
        n, x = self.prefix_len, self.embed(1, self.prefix_len)
        table, length = self.prefix_pages[None], torch.tensor([n], dtype=torch.int32, device=self.device)
        for i, layer in enumerate(self.layers):
            q, k, v = layer.project(x)
            q = fm.paged_append(k, v, self.kv.k[i], self.kv.v[i], table, length, q=q, cos_sin=self.angles)
            o = fm.paged_fwd(q, self.kv.k[i], self.kv.v[i], table, length)
            x = x + o.flatten(-2) @ layer.out

    def step(self, x, positions, cu_seqlens=None, max_new=1):
        """All layers over new tokens, whose room extend() has made: x is
        [slots, n, width] or packed [total, width]; positions [3, ...]."""
        trace = []
        for i, layer in enumerate(self.layers):
            q, k, v = layer.project(x)
            kc, vc = self.kv.k[i], self.kv.v[i]
            q = fm.paged_append(k, v, kc, vc, self.kv.table, self.kv.lengths, q=q, cos_sin=self.angles,
                                positions=positions, sections=SECTIONS, cu_seqlens_q=cu_seqlens)
            o = fm.prefix_fwd(q, kc, vc, self.prefix_pages, self.prefix_len, self.kv.table, self.kv.lengths,
                              cu_seqlens_q=cu_seqlens, max_seqlen_q=max_new)
            trace.append((q, o))
            x = x + o.flatten(-2) @ layer.out
        return x, trace

    def prompts(self, lengths: list[int], images: list[int]):
        """The requests' prompts: `images[i]` of the lengths[i] tokens are patches of a
        square image, placed by row and column."""
        self.kv.extend(lengths)
        cu = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        rows = []
        for n, m in zip(lengths, images):
            at = torch.arange(n)
            p = at.repeat(3, 1)  # text: the same position on every axis
            side = max(1, int(m ** 0.5))
            p[0, :m] = 0
            p[1, :m], p[2, :m] = at[:m] // side, at[:m] % side
            rows.append(p + self.prefix_len)
        positions = torch.cat(rows, 1).to(torch.int32).to(self.device)
        return self.step(self.embed(sum(lengths)), positions, cu.to(self.device), max(lengths))

    def decode(self):
        """One token more for every request."""
        self.kv.extend([1] * self.slots)
        place = (self.kv.lengths - 1 + self.prefix_len)[:, None]
        return self.step(self.embed(self.slots, 1), place.expand(3, -1, -1).contiguous())


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prefix", type=int, default=2000)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args(argv)
    srv = Server(layers=a.layers, slots=a.requests, prefix_len=a.prefix, max_len=1024 + a.steps)
    srv.prompts([64 + (i * 97) % 900 for i in range(a.requests)], [(i % 3) * 16 for i in range(a.requests)])
    srv.decode()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        _, trace = srv.decode()
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    if fm.status() != fm.FMHA_OK:
        raise fm.FmhaError(fm.FMHA_ERR_INDEX, "serve")
    out = {"requests": a.requests, "prefix": a.prefix, "tokens_per_s": a.requests * a.steps / dt,
           "us_per_step": dt / a.steps * 1e6}
    print(f"{a.requests} requests under {a.prefix} shared tokens, {a.layers} layers: "
          f"{out['us_per_step']:.0f} us a step, {out['tokens_per_s']:.0f} tokens/s")
    return out


if __name__ == "__main__":
    main()
