"""Inputs and 64-bit references for the paged-cache operators' tests.

Caches start out as NaN everywhere, so whatever an operator reads beyond a
sequence's keys shows in its result; page tables hold shuffled pages, and their
unused entries an id far outside the cache."""
import math

import torch

import fmha_native_b200 as fm

UNUSED_PAGE = 1 << 30


def normal(shape, seed, by=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * by).to(torch.bfloat16)


class Problem:
    """Sequences with `new[b]` tokens of which the cache holds `keys[b]` keys,
    the new ones included; optionally `prefix` shared keys before them."""

    def __init__(self, new, keys, hq, hk, page=16, packed=None, prefix=0, heads_first=False, seed=1, spare=3, q_by=1.5):
        self.new, self.keys, self.hq, self.hk, self.page, self.prefix = list(new), list(keys), hq, hk, page, prefix
        b = len(self.new)
        packed = len(set(self.new)) > 1 if packed is None else packed
        self.packed, self.tokens = packed, sum(self.new)
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in self.keys]
        pre = -(-prefix // page)
        pages = sum(need) + pre + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((b, max(need + [1]) + 2), UNUSED_PAGE, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.prefix_pages = order[at:at + pre].clone().cuda()
        self.table = self.table.cuda()
        shape = (pages, hk, page, 64) if heads_first else (pages, page, hk, 64)
        self.k_cache = torch.full(shape, math.nan, dtype=torch.bfloat16, device="cuda")
        self.v_cache = torch.full(shape, math.nan, dtype=torch.bfloat16, device="cuda")
        if heads_first:
            self.k_cache, self.v_cache = self.k_cache.transpose(1, 2), self.v_cache.transpose(1, 2)
        self.k, self.v = [], []
        for i, n in enumerate(self.keys):
            k, v = normal((n, hk, 64), seed * 1000 + 2 * i), normal((n, hk, 64), seed * 1000 + 2 * i + 1)
            self._put(self.table[i], k, v)
            self.k.append(k)
            self.v.append(v)
        if prefix:
            self.pk, self.pv = normal((prefix, hk, 64), seed + 77), normal((prefix, hk, 64), seed + 78)
            self._put(self.prefix_pages, self.pk, self.pv)
        self.seqlens = torch.tensor(self.keys, dtype=torch.int32, device="cuda")
        self.cu = None
        if packed:
            self.cu = torch.tensor([0] + list(torch.tensor(self.new).cumsum(0)), dtype=torch.int32, device="cuda")
            self.q = normal((self.tokens, hq, 64), seed + 5, q_by)
        else:
            self.q = normal((b, self.new[0], hq, 64), seed + 5, q_by)

    def _put(self, pages, k, v):
        n = k.shape[0]
        at = torch.arange(n, device="cuda")
        page = pages[(at // self.page).long()].long()
        self.k_cache[page, at % self.page] = k
        self.v_cache[page, at % self.page] = v

    def run(self, q=None, **kw):
        q = self.q if q is None else q
        kw.setdefault("cu_seqlens_q", self.cu)
        kw.setdefault("max_seqlen_q", max(self.new))
        if self.prefix:
            return fm.prefix_fwd(q, self.k_cache, self.v_cache, self.prefix_pages, self.prefix, self.table, self.seqlens, **kw)
        return fm.paged_fwd(q, self.k_cache, self.v_cache, self.table, self.seqlens, **kw)

    def exact(self, causal=True, scale=0.125):
        """(O, LSE, weighted |V|) in 64 bits: [tokens, hq, 64], [tokens, hq], [tokens, hq, 64]."""
        q = self.q.reshape(-1, self.hq, 64).double()
        o, a = torch.zeros_like(q), torch.zeros_like(q)
        lse = torch.full((q.shape[0], self.hq), -math.inf, dtype=torch.float64, device="cuda")
        g, at = self.hq // self.hk, 0
        for b, n in enumerate(self.new):
            k, v, ahead = self.k[b].double(), self.v[b].double(), self.prefix
            if ahead:
                k, v = torch.cat([self.pk.double(), k]), torch.cat([self.pv.double(), v])
            if n and k.shape[0]:
                k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
                s = torch.einsum("qhd,khd->hqk", q[at:at + n], k) * scale
                if causal:
                    last = ahead + self.keys[b] - n + torch.arange(n, device="cuda")
                    last = last.clamp_min(ahead - 1)
                    s.masked_fill_(torch.arange(k.shape[0], device="cuda") > last[:, None], -math.inf)
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - m.clamp_min(-1e300))
                t = e.sum(-1, keepdim=True)
                p = torch.where(t > 0, e / t, 0.0)
                o[at:at + n] = torch.einsum("hqk,khd->qhd", p, v)
                a[at:at + n] = torch.einsum("hqk,khd->qhd", p, v.abs())
                lse[at:at + n] = (m + t.log()).squeeze(-1).t()
            at += n
        return o, lse, a

    def check(self, causal=True, scale=0.125, lse=True, **kw):
        got = self.run(causal=causal, return_lse=lse, **kw, **({} if scale == 0.125 else {"scale": scale}))
        o, l = got if lse else (got, None)
        assert fm.status() == fm.FMHA_OK
        self.compare(o, l, causal, scale)
        return got

    def compare(self, o, l, causal=True, scale=0.125):
        """Each weight may be rounded to bf16 (8 significant bits: 2^-8 of itself) and
        the output once (2^-8 of itself); scores, exponentials and sums are fp32 (a generous 2^-13).
        The LSE: 64 products of a score err by at most 64 * 2^-24 of the sum of
        their magnitudes (below 16 here), the rest by a few 2^-22: 1e-4."""
        eo, el, ea = self.exact(causal, scale)
        o = o.reshape(-1, self.hq, 64).double()
        assert torch.isfinite(o).all()
        over = (o - eo).abs() - (2.0 ** -8 * (ea + eo.abs()) + 2.0 ** -13 * ea)
        assert over.max().item() <= 0, f"O is off by {(o - eo).abs().max().item()}"
        if l is None:
            return
        l = l.t() if self.packed else l.transpose(1, 2).reshape(-1, self.hq)
        none = torch.isinf(el)
        assert torch.equal(torch.isinf(l), none) and (l[none] < 0).all()
        assert ((l.double() - el)[~none].abs() <= 1e-4).all()
