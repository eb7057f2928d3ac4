"""NaN and infinities among what a query row sees: they reach its result, and
only its, whichever kernel, key range and column they fall to."""
import math

import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


# Single tokens and drafts (also with keys that blocks share), chunks whose key
# ranges are shared out, prompts whose work is listed, all of it under a prefix.
CASES = {
    "token": dict(new=[1, 1], keys=[300, 40], hq=8, hk=2),
    "long_token": dict(new=[1], keys=[20001], hq=8, hk=2),
    "drafts": dict(new=[3, 3], keys=[300, 500], hq=4, hk=2),
    "chunk": dict(new=[40, 40], keys=[600, 300], hq=8, hk=2),
    "long_chunk": dict(new=[33], keys=[9000], hq=4, hk=1),
    "prompts": dict(new=[1500, 1500], keys=[1700, 1500], hq=16, hk=16, page=64),
    "mixed": dict(new=[40, 1, 5], keys=[600, 90, 200], hq=8, hk=2),
    "prefix": dict(new=[1] * 5, keys=[300, 1, 0, 77, 200], hq=8, hk=2, prefix=1000),
    "prefix_long_token": dict(new=[1, 1], keys=[9000, 40], hq=4, hk=1, prefix=300),
    "prefix_chunk": dict(new=[40, 70], keys=[300, 300], hq=8, hk=2, prefix=700),
}


def problem(name):
    return Problem(**CASES[name], seed=3)


def flat(p, o, lse):
    o = o.reshape(-1, p.hq, 64).double()
    return o, (lse.t() if p.packed else lse.transpose(1, 2).reshape(-1, p.hq)).double()


def close(o, lse, eo, el, ea, rows):
    """The bounds of Problem.compare, at `rows` ([tokens, heads])."""
    over = (o - eo).abs() - (2.0 ** -8 * (ea + eo.abs()) + 2.0 ** -13 * ea)
    same_lse = (lse == el) | ((lse - el).abs() <= 1e-4)
    return bool((over[rows] <= 0).all()) and bool(same_lse[rows].all())


def put(p, b, at, head, k=None, v=None, dim=5):
    """Into key `at` of sequence b (None: of the prefix)."""
    keys, values, pages = (p.pk, p.pv, p.prefix_pages) if b is None else (p.k[b], p.v[b], p.table[b])
    if k is not None:
        keys[at, head, dim] = k
    if v is not None:
        values[at, head, dim] = v
    p._put(pages, keys, values)


def sees(p, b, at):
    """[tokens]: which tokens see key `at` of sequence b (None: of the prefix)."""
    if b is None:
        return torch.ones(p.tokens, dtype=torch.bool, device="cuda")
    n, first = p.new[b], sum(p.new[:b])
    t = torch.arange(p.tokens, device="cuda") - first
    return (t >= 0) & (t < n) & (at <= p.keys[b] - n + t)


def group_of(p, head):
    h = torch.arange(p.hq, device="cuda")
    return h // (p.hq // p.hk) == head


@pytest.mark.parametrize("name", CASES)
def test_nan_in_a_key(name):
    """At every position modulo 16, of the sequence's first keys and of the prefix's."""
    p = problem(name)
    eo, el, ea = p.exact()
    for b in [0] + ([None] if p.prefix else []):
        k = p.pk if b is None else p.k[b]
        for at in range(64, 80):
            head = at % p.hk
            keep = k[at].clone()
            put(p, b, at, head, k=math.nan)
            o, lse = flat(p, *p.run(return_lse=True))
            k[at] = keep
            rows = sees(p, b, at)[:, None] & group_of(p, head)
            where = f"{'prefix' if b is None else 'sequence'} key {at}"
            assert rows.any() and torch.isnan(o[rows]).all() and torch.isnan(lse[rows]).all(), where
            assert close(o, lse, eo, el, ea, ~rows), where
        put(p, b, 64, 0)
    assert fm.status() == fm.FMHA_OK


@pytest.mark.parametrize("name", CASES)
def test_nan_in_a_query(name):
    p = problem(name)
    eo, el, ea = p.exact()
    rows = torch.zeros(p.tokens, p.hq, dtype=torch.bool, device="cuda")
    for token, head in ((0, 1), (p.tokens - 1, p.hq - 1)):
        rows[token, head] = True
    p.q.view(-1, p.hq, 64)[..., 9][rows] = math.nan
    o, lse = flat(p, *p.run(return_lse=True))
    assert torch.isnan(o[rows]).all() and torch.isnan(lse[rows]).all()
    assert close(o, lse, eo, el, ea, ~rows)


def formula(p):
    """Problem.exact with whatever the formula gives (causal): NaN where a row has no softmax."""
    q = p.q.reshape(-1, p.hq, 64).double()
    o, a = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((q.shape[0], p.hq), -math.inf, dtype=torch.float64, device="cuda")
    g, first = p.hq // p.hk, 0
    for b, n in enumerate(p.new):
        k, v = p.k[b].double(), p.v[b].double()
        if p.prefix:
            k, v = torch.cat([p.pk.double(), k]), torch.cat([p.pv.double(), v])
        for i in range(n):
            seen = p.prefix + max(0, p.keys[b] - n + i + 1)
            if seen:
                s = torch.einsum("hd,khd->hk", q[first + i], k[:seen].repeat_interleave(g, 1)) * 0.125
                w = torch.exp(s - s.amax(-1, keepdim=True))
                lse[first + i] = s.amax(-1) + w.sum(-1).log()
                w = w / w.sum(-1, keepdim=True)
                x = v[:seen].repeat_interleave(g, 1)
                o[first + i], a[first + i] = torch.einsum("hk,khd->hd", w, x), torch.einsum("hk,khd->hd", w, x.abs())
        first += n
    return o, lse, a


@pytest.mark.parametrize("at", [64, 70, 71, 77])
@pytest.mark.parametrize("name", [n for n in CASES if n != "prompts"])
def test_infinite_key(name, at):
    """A row with score +inf has no softmax (inf - inf): NaN.  Score -inf: weight 0."""
    p = problem(name)
    for b in [0] + ([None] if p.prefix else []):
        put(p, b, at, 0, k=math.inf)
        o, lse = flat(p, *p.run(return_lse=True))
        hit = sees(p, b, at)[:, None] & group_of(p, 0) & (p.q.view(-1, p.hq, 64)[..., 5] > 0)
        eo, el, ea = formula(p)
        assert torch.equal(torch.isnan(el), hit) and hit.any()
        assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
        assert close(o, lse, eo, el, ea, ~hit)
        put(p, b, at, 0, k=0.25)
