"""NaN and infinities among the values: they reach the rows that see their key
and no others."""
import math

import pytest
import torch

import fmha_native_b200 as fm
from test_paged_nonfinite import CASES, close, flat, group_of, problem, put, sees
from paged_harness import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("name", CASES)
def test_value_that_all_rows_see(name, bad):
    p = problem(name)
    eo, el, ea = p.exact()
    put(p, 0, 70, p.hk - 1, v=bad)
    o, lse = flat(p, *p.run(return_lse=True))
    rows = sees(p, 0, 70)[:, None] & group_of(p, p.hk - 1)
    assert (torch.isnan if math.isnan(bad) else torch.isposinf)(o[rows][..., 5]).all()
    o[..., 5] = torch.where(rows, eo[..., 5], o[..., 5])
    assert close(o, lse, eo, el, ea, torch.ones_like(rows))


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("new", [5, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_that_see_nothing_are_zero(bad, new, prefix):
    """Beside rows that see an infinite or NaN value: O = 0 and LSE = -inf, or what the prefix gives."""
    p = Problem([new, new], [new - 2, 300], 8, 2, prefix=prefix, seed=4)
    eo, el, ea = p.exact()
    for head in range(2):
        put(p, 0, 0, head, v=bad)
    o, lse = flat(p, *p.run(return_lse=True))
    blind = torch.zeros(p.tokens, p.hq, dtype=torch.bool, device="cuda")
    blind[:2] = True
    if not prefix:
        assert not o[blind].any() and torch.isneginf(lse[blind]).all()
    assert close(o, lse, eo, el, ea, blind)


# Positions of the keys of sequence 0 that some tokens see and some do not.
PARTLY_SEEN = {name: c for name, c in CASES.items() if c["new"][0] > 1}


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("name", PARTLY_SEEN)
def test_value_that_some_rows_see(name, bad):
    n, keys = CASES[name]["new"][0], CASES[name]["keys"][0]
    for at in sorted({keys - 1, keys - n // 2, keys - n + 1}):
        p = problem(name)
        eo, el, ea = p.exact()
        head = at % p.hk
        put(p, 0, at, head, v=bad, dim=37)
        o, lse = flat(p, *p.run(return_lse=True))
        rows = sees(p, 0, at)[:, None] & group_of(p, head)
        assert rows.any()
        hit = o[rows][..., 37]
        assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all(), f"key {at}"
        o[..., 37] = torch.where(rows, eo[..., 37], o[..., 37])
        assert close(o, lse, eo, el, ea, torch.ones_like(rows)), f"key {at}"


@pytest.mark.parametrize("name", PARTLY_SEEN)
def test_both_infinities(name):
    """Their sum is NaN where both are seen."""
    n, keys = CASES[name]["new"][0], CASES[name]["keys"][0]
    p = problem(name)
    eo, el, ea = p.exact()
    put(p, 0, keys - 1, 0, v=math.inf)
    put(p, 0, keys - 2, 0, v=-math.inf)
    o, lse = flat(p, *p.run(return_lse=True))
    both = sees(p, 0, keys - 1)[:, None] & group_of(p, 0)
    one = sees(p, 0, keys - 2)[:, None] & group_of(p, 0) & ~both
    assert torch.isnan(o[both][..., 5]).all() and torch.isneginf(o[one][..., 5]).all()
    o[..., 5] = torch.where(both | one, eo[..., 5], o[..., 5])
    assert close(o, lse, eo, el, ea, torch.ones_like(both))


@pytest.mark.parametrize("new, keys, hq, hk", [(4, 40, 4, 2), (16, 100, 1, 1), (3, 33, 15, 3), (130, 300, 2, 2), (257, 257, 3, 1)])
@pytest.mark.parametrize("page", [8, 32, 256])
def test_whole_keys_that_nobody_else_sees(new, keys, hq, hk, page):
    """Every value of the last token's key is NaN, as a token that failed leaves it: only its own rows are."""
    p = Problem([new, new], [keys, keys + 31], hq, hk, page=page, seed=6)
    eo, el, ea = p.exact()
    for b in range(2):
        p.v[b][-1] = math.nan
        p._put(p.table[b], p.k[b], p.v[b])
    o, lse = flat(p, *p.run(return_lse=True))
    last = torch.zeros(2 * new, hq, dtype=torch.bool, device="cuda")
    last[new - 1], last[-1] = True, True
    assert torch.isnan(o[last]).all()
    assert close(o, lse, eo, el, ea, ~last)
    assert bool(((lse - el).abs() <= 1e-4).all())
