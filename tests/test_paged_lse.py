"""How exact the LSE of the attention over pages is."""
import math

import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


@pytest.mark.parametrize("new, prefix, group", [(1, 0, 1), (1, 0, 8), (40, 0, 2), (700, 0, 1), (1, 300, 1), (40, 300, 2)])
def test_one_key_dominates(new, prefix, group):
    """Score 16 at one key and 0 at the others, at every position modulo 16.

    All products and sums of the scores are exact.  In units of log2 the LSE is
    23.1: the scale (2^-24 of it), the reference's product, the sum with the
    logarithm and, under a prefix, the fold round to 2^-24 of it each (at most 6
    times: 8.3e-6 * ln 2 = 5.7e-6); the exponentials and the logarithm err by a
    few 2^-22 (7e-7); the last product by 2^-24 of 16 (1e-6).  Below 1e-5."""
    keys = 900
    p = Problem([new], [keys], 2 * group, 2, page=64, prefix=prefix)
    p.q.fill_(1.0)
    k, pages = (p.pk, p.prefix_pages) if prefix else (p.k[0], p.table[0])
    v = p.pv if prefix else p.v[0]
    if prefix:
        p.k[0].zero_()
        p._put(p.table[0], p.k[0], p.v[0])
    for at in range(32, 48):
        k.zero_()
        k[at] = 2.0
        p._put(pages, k, v)
        o, lse = p.run(return_lse=True)
        seen = prefix + keys - new + 1 + torch.arange(new, device="cuda", dtype=torch.float64)
        want = torch.log(math.exp(16.0) + seen - 1)
        assert (lse.double().view(2 * group, new) - want).abs().max() <= 1e-5, f"key {at}"
    assert fm.status() == fm.FMHA_OK
