"""Index data that is out of range: reported, and nothing written but the
call's own results and scratch."""
import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import normal

pytestmark = pytest.mark.gpu

GUARD = 1 << 16


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


class Guarded:
    """Caches, scratch and output with guards around what a call may write."""

    def __init__(self, cu, most, tokens, hq, hk, keys, prefix=0, fill=7, page=16):
        batch = len(cu) - 1
        self.most, self.prefix, self.hq, self.hk = most, prefix, hq, hk
        pages = -(-max(max(keys), prefix, 1) // page)
        self.k, self.v = normal((pages, page, hk, 64), 1), normal((pages, page, hk, 64), 2)
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
        self.lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        self.q = normal((tokens, hq, 64), 3)
        n = fm.paged_workspace_bytes(batch, most, hq, hk, tokens, prefix)
        self.space = torch.full((n // 4 + 2 * GUARD,), fill, dtype=torch.int32, device="cuda")
        self.work = self.space[GUARD:-GUARD].view(torch.uint8)
        self.rows = torch.full((tokens * hq * 64 + 2 * GUARD,), 3.0, dtype=torch.bfloat16, device="cuda")
        self.o = self.rows[GUARD:-GUARD].view(tokens, hq, 64)
        self.sums = torch.full((tokens * hq + 2 * GUARD,), 3.0, device="cuda")
        self.lse = self.sums[GUARD:-GUARD].view(hq, tokens)
        self.fill = fill

    def run(self):
        kw = dict(cu_seqlens_q=self.cu, max_seqlen_q=self.most, out=self.o, lse_out=self.lse, return_lse=True,
                  workspace=self.work)
        if self.prefix:
            fm.prefix_fwd(self.q, self.k, self.v, self.table[0], self.prefix, self.table, self.lengths, **kw)
        else:
            fm.paged_fwd(self.q, self.k, self.v, self.table, self.lengths, **kw)
        status = fm.status()
        for buf, v in ((self.space, self.fill), (self.rows, 3.0), (self.sums, 3.0)):
            assert (buf[:GUARD] == v).all() and (buf[-GUARD:] == v).all()
        return status


OVERLAPS = {
    # one long sequence among many short ones, all of them over the same 40 tokens
    "planned_by_every_block": dict(cu=[0, 40] * 100 + [0], most=40, tokens=40, hq=4, hk=4, keys=[12800] + [128] * 199),
    "few": dict(cu=[0, 40, 0, 40], most=40, tokens=40, hq=4, hk=2, keys=[300, 50, 600]),
    "listed": dict(cu=[0, 1500] * 30 + [0], most=1500, tokens=1500, hq=8, hk=8, keys=[5000] + [1500] * 59),
    "listed_long": dict(cu=[0, 1500] * 200 + [0], most=1500, tokens=1500, hq=16, hk=16, keys=[9000] * 400),
    "rows": dict(cu=[0, 9] * 300 + [0], most=9, tokens=9, hq=4, hk=4, keys=[700] + [90] * 599),
    "both": dict(cu=[0, 40, 38] * 100 + [0], most=40, tokens=40, hq=4, hk=4, keys=[3000] + [128] * 299),
}


@pytest.mark.parametrize("fill", [0, 1, 7, -1])
@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("name", OVERLAPS)
def test_prefix_sums_that_decrease(name, prefix, fill):
    """More row tiles than the tokens have: whatever the scratch held before, no
    block folds what no block wrote."""
    g = Guarded(**OVERLAPS[name], prefix=prefix, fill=fill)
    assert g.run() == fm.FMHA_ERR_INDEX
    good = dict(OVERLAPS[name], cu=[0, g.most], keys=OVERLAPS[name]["keys"][:1])
    assert Guarded(**good, prefix=prefix, fill=fill).run() == fm.FMHA_OK


@pytest.mark.parametrize("name", ["planned_by_every_block", "listed"])
def test_overlapping_tiles_are_left_alone(name):
    g = Guarded(**OVERLAPS[name])
    assert g.run() == fm.FMHA_ERR_INDEX
    assert (g.o == 3.0).all() and (g.lse == 3.0).all()


@pytest.mark.parametrize("cu", [[-5, 35, 40], [0, 41, 40], [0, 2 ** 31 - 1, 40], [-2 ** 31, 2 ** 31 - 1, 0], [40, 0, 40]], ids=str)
@pytest.mark.parametrize("hq", [1, 4, 16])
def test_prefix_sums_that_leave_the_tokens(cu, hq):
    g = Guarded(cu, 40, 40, hq, 1, [500, 700])
    assert g.run() == fm.FMHA_ERR_INDEX


@pytest.mark.parametrize("new, prefix", [(1, 0), (40, 0), (1, 100), (40, 100)])
def test_a_cache_of_no_pages_is_not_read(new, prefix):
    """Page id 0 of a cache that has no pages: reported, zeros instead of what lies there."""
    import ctypes

    batch, hq, hk, page = 2, 4, 2, 16
    k, v = normal((16, page, hk, 64), 1), normal((16, page, hk, 64), 2)
    table = torch.zeros(batch, 16, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([90, 200], dtype=torch.int32, device="cuda")
    q = normal((batch, new, hq, 64), 3)
    o = torch.full_like(q, 3.0)
    n = fm.paged_workspace_bytes(batch, new, hq, hk, 0, prefix)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    p = fm.FmhaPagedParams()
    for name, t in (("q", q), ("k_cache", k), ("v_cache", v), ("o", o), ("page_table", table), ("seqlens_k", lengths),
                    ("prefix_pages", table), ("workspace", work)):
        setattr(p, name, t.data_ptr())
    p.workspace_bytes = n
    for t in ("q", "o"):
        for name, s in (("stride", hq * 64), ("nhead_stride", 64), ("batch_stride", new * hq * 64)):
            setattr(p, f"{name}_{t}", s)
    for t in ("k", "v"):
        for name, s in (("stride", hk * 64), ("nhead_stride", 64), ("page_stride", page * hk * 64)):
            setattr(p, f"{name}_{t}", s)
    p.batch, p.seqlen_q, p.nhead_q, p.nhead_k = batch, new, hq, hk
    p.page_size, p.num_pages, p.max_pages, p.table_stride, p.prefix_len, p.causal, p.scale = page, 0, 16, 16, prefix, 1, 0.18
    lib = fm.load_library()
    call = lib.fmha_prefix_fwd_d64_bf16 if prefix else lib.fmha_paged_fwd_d64_bf16
    assert call(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == fm.FMHA_OK
    assert fm.status() == fm.FMHA_ERR_INDEX
    assert not o.any()
    p.num_pages = 16
    assert call(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == fm.FMHA_OK
    assert fm.status() == fm.FMHA_OK and o.any()
