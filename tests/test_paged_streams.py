"""Calls on a named stream (``stream=``): their scratch and their results are
that stream's, whatever the caller's own stream does meanwhile."""
import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import Problem, normal

pytestmark = pytest.mark.gpu

PROBLEMS = {
    "rows": dict(new=[1] * 3, keys=[7000, 30, 2000], hq=8, hk=2),
    "tiles": dict(new=[60, 90], keys=[60, 4000], hq=8, hk=2),
    "list": dict(new=[1500, 1400], keys=[1500, 3000], hq=16, hk=16, page=64),
    "prefix": dict(new=[1] * 9, keys=[70 + 100 * i for i in range(9)], hq=8, hk=2, prefix=5000),
}


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()  # what is freed from here on is what the next request gets


def wait_a_while(stream):
    """About 20 ms of nothing on `stream`."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(40_000_000)


def churn(nbytes):
    """Requests on the current stream that would fit a call's freed blocks, filled."""
    keep = []
    for n in (nbytes, nbytes, nbytes // 2, nbytes // 4):
        keep.append(torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda"))
    return keep


@pytest.mark.parametrize("name", PROBLEMS)
def test_scratch_stays_the_calls(name):
    p = Problem(**PROBLEMS[name], seed=8)
    want = p.run(return_lse=True)
    nbytes = fm.paged_workspace_bytes(len(p.new), max(p.new), p.hq, p.hk, p.tokens if p.packed else 0, p.prefix)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    wait_a_while(side)
    a = p.run(return_lse=True, stream=side.cuda_stream)
    kept = churn(nbytes)
    b = p.run(return_lse=True)  # another call meanwhile, here
    c = p.run(return_lse=True, stream=side.cuda_stream)
    kept += churn(nbytes)
    torch.cuda.synchronize()
    for got in (a, b, c):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all((x == 255).all() for x in kept)
    assert fm.status() == fm.FMHA_OK


def test_results_may_be_dropped_while_this_stream_reads_them():
    p = Problem(**PROBLEMS["rows"], seed=8)
    q = Problem(**PROBLEMS["rows"], seed=9)
    want = p.run()
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    o = p.run(stream=side.cuda_stream)
    here.wait_stream(side)
    wait_a_while(here)
    copy = torch.empty_like(want).copy_(o)
    del o
    for _ in range(3):  # these may not write where the copy still reads
        q.run(stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(copy, want)


def test_rope_and_append():
    table = fm.rope_table(64)
    q, k = normal((8, 1, 4, 64), 1), normal((8, 1, 2, 64), 2)
    pos = torch.arange(8, dtype=torch.int32, device="cuda")[:, None].contiguous()
    t, n = pos.clone(), torch.ones(8, dtype=torch.int32, device="cuda")
    kc, vc = (torch.zeros(8, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want = fm.rope(q, k, table, pos)
    want_q = fm.paged_append(k, k, kc, vc, t, n, q=q, cos_sin=table)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    wait_a_while(side)
    a = fm.rope(q, k, table, pos, stream=side.cuda_stream)
    b = fm.paged_append(k, k, kc, vc, t, n, q=q, cos_sin=table, stream=side.cuda_stream)
    kept = churn(q.nbytes) + churn(k.nbytes)
    torch.cuda.synchronize()
    assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1]) and torch.equal(b, want_q)
    assert all((x == 255).all() for x in kept)


def test_the_named_stream_is_the_one_used():
    """The call comes after what the named stream was given to do first."""
    p = Problem(**PROBLEMS["rows"], seed=8)
    want, q = p.run(), p.q.clone()
    p.q.zero_()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    wait_a_while(side)
    with torch.cuda.stream(side):
        p.q.copy_(q)
    o = p.run(stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(o, want)
    current = torch.cuda.current_stream()
    with pytest.raises(fm.FmhaError):
        p.run(scale=-1.0, stream=side.cuda_stream)
    assert torch.cuda.current_stream() == current  # also after a refusal
    for handle in (0, 1):  # the default stream's names
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            o = p.run(stream=handle)
        torch.cuda.synchronize()
        assert torch.equal(o, p.run())
