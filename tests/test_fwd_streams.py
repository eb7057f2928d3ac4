"""fmha_fwd on a named stream: its scratch and results are that stream's."""
import pytest
import torch

import fmha_native_b200 as fm
from fmha_native_b200 import shard

pytestmark = pytest.mark.gpu


def normal(shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def forms(q, k, v):
    b, s, h = q.shape[:3]
    blocks = shard.plan_blocks(b, h, s, s, True)
    tiles = torch.from_numpy(shard.tiles_array(blocks)).cuda()
    items = torch.from_numpy(shard.items_array(shard.plan_items(blocks))).cuda()
    cu = torch.arange(b + 1, dtype=torch.int32, device="cuda") * s
    flat = [x.flatten(0, 1) for x in (q, k, v)]
    return {
        "whole": lambda **kw: fm.fmha_fwd(q, k, v, causal=True, return_lse=True, **kw),
        "splits": lambda **kw: fm.fmha_fwd(q, k, v, causal=True, return_lse=True, tiles=tiles, num_splits=4, **kw),
        "items": lambda **kw: fm.fmha_fwd(q, k, v, causal=True, return_lse=True, items=items, **kw),
        "varlen": lambda **kw: fm.fmha_fwd(*flat, causal=True, return_lse=True, layout="thd", cu_seqlens_q=cu,
                                           cu_seqlens_k=cu, **kw),
    }


@pytest.mark.parametrize("form", ["whole", "splits", "items", "varlen"])
def test_memory_is_the_named_streams(cuda_device, form):
    q, k, v = (normal((1, 1100, 3, 64), i) for i in range(3))
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    f = forms(q, k, v)[form]
    want = f()
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
    got = f(stream=side.cuda_stream)
    assert torch.cuda.current_stream() == here
    kept = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in [1 << 22, 1 << 20] * 4]
    again = f()
    torch.cuda.synchronize()
    for a in (got, again):
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    assert all((x == 255).all() for x in kept)
    o, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    got = f(stream=side.cuda_stream, out=o, lse_out=lse)
    side.synchronize()
    assert got[0] is o and got[1] is lse and torch.equal(o, want[0]) and torch.equal(lse, want[1])
    # the default stream by its handles: after what it was given to do first
    new = normal(q.shape, 9)
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)
    q.copy_(new)
    with torch.cuda.stream(side):
        got = [f(stream=handle) for handle in (0, 1)]
    torch.cuda.synchronize()
    want = f()
    assert all(torch.equal(a[0], want[0]) and torch.equal(a[1], want[1]) for a in got)
    assert fm.status() == fm.FMHA_OK
