"""Attention over the paged cache and under a shared prefix, against 64 bits."""
import math

import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import Problem, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


# Lengths of nothing and of one; ends of units, tiles and pages; empty slots of
# a batch; sequences with more new tokens than keys, whose first rows see none.
LENGTHS = {
    "one": ([1], [1]),
    "short": ([1] * 6, [1, 2, 7, 8, 9, 31]),
    "ends": ([1] * 9, [32, 33, 63, 64, 65, 127, 128, 129, 257]),
    "empty_slots": ([1] * 5, [0, 40, 0, 0, 513]),
    "none": ([1, 1], [0, 0]),
    "drafts": ([4] * 4, [4, 5, 131, 700]),
    "more_new_than_keys": ([5] * 4, [0, 1, 4, 6]),
    "ragged": ([0, 3, 1, 0, 8, 2], [0, 3, 90, 17, 8, 1000]),
    "long_and_short": ([1] * 4, [9001, 3, 130, 2]),
}


@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (3, 1), (12, 1)], ids=str)
@pytest.mark.parametrize("name", LENGTHS)
def test_lengths(name, heads):
    new, keys = LENGTHS[name]
    Problem(new, keys, *heads).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 4096])
def test_page_sizes(page):
    Problem([1] * 5, [page - 1, page, page + 1, 3 * page + 5, 1], 8, 2, page=page).check()
    Problem([3, 70], [page + 40, 2 * page + 75], 8, 2, page=page).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [1, 2, 5, 16, 17, 33, 64, 129])
@pytest.mark.parametrize("heads", [(2, 2), (6, 1), (16, 2)], ids=str)
def test_new_tokens(new, heads, causal):
    """Rows per K/V head from 2 to over a thousand."""
    Problem([new] * 3, [new, new + 61, new + 500], *heads).check(causal=causal)


@pytest.mark.parametrize("group", [1, 2, 5, 7, 8, 16, 24, 33, 130])
def test_groups(group):
    Problem([1, 1, 1], [5, 300, 77], group * 2, 2, page=32).check()


@pytest.mark.parametrize("heads", [(8, 8), (24, 4)], ids=str)
def test_prompts(heads):
    """Long row tiles: whole prompts, chunks behind a context, single tokens among them."""
    Problem([257, 1, 130, 1, 640, 5], [257, 2000, 1030, 3, 640, 900], *heads, page=64).check()


def test_non_causal_packed():
    Problem([40, 0, 1, 7], [200, 50, 33, 6], 8, 2).check(causal=False)


def test_many_sequences():
    """More sequences than threads of a block."""
    n = 700
    keys = [(i * 37) % 90 for i in range(n)]
    Problem([1] * n, keys, 4, 2).check()


def test_long_context_across_all_blocks():
    Problem([1], [60001], 8, 1, page=64).check()
    Problem([1, 1], [30001, 25000], 4, 4, page=128).check()


@pytest.mark.parametrize("scale", [0.125, 0.01, 1.0])
def test_scale(scale):
    Problem([1, 3], [400, 90], 4, 2).check(scale=scale)


def test_large_scores():
    """Scores over a thousand: the running maximum carries them."""
    Problem([1, 40], [600, 300], 4, 2, q_by=400.0).check(lse=False)


@pytest.mark.parametrize("new", [[1, 1], [90, 90]])
def test_strides_and_layouts(new):
    p = Problem(new, [150, 333], 8, 2, heads_first=True)
    want, want_lse = p.check()
    b, n = len(new), new[0]
    fused = normal((b, n, 12, 64), 9)
    q = fused[:, :, :8]
    q.copy_(p.q)
    wide = torch.empty(b, n, 8, 96, device="cuda", dtype=torch.bfloat16)
    o = p.run(q, out=wide[..., :64])
    assert torch.equal(o, want) and o.data_ptr() == wide.data_ptr()
    t = p.q.transpose(1, 2).contiguous()
    assert torch.equal(p.run(t, layout="bhsd").transpose(1, 2), want)
    # packed forms of the same tokens
    cu = torch.arange(b + 1, device="cuda", dtype=torch.int32) * n
    o, lse = p.run(p.q.flatten(0, 1), cu_seqlens_q=cu, return_lse=True)
    assert torch.equal(o.view_as(want), want)
    assert torch.equal(lse.view(8, b, n).transpose(0, 1), want_lse)
    o = p.run(p.q.flatten(0, 1).transpose(0, 1).contiguous(), cu_seqlens_q=cu, layout="htd")
    assert torch.equal(o.transpose(0, 1).reshape_as(want), want)


def test_shared_query_heads():
    """Queries broadcast over the heads (stride 0)."""
    p = Problem([1, 1], [70, 200], 4, 2)
    one = p.q[:, :, :1]
    p.q = one.expand(-1, -1, 4, -1).contiguous()
    want = p.check(lse=False)
    assert torch.equal(p.run(one.expand(-1, -1, 4, -1), out=torch.empty_like(want)), want)


def test_offsets_beyond_32_bits():
    """A cache of over 2^31 values a tensor, the sequence in its last pages."""
    pages, page, hk = 70000, 128, 4
    k = torch.empty(pages, page, hk, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 1 << 31
    for new, keys in (([1], [300]), ([150], [300])):
        p = Problem(new, keys, 8, hk, page=page, spare=0)
        n = p.k_cache.shape[0]
        k[-n:], v[-n:] = p.k_cache, p.v_cache
        p.k_cache, p.v_cache = k, v
        p.table = p.table + (pages - n)
        p.check()


def test_same_bits_every_time():
    for p in (Problem([1] * 7, [5000, 1, 900, 333, 64, 10, 4000], 8, 2),
              Problem([300, 40], [300, 5000], 8, 2, packed=True),
              Problem([1] * 9, [100] * 9, 8, 2, prefix=3001)):
        a = p.run(return_lse=True)
        for _ in range(3):
            b = p.run(return_lse=True)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_other_stream_graph_and_workspace():
    for p in (Problem([1] * 3, [700, 30, 2000], 8, 2), Problem([60, 90], [60, 800], 8, 2),
              Problem([1] * 3, [70, 30, 200], 8, 2, prefix=500)):
        want = p.run()
        nbytes = fm.paged_workspace_bytes(len(p.new), max(p.new), p.hq, p.hk, p.tokens if p.packed else 0, p.prefix)
        ws = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            o = p.run(workspace=ws)
        side.synchronize()
        assert torch.equal(o, want)
        graph = torch.cuda.CUDAGraph()
        o = torch.zeros_like(want)
        with torch.cuda.graph(graph):
            p.run(out=o, workspace=ws)
        for _ in range(2):
            o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)
        # lengths are read on the device: the same graph follows them
        keys = p.keys
        p.seqlens.copy_(torch.tensor([max(1, k - 7) if k > 100 else k for k in keys], dtype=torch.int32))
        graph.replay()
        assert torch.equal(o, p.run())


# ------------------------------------------------------------ shared prefix

@pytest.mark.parametrize("prefix", [1, 15, 128, 129, 1000, 5003])
@pytest.mark.parametrize("batch,heads", [(1, (4, 4)), (5, (8, 2)), (40, (8, 1)), (150, (4, 4))], ids=str)
def test_prefix(prefix, batch, heads):
    keys = [1 + (i * 53) % 200 for i in range(batch)]
    Problem([1] * batch, keys, *heads, prefix=prefix).check()


def test_prefix_with_several_tokens():
    Problem([3] * 6, [3, 4, 50, 0, 2, 300], 8, 2, prefix=777, page=32).check()
    Problem([3, 0, 1, 60, 17], [3, 9, 50, 60, 170], 8, 2, prefix=777, page=64).check()


def test_prefix_empty_slots():
    """A slot without keys of its own sees the prefix alone."""
    Problem([1] * 4, [0, 0, 5, 0], 8, 2, prefix=100).check()


def test_prefix_is_what_paged_gives():
    """The same keys, once as a prefix and once in every sequence's own pages."""
    p = Problem([1] * 8, [10 + 9 * i for i in range(8)], 8, 2, prefix=640, page=16)
    o = p.run()
    own = p.prefix_pages[None].expand(8, -1)
    p.table = torch.cat([own, p.table], 1).contiguous()
    p.seqlens += 640
    q = fm.paged_fwd(p.q, p.k_cache, p.v_cache, p.table, p.seqlens)
    assert (o.double() - q.double()).abs().max() <= 2.0 ** -7 * q.double().abs().max()


@pytest.mark.parametrize("hk", [5, 10, 12, 17, 24, 32])
@pytest.mark.parametrize("new, group", [(1, 1), (1, 4), (2, 4), (5, 3)])
def test_heads_shared_out_to_blocks(hk, new, group):
    Problem([new] * 3, [5000, 37, 777], hk * group, hk, 32).check()


def test_heads_shared_out_under_a_prefix():
    Problem([1] * 5, [1500, 0, 33, 700, 1], 48, 24, 16, prefix=300).check()


def test_sequences_of_both_kernels_mixed():
    """More sequences than threads, most of them many-row ones."""
    new = [1 if i % 7 == 3 else 20 + i % 5 for i in range(300)]
    Problem(new, [n + (11 * i) % 150 for i, n in enumerate(new)], 4, 4, 16, packed=True).check()
    new = [1 if 250 < i < 255 else 0 for i in range(300)]
    Problem(new, [n + (11 * i) % 150 for i, n in enumerate(new)], 4, 4, 16, packed=True).check()


# ------------------------------------------------------------ refusals

def test_index_errors_are_reported():
    def status_after(change, **kw):
        p = Problem([1, 1], [40, 70], 4, 2, **kw)
        change(p)
        p.run()
        return fm.status()

    assert status_after(lambda p: None) == fm.FMHA_OK
    assert status_after(lambda p: p.table[1].fill_(10 ** 6)) == fm.FMHA_ERR_INDEX
    assert status_after(lambda p: p.table[0].fill_(-1)) == fm.FMHA_ERR_INDEX
    assert status_after(lambda p: p.seqlens.fill_(10 ** 6)) == fm.FMHA_ERR_INDEX
    assert status_after(lambda p: p.cu.copy_(torch.tensor([0, 5, 2])), packed=True) == fm.FMHA_ERR_INDEX
    assert status_after(lambda p: p.cu.copy_(torch.tensor([0, 1, 9])), packed=True) == fm.FMHA_ERR_INDEX
    assert status_after(lambda p: p.seqlens.fill_(-3)) == fm.FMHA_OK  # an empty slot
    assert fm.status() == fm.FMHA_OK  # reported once


def test_more_tokens_than_said_is_reported():
    p = Problem([1, 60], [1, 60], 4, 2)
    p.run(max_seqlen_q=1)
    assert fm.status() == fm.FMHA_ERR_INDEX


@pytest.mark.parametrize("new, said, prefix", [(9, 2, 0), (40, 9, 0), (300, 40, 0), (40, 9, 700)])
def test_tokens_within_what_was_said_keep_their_results(new, said, prefix):
    """A sequence of more tokens than said: reported, the first ones as they are."""
    p = Problem([said, new, 1], [900, 1300, 800], 8, 2, packed=True, prefix=prefix)
    o = p.run()
    assert fm.status() == fm.FMHA_OK
    few = p.run(max_seqlen_q=said)
    assert fm.status() == fm.FMHA_ERR_INDEX
    for at in (slice(0, 2 * said), slice(said + new, None)):
        assert (o[at].double() - few[at].double()).abs().max() <= 2.0 ** -7 * o[at].double().abs().max()


def test_refusals():
    p = Problem([1, 1], [40, 70], 4, 2)
    q, kc, vc, t, n = p.q, p.k_cache, p.v_cache, p.table, p.seqlens
    bad = [
        lambda: fm.paged_fwd(q.float(), kc, vc, t, n),
        lambda: fm.paged_fwd(q[..., :32], kc, vc, t, n),
        lambda: fm.paged_fwd(q[:, :, :3], kc, vc, t, n),                       # 3 heads over 2
        lambda: fm.paged_fwd(q, kc, vc[:-1], t, n),
        lambda: fm.paged_fwd(q, kc[:, :12], vc[:, :12], t, n),                 # page of 12
        lambda: fm.paged_fwd(q, kc, vc, t.long(), n),
        lambda: fm.paged_fwd(q, kc, vc, t, n.long()),
        lambda: fm.paged_fwd(q, kc, vc, t[:1], n),
        lambda: fm.paged_fwd(q, kc, vc, t, n.cpu()),
        lambda: fm.paged_fwd(q, kc, vc, t, n, scale=0.0),
        lambda: fm.paged_fwd(q, kc, vc, t, n, scale=-1.0),
        lambda: fm.paged_fwd(q, kc, vc, t, n, out=torch.empty_like(q)[:1]),
        lambda: fm.paged_fwd(q, kc, vc, t, n, workspace=torch.empty(16, device="cuda")),
        lambda: fm.paged_fwd(q, kc, vc, t, n, cu_seqlens_q=n),
        lambda: fm.paged_fwd(q.flatten(0, 1), kc, vc, t, n),                   # packed without prefix sums
        lambda: fm.paged_fwd(q, kc, vc, t, n, layout="sbhd"),
        lambda: fm.paged_fwd(q, kc, vc, t, n, return_lse=True, lse_out=torch.empty(2, 4, 1, device="cuda").half()),
        lambda: fm.prefix_fwd(q, kc, vc, t[0], 0, t, n),
        lambda: fm.prefix_fwd(q, kc, vc, t[0], 10 ** 6, t, n),
    ]
    for f in bad:
        with pytest.raises(fm.FmhaError):
            f()
    odd = torch.empty(2 * 4 * 64 + 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(fm.FmhaError):  # a base that is not 16-byte aligned
        fm.paged_fwd(odd[1:513].view(2, 1, 4, 64), kc, vc, t, n)
    assert fm.status() == fm.FMHA_OK


def test_no_tokens():
    p = Problem([0, 0], [40, 70], 4, 2, packed=True)
    o, lse = p.run(return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
