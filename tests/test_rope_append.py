"""Rotary positions and appending to the paged cache, against 64 bits."""
import math

import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import UNUSED_PAGE, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


def turn(x, table, axis_of, pos, interleaved, sign=1.0):
    """x [tokens, heads, 64] in 64 bits, pair by pair; pos [axes, tokens]."""
    x = x.double()
    y = x.clone()
    n = len(axis_of)
    for j, axis in enumerate(axis_of):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
        row = table[pos[axis].long()].double()
        c, s = row[:, j, None], sign * row[:, j + n, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def close(got, want):
    """One rounding to bf16 (8 significant bits: at most 2^-8 of the value) of a
    fp32 result (2^-21 of its two terms, below 8 each)."""
    got, want = got.double().reshape(want.shape), want
    return bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all())


SECTIONS = [(32,), (8, 12, 12), (16, 16), (1, 2, 3, 26), (8,), (4, 4), (16,), (5, 11), (24,), (8, 8, 8)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", SECTIONS, ids=str)
def test_rope(sections, interleaved):
    n = sum(sections)
    table = fm.rope_table(1000, 2 * n)
    axis_of = [a for a, m in enumerate(sections) for _ in range(m)]
    for tokens, hq, hk in ((1, 1, 1), (7, 3, 1), (130, 8, 2), (333, 5, 5)):
        q, k = normal((tokens, hq, 64), 1), normal((tokens, hk, 64), 2)
        pos = torch.randint(0, 1000, (len(sections), tokens), device="cuda", dtype=torch.int32)
        qr, kr = fm.rope(q, k, table, pos, sections=sections, interleaved=interleaved)
        assert close(qr, turn(q, table, axis_of, pos, interleaved))
        assert close(kr, turn(k, table, axis_of, pos, interleaved))
        # the gradient: the transpose of the same map
        dq, dk = fm.rope_bwd(q, k, table, pos, sections=sections, interleaved=interleaved)
        assert close(dq, turn(q, table, axis_of, pos, interleaved, -1.0))
        assert close(dk, turn(k, table, axis_of, pos, interleaved, -1.0))
    assert fm.status() == fm.FMHA_OK


def test_gradient_against_differences():
    """<dy, rope(x + h e) - rope(x - h e)> / 2h along random directions e.  The
    map is linear, so h may be 1; the inputs' and outputs' roundings to bf16 are
    at most 2^-8 of values of the size of x and do not add up in one direction:
    their sum over the 8192 products stays below 2^-8 * sqrt(8192) * 4 = 1.4 of a
    result of about 4000.  2 % holds ten times that."""
    table = fm.rope_table(500)
    t, h = 64, 2
    pos = torch.randint(0, 500, (3, t), device="cuda", dtype=torch.int32)
    kw = dict(sections=(8, 12, 12))
    x, dy = normal((t, h, 64), 3), normal((t, h, 64), 4)
    dx, none = fm.rope_bwd(dy, None, table, pos, **kw)
    assert none is None
    for seed in range(3):
        # a direction that the gradient is not orthogonal to
        e = (dx.float() * (torch.rand(dx.shape, device="cuda") > 0.5)).to(torch.bfloat16)
        up = fm.rope((x.float() + e.float()).to(torch.bfloat16), None, table, pos, **kw)[0].double()
        down = fm.rope((x.float() - e.float()).to(torch.bfloat16), None, table, pos, **kw)[0].double()
        want = (dy.double() * (up - down)).sum() / 2
        got = (dx.double() * e.double()).sum()
        assert abs(got - want) <= 0.02 * abs(want)


def test_axis_of_interleaves_axes():
    table = fm.rope_table(300)
    pos = torch.randint(0, 300, (3, 50), device="cuda", dtype=torch.int32)
    axis_of = [j % 3 for j in range(32)]
    q = normal((50, 4, 64), 5)
    assert close(fm.rope(q, None, table, pos, axis_of=axis_of)[0], turn(q, table, axis_of, pos, False))


def test_rope_layouts_strides_in_place():
    table = fm.rope_table(300)
    b, s, hq, hk = 3, 11, 6, 2
    fused = normal((b, s, hq + 2 * hk, 64), 6)
    q, k = fused[:, :, :hq], fused[:, :, hq:hq + hk]
    pos = torch.randint(0, 300, (2, b, s), device="cuda", dtype=torch.int32)
    kw = dict(sections=(20, 12))
    qr, kr = fm.rope(q.contiguous(), k.contiguous(), table, pos, **kw)
    axis_of = [0] * 20 + [1] * 12
    assert close(qr, turn(q.reshape(-1, hq, 64), table, axis_of, pos.flatten(1), False).view(b, s, hq, 64))
    flat = pos.flatten(1)
    a = fm.rope(q.reshape(-1, hq, 64), k.reshape(-1, hk, 64), table, flat, **kw)
    assert torch.equal(a[0].view_as(qr), qr) and torch.equal(a[1].view_as(kr), kr)
    a = fm.rope(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), table, pos, layout="bhsd", **kw)
    assert torch.equal(a[0].transpose(1, 2), qr) and torch.equal(a[1].transpose(1, 2), kr)
    a = fm.rope(q.reshape(-1, hq, 64).transpose(0, 1).contiguous(), None, table, flat, layout="htd", **kw)
    assert torch.equal(a[0].transpose(0, 1).reshape_as(qr), qr) and a[1] is None
    v = fused[:, :, hq + hk:].clone()
    fm.rope(q, k, table, pos, out=(q, k), **kw)  # in place, inside the fused projection
    assert torch.equal(q, qr) and torch.equal(k, kr) and torch.equal(fused[:, :, hq + hk:], v)
    one = normal((b, s, 1, 64), 7)
    assert torch.equal(fm.rope(one.expand(-1, -1, 4, -1), None, table, pos, out=(torch.empty(b, s, 4, 64, device="cuda", dtype=torch.bfloat16), None), **kw)[0],
                       fm.rope(one, None, table, pos, **kw)[0].expand(-1, -1, 4, -1))


def test_rope_table():
    t = fm.rope_table(70000, 32, theta=500000.0)
    p = torch.arange(70000, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert torch.equal(t.cpu(), torch.cat([p.cos(), p.sin()], 1).float())


def test_rope_position_outside_the_table():
    table = fm.rope_table(100)
    q = normal((5, 3, 64), 8)
    pos = torch.tensor([0, 99, 100, -1, 50], device="cuda", dtype=torch.int32)
    r = fm.rope(q, None, table, pos)[0]
    assert fm.status() == fm.FMHA_ERR_INDEX and fm.status() == fm.FMHA_OK
    assert not r[2:4].any()
    ok = torch.tensor([0, 1, 4], device="cuda")
    assert close(r[ok], turn(q[ok], table, [0] * 32, pos[ok][None], False))


# ------------------------------------------------------------ append

def check_append(new, keys, hq, hk, page, rot=64, sections=None, interleaved=False, packed=False, heads_first=False,
                 with_q=True, with_table=True, given=False, slack=0):
    b, tokens = len(new), sum(new)
    need = [-(-max(n, 0) // page) for n in keys]
    pages = sum(need) + 2
    order = torch.randperm(pages).to(torch.int32)
    table = torch.full((b, max(need + [1]) + slack), UNUSED_PAGE, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (pages, hk, page, 64) if heads_first else (pages, page, hk, 64)
    kc, vc = normal(shape, 11), normal(shape, 12)
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    lead = (tokens,) if packed else (b, new[0])
    q, k, v = normal((*lead, hq, 64), 13), normal((*lead, hk, 64), 14), normal((*lead, hk, 64), 15)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda") if packed else None
    place = torch.cat([torch.arange(l - n, l) for n, l in zip(new, keys)]).cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
    sections = sections or (rot // 2,)
    axis_of = [a for a, m in enumerate(sections) for _ in range(m)]
    angles = fm.rope_table(max(max(keys), 1), rot) if with_table else None
    pos = place.clamp_min(0).to(torch.int32).expand(len(sections), -1)
    given_pos = None
    if given:
        pos = torch.randint(0, max(keys), (len(sections), tokens), device="cuda", dtype=torch.int32)
        given_pos = pos.view(len(sections), *lead)
    want_k, want_v = kc.double(), vc.double()
    kr, qr = k.reshape(-1, hk, 64).double(), q.reshape(-1, hq, 64).double()
    if with_table:
        kr, qr = turn(kr, angles, axis_of, pos, interleaved), turn(qr, angles, axis_of, pos, interleaved)
    stored = place >= 0
    pg = table.cuda()[seq[stored], place[stored] // page].long()
    want_k[pg, place[stored] % page] = kr[stored]
    want_v[pg, place[stored] % page] = v.reshape(-1, hk, 64).double()[stored]
    got = fm.paged_append(k, v, kc, vc, table.cuda(), torch.tensor(keys, dtype=torch.int32, device="cuda"),
                          q=q if with_q else None, cos_sin=angles, positions=given_pos,
                          sections=sections if with_table else None, interleaved=interleaved, cu_seqlens_q=cu)
    assert fm.status() == fm.FMHA_OK
    assert close(kc, want_k) and torch.equal(vc.double(), want_v)
    if with_q:
        assert close(got, torch.where(stored[:, None, None], qr, 0.0).view(q.shape))
    else:
        assert got is None


@pytest.mark.parametrize("page", [8, 16, 128, 4096])
@pytest.mark.parametrize("heads", [(4, 4), (7, 1), (12, 3)], ids=str)
def test_append_steps(page, heads):
    check_append([1] * 7, [1, 8, 9, 16, 17, 129, 300], *heads, page)
    check_append([1] * 4, [0, 5, 0, 33], *heads, page)          # empty slots
    check_append([4] * 3, [2, 4, 130], *heads, page)            # more new tokens than places


@pytest.mark.parametrize("sections,rot,interleaved", [((32,), 64, True), ((8, 12, 12), 64, False), ((8, 8), 32, False), ((3, 5), 16, True)])
def test_append_prompts(sections, rot, interleaved):
    check_append([130, 0, 1, 77, 64], [130, 20, 50, 80, 64], 8, 2, 16, rot, sections, interleaved, packed=True, given=True)
    check_append([130, 0, 1, 77, 64], [130, 20, 50, 80, 64], 8, 2, 16, rot, (rot // 2,), interleaved, packed=True)


def test_append_forms():
    check_append([3, 3], [40, 70], 4, 2, 16, heads_first=True)
    check_append([3, 3], [40, 70], 4, 2, 16, with_q=False)
    check_append([3, 3], [40, 70], 4, 2, 16, with_table=False)
    check_append([1] * 600, [1 + i % 40 for i in range(600)], 4, 2, 8, packed=True)


def test_append_index_errors():
    def run(keys, table, max_pos=100, cu=None):
        t = torch.tensor(table, dtype=torch.int32, device="cuda")
        kc, vc = torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
        k = normal((2, 1, 2, 64), 3)
        if cu is not None:
            k, cu = k.flatten(0, 1), torch.tensor(cu, dtype=torch.int32, device="cuda")
        fm.paged_append(k, k, kc, vc, t, torch.tensor(keys, dtype=torch.int32, device="cuda"), cos_sin=fm.rope_table(max_pos), cu_seqlens_q=cu)
        return fm.status(), int(kc.flatten(2).any(-1).sum())

    assert run([1, 20], [[0, 1], [2, 1]]) == (fm.FMHA_OK, 2)
    assert run([1, 20], [[0, 1], [2, 3]]) == (fm.FMHA_ERR_INDEX, 1)     # no such page
    assert run([1, 20], [[0, 1], [2, -1]]) == (fm.FMHA_ERR_INDEX, 1)
    assert run([1, 33], [[0, 1], [2, 1]]) == (fm.FMHA_ERR_INDEX, 1)     # past the table
    assert run([1, 20], [[0, 1], [2, 1]], max_pos=19) == (fm.FMHA_ERR_INDEX, 1)
    assert run([1, 20], [[0, 1], [2, 1]], cu=[0, 1, 1]) == (fm.FMHA_ERR_INDEX, 1)
    assert run([0, -4], [[0, 1], [2, 1]]) == (fm.FMHA_OK, 0)


def test_refusals():
    q, k, table = normal((4, 4, 64), 1), normal((4, 2, 64), 2), fm.rope_table(50)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [
        lambda: fm.rope(q.float(), k, table, pos),
        lambda: fm.rope(q, k[:3], table, pos),
        lambda: fm.rope(q, k, table.double(), pos),
        lambda: fm.rope(q, k, table[:, :20].contiguous(), pos),             # 10 pairs
        lambda: fm.rope(q, k, table, pos.long()),
        lambda: fm.rope(q, k, table, pos[:3]),
        lambda: fm.rope(q, k, table, pos, sections=(16, 16)),               # one row of positions, two axes
        lambda: fm.rope(q, k, table, pos[None].expand(2, -1).contiguous(), sections=(16, 15)),
        lambda: fm.rope(q, k, table, pos[None].expand(5, -1).contiguous(), axis_of=[4] * 32),
        lambda: fm.rope(q, k, table, pos, out=(q[:3], k)),
        lambda: fm.rope(q, k, table, pos, layout="bshd"),
        lambda: fm.rope_table(0),
        lambda: fm.rope_table(5, 30),
    ]
    kc = torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    t, n = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    kd, qd = k[:, None], q[:, None]
    bad += [
        lambda: fm.paged_append(kd, kd[:3], kc, kc, t, n),
        lambda: fm.paged_append(kd[:, :, :1], kd[:, :, :1], kc, kc, t, n),
        lambda: fm.paged_append(kd, kd, kc, kc[:, :8], t, n),
        lambda: fm.paged_append(kd, kd, kc[:, :10], kc[:, :10], t, n),
        lambda: fm.paged_append(kd, kd, kc, kc, t[:2], n),
        lambda: fm.paged_append(kd, kd, kc, kc, t, n, q=qd[:3]),
        lambda: fm.paged_append(kd, kd, kc, kc, t, n, positions=pos),
        lambda: fm.paged_append(k, k, kc, kc, t, n),
        lambda: fm.paged_append(kd, kd, kc, kc, t, n, cu_seqlens_q=n),
    ]
    for f in bad:
        with pytest.raises(fm.FmhaError):
            f()
    assert fm.status() == fm.FMHA_OK


def test_no_tokens():
    table = fm.rope_table(50)
    q = normal((0, 4, 64), 1)
    assert fm.rope(q, None, table, torch.zeros(0, dtype=torch.int32, device="cuda"))[0].shape == q.shape


def test_other_stream_and_graph():
    table = fm.rope_table(64)
    q, k = normal((8, 1, 4, 64), 1), normal((8, 1, 2, 64), 2)
    kc, vc = torch.zeros(8, 16, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(8, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.arange(8, dtype=torch.int32, device="cuda")[:, None].contiguous()
    n = torch.ones(8, dtype=torch.int32, device="cuda")
    want = fm.paged_append(k, k, kc, vc, t, n, q=q, cos_sin=table)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fm.paged_append(k, k, kc, vc, t, n, q=q, cos_sin=table, q_out=out)
    for step in range(1, 17):  # the graph follows the lengths
        n.fill_(step)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(vc, k.expand(-1, 16, -1, -1))
    assert close(out, turn(q.view(8, 4, 64), table, [0] * 32, (n - 1)[None], False).view(q.shape))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n.fill_(1)
        got = fm.paged_append(k, k, kc, vc, t, n, q=q, cos_sin=table)
    side.synchronize()
    assert torch.equal(got, want)
