"""rope under autograd: its gradient, and what it writes in place."""
import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


def inputs(shape=(33,), hq=6, hk=2, axes=3):
    q, k = normal((*shape, hq, 64), 1), normal((*shape, hk, 64), 2)
    pos = torch.randint(0, 200, (axes, *shape), device="cuda", dtype=torch.int32)
    return q, k, fm.rope_table(200), pos


@pytest.mark.parametrize("kw", [dict(sections=(8, 12, 12)), dict(sections=(8, 12, 12), interleaved=True),
                                dict(axis_of=[j % 3 for j in range(32)], inverse=True)], ids=str)
def test_gradients_are_rope_bwd(kw):
    q, k, table, pos = inputs()
    dq, dk = normal(q.shape, 3), normal(k.shape, 4)
    plain = fm.rope(q, k, table, pos, **kw)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    a, b = fm.rope(x, y, table, pos, **kw)
    assert torch.equal(a, plain[0]) and torch.equal(b, plain[1])
    torch.autograd.backward([a, b], [dq, dk])
    turned = dict(kw, inverse=not kw.get("inverse", False))
    want = fm.rope(dq, dk, table, pos, **turned)
    assert torch.equal(x.grad, want[0]) and torch.equal(y.grad, want[1])
    if not kw.get("inverse"):
        bwd = fm.rope_bwd(dq, dk, table, pos, **kw)
        assert torch.equal(x.grad, bwd[0]) and torch.equal(y.grad, bwd[1])


def test_one_of_both_requires_grad():
    q, k, table, pos = inputs()
    kw = dict(sections=(8, 12, 12))
    y = k.clone().requires_grad_()
    a, b = fm.rope(q, y, table, pos, **kw)
    assert not a.requires_grad
    b.sum().backward()  # a gradient that is one value, expanded over all dimensions
    assert torch.equal(y.grad, fm.rope_bwd(torch.ones_like(k), None, table, pos, **kw)[0])
    x = q.clone().requires_grad_()
    a, b = fm.rope(x, None, table, pos, **kw)
    assert b is None
    a[:5].float().square().sum().backward()
    assert x.grad[:5].any() and not x.grad[5:].any()
    x.grad = None
    a, b = fm.rope(x, y, table, pos, **kw)  # only q's result is used
    a.sum().backward()
    assert x.grad is not None


def test_projection_before_it_gets_its_gradient():
    q, k, table, pos = inputs((2, 9))
    w = normal((64, 64), 5).requires_grad_()
    r, _ = fm.rope(q @ w, None, table, pos, sections=(8, 12, 12))
    dy = normal(r.shape, 6)
    r.backward(dy)
    back = fm.rope_bwd(dy, None, table, pos, sections=(8, 12, 12))[0]
    want = q.reshape(-1, 64).double().t() @ back.reshape(-1, 64).double()
    # fp32 sums of 108 products, and one rounding to bf16
    size = q.reshape(-1, 64).double().abs().t() @ back.reshape(-1, 64).double().abs()
    assert ((w.grad.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * size).all()


def test_layouts_and_strides():
    q, k, table, pos = inputs((2, 9))
    kw = dict(sections=(8, 12, 12))
    dy = normal(q.shape, 6)
    want = fm.rope_bwd(dy, None, table, pos, **kw)[0]
    x = q.transpose(1, 2).contiguous().requires_grad_()
    fm.rope(x, None, table, pos, layout="bhsd", **kw)[0].backward(dy.transpose(1, 2))
    assert torch.equal(x.grad, want.transpose(1, 2))
    f = torch.cat([q, k, k], 2).requires_grad_()
    a, b = fm.rope(f[:, :, :6], f[:, :, 6:8], table, pos, **kw)
    torch.autograd.backward([a, b], [dy, torch.zeros_like(k)])
    assert torch.equal(f.grad[:, :, :6], want) and not f.grad[:, :, 6:].any()


def test_another_stream():
    q, k, table, pos = inputs()
    kw = dict(sections=(8, 12, 12))
    dy = normal(q.shape, 6)
    want = fm.rope_bwd(dy, None, table, pos, **kw)[0]
    side = torch.cuda.Stream()
    x = q.clone().requires_grad_()
    side.wait_stream(torch.cuda.current_stream())
    r = fm.rope(x, None, table, pos, stream=side.cuda_stream, **kw)[0]
    torch.cuda.current_stream().wait_stream(side)
    r.backward(dy)
    torch.cuda.synchronize()
    assert torch.equal(x.grad, want)


def test_no_graph_where_none_is_wanted():
    q, k, table, pos = inputs()
    kw = dict(sections=(8, 12, 12))
    assert fm.rope(q, k, table, pos, **kw)[0].grad_fn is None
    with torch.no_grad():
        assert fm.rope(q.clone().requires_grad_(), k, table, pos, **kw)[0].grad_fn is None


def test_out_has_no_gradient():
    q, k, table, pos = inputs()
    kw = dict(sections=(8, 12, 12))
    x = q.clone().requires_grad_()
    with pytest.raises(fm.FmhaError):
        fm.rope(x, k, table, pos, out=(torch.empty_like(q), torch.empty_like(k)), **kw)
    with torch.no_grad():
        fm.rope(x, k, table, pos, out=(x, k), **kw)
