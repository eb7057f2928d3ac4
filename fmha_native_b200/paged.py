"""Serving operators around the attention forward: rotary positions, the paged
K/V cache and attention over it (C ABI: ``include/fmha_paged.h``).

* :func:`rope_table`, :func:`rope`, :func:`rope_bwd` -- rotation of Q and K by
  positions with up to four axes, and its gradient.
* :func:`paged_append` -- new K and V, K rotated on the way, into a cache's
  pages; the rotated Q beside them.
* :func:`paged_fwd` -- attention of one or many new tokens per sequence over
  the pages.
* :func:`prefix_fwd` -- the same for a batch under one shared prefix, whose
  keys are read once for all sequences.

A cache is two bf16 tensors ``[num_pages, page_size, heads_k, 64]`` (any
strides that are multiples of 8; a heads-before-tokens cache is passed as
``cache.transpose(1, 2)``), an int32 ``page_table [batch, max_pages]`` and int32
``seqlens_k [batch]``: the sequences' lengths WITH the new tokens, so new token
i of n has place ``seqlens_k[b] - n + i``.  Tokens are dense (``[batch,
seqlen_q, heads, 64]``) or packed (``[total, heads, 64]`` with int32
``cu_seqlens_q``).  Calls run on the current stream, allocate only through
torch, read nothing back, and may be captured in CUDA graphs after a first
call on the device.  Index data that only the device can check is reported by
``fmha_native_b200.status()`` as ``FMHA_ERR_INDEX``.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional, Sequence

import torch

import fmha_native_b200 as _fm

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32
_LOG2E_8 = _fm.LOG2E / math.sqrt(_fm.HEAD_DIM)


class FmhaRopeParams(ctypes.Structure):
    """Argument block of the rope and append entries (include/fmha_paged.h)."""

    _fields_ = [
        *((n, _P) for n in ("q", "k", "v", "q_out", "k_out", "v_out", "cos_sin", "positions", "seqstart_q",
                            "page_table", "seqlens_k")),
        *((f"{s}_{t}", _L) for t in ("q", "k", "v", "qo", "ko", "vo")
          for s in ("stride", "nhead_stride", "batch_stride")),
        ("axis_stride", _L), ("table_stride", _L),
        *((n, _I) for n in ("batch", "seqlen_q", "total_q", "nhead_q", "nhead_k", "max_pos", "n_pairs",
                            "interleaved", "inverse", "page_size", "num_pages", "max_pages")),
        ("axis_of", ctypes.c_uint8 * 32),
    ]


class FmhaPagedParams(ctypes.Structure):
    """Argument block of the paged and prefix attention entries."""

    _fields_ = [
        *((n, _P) for n in ("q", "k_cache", "v_cache", "o", "lse", "seqstart_q", "page_table", "seqlens_k",
                            "prefix_pages", "workspace")),
        ("workspace_bytes", _L),
        *((f"{s}_{t}", _L) for t in ("q", "o") for s in ("stride", "nhead_stride", "batch_stride")),
        *((f"{s}_{t}", _L) for t in ("k", "v") for s in ("stride", "nhead_stride", "page_stride")),
        ("table_stride", _L),
        *((n, _I) for n in ("batch", "seqlen_q", "total_q", "nhead_q", "nhead_k", "page_size", "num_pages",
                            "max_pages", "prefix_len", "causal")),
        ("scale", _F),
    ]


# The blocks are packed in one go: field by field, ctypes costs several
# microseconds a call.  Sizes and offsets are those of the structures above.
_pack_rope = struct.Struct("@11P20q12i32s").pack
_pack_paged = struct.Struct("@10P14q10if4x").pack


def _bad(what: str):
    return _fm.FmhaError(_fm.FMHA_ERR_ARG, what)


def _call(fn: str, params: bytes, device: int, stream) -> None:
    lib = _fm.load_library()
    if torch.cuda.current_device() != device:
        with torch.cuda.device(device):
            return _call(fn, params, device, stream)
    if stream is None:
        stream = torch.cuda.current_stream(device).cuda_stream
    st = getattr(lib, fn)(params, stream)
    if st:
        raise _fm.FmhaError(st, fn)


def _heads(x, what: str, axes):
    """(device, strides of token, head and batch) of a bf16 head tensor."""
    if x.dtype is not _BF16 or not x.is_cuda or x.shape[-1] != 64:
        raise _bad(f"{what} must be a CUDA bf16 tensor with head_dim 64")
    st = x.stride()
    if st[-1] != 1:
        raise _bad(f"{what}: the head dimension must be contiguous")
    return st[axes[0]], st[axes[1]], (st[0] if axes[2] else 0)


def _axes(ndim: int, layout: Optional[str]):
    """(token axis, head axis, has batch) of a 3- or 4-dimensional head tensor."""
    if layout is None:
        layout = "thd" if ndim == 3 else "bshd"
    try:
        a = _LAYOUTS[layout]
    except KeyError:
        raise _bad(f"unknown layout {layout!r}") from None
    if ndim != (4 if a[2] else 3):
        raise _bad(f"layout {layout!r} does not fit a tensor of {ndim} dimensions")
    return a


_LAYOUTS = {"thd": (0, 1, False), "htd": (1, 0, False), "bshd": (1, 2, True), "bhsd": (2, 1, True)}


def _ints(x, what: str, device: int):
    if x.dtype is not _I32 or x.get_device() != device or x.stride(-1) != 1 and x.shape[-1] > 1:
        raise _bad(f"{what} must be an int32 tensor on q's device, its last dimension contiguous")
    return x.data_ptr()


@functools.lru_cache(maxsize=256)
def _axis_map(sections: Optional[tuple], axis_of: Optional[tuple], n_pairs: int):
    """(axis of each pair as 32 bytes, axes named)."""
    if n_pairs not in (8, 16, 24, 32):
        raise _bad("cos_sin must be [max_pos, rot_dim] with rot_dim 16, 32, 48 or 64")
    if axis_of is None:
        axis_of = tuple(a for a, n in enumerate(sections or (n_pairs,)) for _ in range(n))
    if len(axis_of) != n_pairs or min(axis_of) < 0 or max(axis_of) > 3:
        raise _bad(f"sections / axis_of must assign the {n_pairs} pairs to at most 4 axes")
    return bytes(axis_of) + bytes(32 - n_pairs), max(axis_of) + 1


def _table(cos_sin, sections, axis_of, device: int):
    """(pointer, max_pos, n_pairs, axis bytes, axes) of an angle table."""
    if (cos_sin.dtype is not _F32 or cos_sin.get_device() != device or cos_sin.dim() != 2
            or not cos_sin.is_contiguous()):
        raise _bad("cos_sin must be a contiguous fp32 [max_pos, rot_dim] tensor on q's device")
    max_pos, rot = cos_sin.shape
    axes, n = _axis_map(None if sections is None else tuple(sections),
                        None if axis_of is None else tuple(axis_of), rot // 2)
    return cos_sin.data_ptr(), max_pos, rot // 2, axes, n


def _positions(positions, lead: tuple, axes: int, device: int):
    """(pointer, stride between axes) of positions [lead] or [axes, lead]."""
    ptr = _ints(positions, "positions", device)
    shape = tuple(positions.shape)
    if shape == lead:
        have, stride, rows = 1, 0, positions
    elif shape[1:] == lead:
        have, stride, rows = shape[0], positions.stride(0), positions[0] if shape[0] else positions
    else:
        raise _bad(f"positions must be {list(lead)} or [axes, {', '.join(map(str, lead))}]")
    if have < axes or not rows.is_contiguous():
        raise _bad("positions needs a row for every axis, contiguous over the tokens")
    return ptr, stride


def rope_table(max_pos: int, rot_dim: int = 64, theta: float = 10000.0, inv_freq: Optional[Sequence[float]] = None,
               device=None):
    """fp32 ``[max_pos, rot_dim]``: row p holds the cosines, then the sines, of
    ``p * inv_freq`` (default ``theta ** (-2 j / rot_dim)``), computed in 64 bits."""
    n = rot_dim // 2
    f = (theta ** (-torch.arange(n, dtype=torch.float64) / n) if inv_freq is None
         else torch.as_tensor(inv_freq, dtype=torch.float64))
    if f.numel() != n or rot_dim not in (16, 32, 48, 64) or max_pos < 1:
        raise _bad("rope_table: rot_dim must be 16, 32, 48 or 64, with rot_dim / 2 frequencies, and max_pos positive")
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * f.cpu()
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device if device is not None else "cuda")


def rope(q, k, cos_sin, positions, *, sections=None, axis_of=None, interleaved: bool = False, inverse: bool = False,
         layout: Optional[str] = None, out=None, stream=None):
    """Q and K (or None) with their pairs rotated by the tokens' positions.

    ``positions``: int32 over q's token dimensions (``[total]`` or ``[batch,
    seqlen]``), or ``[axes, ...]`` for positions with several axes (time,
    height, width).  ``sections`` gives how many consecutive pairs each axis
    turns; ``axis_of`` names the axis of every pair instead.  ``interleaved``:
    pairs (2j, 2j+1) instead of (j, j + rot_dim/2).  Dimensions from rot_dim on
    pass through.  ``out``: the tensors to write, which may be q and k
    themselves.  Layouts: "thd", "htd", "bshd", "bhsd".
    """
    ax = _axes(q.dim(), layout)
    dev = q.get_device()
    sq = _heads(q, "q", ax)
    qo, ko = out if out is not None else (torch.empty_like(q), None if k is None else torch.empty_like(k))
    if qo.shape != q.shape or qo.get_device() != dev:
        raise _bad("out must have q's and k's shapes and device")
    sqo = _heads(qo, "out", ax)
    shape = q.shape
    lead = (shape[0], shape[ax[0]]) if ax[2] else (shape[ax[0]],)
    kp = kop = None
    sk = sko = (0, 0, 0)
    hk = 0
    if k is not None:
        sk, sko = _heads(k, "k", ax), _heads(ko, "out", ax)
        if (k.dim() != q.dim() or k.shape != ko.shape or k.get_device() != dev or ko.get_device() != dev
                or k.shape[ax[0]] != lead[-1] or k.shape[0] != shape[0] and ax != _LAYOUTS["htd"]):
            raise _bad("k must have q's tokens and device, and out the shapes of both")
        kp, kop, hk = k.data_ptr(), ko.data_ptr(), k.shape[ax[1]]
    tp, max_pos, n, axis_bytes, axes = _table(cos_sin, sections, axis_of, dev)
    pp, axis_stride = _positions(positions, lead, axes, dev)
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return qo, ko
    batch, seqlen = lead if ax[2] else (1, lead[0])
    _call("fmha_rope_d64_bf16", _pack_rope(
        q.data_ptr(), kp or 0, 0, qo.data_ptr(), kop or 0, 0, tp, pp, 0, 0, 0,
        *sq, *sk, 0, 0, 0, *sqo, *sko, 0, 0, 0, axis_stride, 0,
        batch, seqlen, 0, shape[ax[1]], hk, max_pos, n, bool(interleaved), bool(inverse), 0, 0, 0, axis_bytes),
        dev, stream)
    return qo, ko


def rope_bwd(dq, dk, cos_sin, positions, **kw):
    """Gradients of :func:`rope`'s inputs from its outputs': the rotation back
    (a rotation's transpose), same arguments."""
    return rope(dq, dk, cos_sin, positions, inverse=True, **kw)


def _cache(k_cache, v_cache, device: int):
    """(page size, heads, pages, strides of both) of a cache."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise _bad("k_cache and v_cache must both be [num_pages, page_size, heads_k, 64]")
    sk, sv = _heads(k_cache, "k_cache", _LAYOUTS["bshd"]), _heads(v_cache, "v_cache", _LAYOUTS["bshd"])
    if k_cache.get_device() != device or v_cache.get_device() != device:
        raise _bad("the cache must be on q's device")
    pages, page, heads, _ = k_cache.shape
    return page, heads, pages, sk, sv


def _batch(page_table, seqlens_k, cu_seqlens_q, lead, device: int):
    """(batch, pointers of the table, the lengths and the prefix sums)."""
    tp, lp = _ints(page_table, "page_table", device), _ints(seqlens_k, "seqlens_k", device)
    batch = seqlens_k.shape[0]
    if page_table.dim() != 2 or seqlens_k.dim() != 1 or page_table.shape[0] != batch:
        raise _bad("page_table must be [batch, max_pages] and seqlens_k [batch]")
    cp = 0
    if len(lead) == 2:
        if cu_seqlens_q is not None or lead[0] != batch:
            raise _bad("dense tokens are [batch, seqlen_q, ...] with page_table's batch and no cu_seqlens_q")
    else:
        if cu_seqlens_q is None:
            raise _bad("packed tokens need cu_seqlens_q")
        cp = _ints(cu_seqlens_q, "cu_seqlens_q", device)
        if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] != batch + 1:
            raise _bad("cu_seqlens_q must be [batch + 1]")
    return batch, tp, lp, cp


def paged_append(k, v, k_cache, v_cache, page_table, seqlens_k, *, q=None, cos_sin=None, positions=None, sections=None,
                 axis_of=None, interleaved: bool = False, cu_seqlens_q=None, layout: Optional[str] = None, q_out=None,
                 stream=None):
    """Writes new K and V into their places in the cache; returns the rotated q
    (None without q).

    With ``cos_sin`` (:func:`rope_table`) K and q are rotated as by
    :func:`rope`, by ``positions`` or, without them, by the tokens' places in
    the cache.  A token whose place is negative (an empty slot of the batch) is
    not stored and its q row comes back zero.
    """
    ax = _axes(k.dim(), layout)
    dev = k.get_device()
    sk, sv = _heads(k, "k", ax), _heads(v, "v", ax)
    shape = k.shape
    if v.shape != shape or v.get_device() != dev:
        raise _bad("v must have k's shape and device")
    lead = (shape[0], shape[ax[0]]) if ax[2] else (shape[ax[0]],)
    page, heads, pages, skc, svc = _cache(k_cache, v_cache, dev)
    if shape[ax[1]] != heads:
        raise _bad("k must have the cache's heads")
    batch, tp, lp, cp = _batch(page_table, seqlens_k, cu_seqlens_q, lead, dev)
    qp = qop = hq = 0
    sq = sqo = (0, 0, 0)
    if q is not None:
        sq = _heads(q, "q", ax)
        if q_out is None:
            q_out = torch.empty_like(q)
        sqo = _heads(q_out, "q_out", ax)
        if (q.dim() != len(shape) or q.shape != q_out.shape or q.shape[ax[0]] != lead[-1]
                or ax[2] and q.shape[0] != lead[0] or q.get_device() != dev or q_out.get_device() != dev):
            raise _bad("q (and q_out) must have k's tokens and device")
        qp, qop, hq = q.data_ptr(), q_out.data_ptr(), q.shape[ax[1]]
    tab = max_pos = pp = axis_stride = 0
    n, axis_bytes = 32, bytes(32)
    if cos_sin is not None:
        tab, max_pos, n, axis_bytes, axes = _table(cos_sin, sections, axis_of, dev)
        if positions is not None:
            pp, axis_stride = _positions(positions, lead, axes, dev)
    elif positions is not None:
        raise _bad("positions need cos_sin")
    if k.numel() == 0:
        return q_out
    _call("fmha_paged_append_d64_bf16", _pack_rope(
        qp, k.data_ptr(), v.data_ptr(), qop, k_cache.data_ptr(), v_cache.data_ptr(), tab, pp, cp, tp, lp,
        *sq, *sk, *sv, *sqo, *skc, *svc, axis_stride, page_table.stride(0),
        batch, lead[-1], 0 if ax[2] else lead[0], hq, heads, max_pos, n, bool(interleaved), 0, page, pages,
        page_table.shape[1], axis_bytes), dev, stream)
    return q_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes) -> int:
    return int(_fm.load_library().fmha_paged_workspace_bytes(*sizes))


def paged_workspace_bytes(batch: int, seqlen_q: int, heads_q: int, heads_k: int, total_q: int = 0,
                          prefix_len: int = 0) -> int:
    """Bytes of device scratch that :func:`paged_fwd` (``prefix_len`` 0) or
    :func:`prefix_fwd` needs for these sizes (``total_q`` > 0: packed tokens, of
    which a sequence has at most ``seqlen_q``)."""
    return _workspace_bytes(batch, seqlen_q, total_q, heads_q, heads_k, prefix_len)


def _attend(fn, q, k_cache, v_cache, page_table, seqlens_k, prefix_pages, prefix_len, causal, cu_seqlens_q,
            max_seqlen_q, scale, return_lse, layout, out, lse_out, workspace, stream):
    ax = _axes(q.dim(), layout)
    dev = q.get_device()
    sq = _heads(q, "q", ax)
    shape = q.shape
    dense = ax[2]
    hq = shape[ax[1]]
    lead = (shape[0], shape[ax[0]]) if dense else (shape[ax[0]],)
    page, heads, pages, skc, svc = _cache(k_cache, v_cache, dev)
    batch, tp, lp, cp = _batch(page_table, seqlens_k, cu_seqlens_q, lead, dev)
    if heads == 0 or hq % heads:
        raise _bad("q's heads must be a multiple of the cache's")
    if out is None:
        out = torch.empty_like(q)
        so = sq if out.stride() == q.stride() else _heads(out, "out", ax)
    else:
        if out.shape != shape or out.get_device() != dev:
            raise _bad("out must have q's shape and device")
        so = _heads(out, "out", ax)
    lse = None
    if return_lse:
        want = (batch, hq, lead[1]) if dense else (hq, lead[0])
        if lse_out is None:
            lse = torch.empty(want, device=q.device, dtype=_F32)
        else:
            lse = lse_out
            if tuple(lse.shape) != want or lse.dtype is not _F32 or not lse.is_contiguous() or lse.get_device() != dev:
                raise _bad(f"lse_out must be a contiguous fp32 {list(want)} tensor on q's device")
    if q.numel() == 0:
        return (out, lse) if return_lse else out
    total = 0 if dense else lead[0]
    longest = lead[1] if dense else (total if max_seqlen_q is None else int(max_seqlen_q))
    need = _workspace_bytes(batch, longest, total, hq, heads, prefix_len)
    if workspace is None:
        workspace = torch.empty(need, device=q.device, dtype=torch.uint8)
        have = need
    else:
        have = workspace.numel() * workspace.element_size()
        if workspace.get_device() != dev or not workspace.is_contiguous() or have < need:
            raise _bad(f"workspace must be a contiguous tensor of {need} bytes on q's device")
    _call(fn, _pack_paged(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
        cp, tp, lp, prefix_pages.data_ptr() if prefix_len else 0, workspace.data_ptr(), have, *sq, *so, *skc, *svc,
        page_table.stride(0), batch, longest, total, hq, heads, page, pages, page_table.shape[1], prefix_len,
        bool(causal), _LOG2E_8 if scale is None else scale * _fm.LOG2E), dev, stream)
    return (out, lse) if return_lse else out


def paged_fwd(q, k_cache, v_cache, page_table, seqlens_k, *, causal: bool = True, cu_seqlens_q=None,
              max_seqlen_q: Optional[int] = None, scale: Optional[float] = None, return_lse: bool = False,
              layout: Optional[str] = None, out=None, lse_out=None, workspace=None, stream=None):
    """O = softmax(scale Q K^T) V of the new tokens over each sequence's pages.

    ``causal``: new token i sees the keys up to its own place (bottom-right
    aligned); otherwise all ``seqlens_k[b]`` keys.  ``scale`` (default 1/8) must
    be positive.  ``max_seqlen_q`` (packed): the most new tokens of any
    sequence, if known; a bound, by which the kernels are chosen.  Returns O
    (and the fp32 LSE, ``[batch, heads, seqlen_q]`` or ``[heads, total]``).
    Rows that see no key: O = 0, LSE = -inf.
    """
    return _attend("fmha_paged_fwd_d64_bf16", q, k_cache, v_cache, page_table, seqlens_k, None, 0, causal, cu_seqlens_q,
                   max_seqlen_q, scale, return_lse, layout, out, lse_out, workspace, stream)


def prefix_fwd(q, k_cache, v_cache, prefix_pages, prefix_len: int, page_table, seqlens_k, *, causal: bool = True,
               cu_seqlens_q=None, max_seqlen_q: Optional[int] = None, scale: Optional[float] = None,
               return_lse: bool = False, layout: Optional[str] = None, out=None, lse_out=None, workspace=None,
               stream=None):
    """:func:`paged_fwd` where every sequence's keys are the ``prefix_len`` keys
    in ``prefix_pages`` (int32 ``[pages]``) followed by its own ``seqlens_k[b]``
    ones in ``page_table``: the prefix is read once for the whole batch.
    ``causal`` concerns the sequences' own keys; all tokens see the prefix."""
    prefix_len = int(prefix_len)
    _ints(prefix_pages, "prefix_pages", q.get_device())
    if prefix_len < 1 or prefix_pages.dim() != 1 or prefix_pages.shape[0] * k_cache.shape[1] < prefix_len:
        raise _bad("prefix_pages must be [pages] with room for prefix_len >= 1 keys")
    return _attend("fmha_prefix_fwd_d64_bf16", q, k_cache, v_cache, page_table, seqlens_k, prefix_pages, prefix_len,
                   causal, cu_seqlens_q, max_seqlen_q, scale, return_lse, layout, out, lse_out, workspace, stream)
