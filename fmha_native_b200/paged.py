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
``cu_seqlens_q``).  Calls run on the current stream or on the one that ``stream``
names (its handle, an integer), allocate only through torch and on that stream,
read nothing back, and may be captured in CUDA graphs after a first call on the
device.  :func:`rope` is differentiable; the cache's operators are for serving,
and their results have no gradient.  Index data that only the device can check
is reported by ``fmha_native_b200.status()`` as ``FMHA_ERR_INDEX``.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import Optional, Sequence

import torch

import fmha_native_b200 as _fm

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


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


def _bad(what: str):
    return _fm.FmhaError(_fm.FMHA_ERR_ARG, what)


def _load_binding():
    """The torch binding (checks, allocation, the calls), bound to the loaded library."""
    path = os.path.join(_fm.PKG_DIR, "_torch_binding.so")
    if not os.path.exists(path):
        raise _fm.FmhaError(_fm.FMHA_ERR_DEVICE, f"torch binding not built: {path} "
                            "(run `python -m fmha_native_b200.build`)")
    lib = _fm.load_library()
    spec = importlib.util.spec_from_file_location("fmha_native_b200._torch_binding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.bind(*(ctypes.cast(getattr(lib, n), _P).value
               for n in ("fmha_rope_d64_bf16", "fmha_paged_append_d64_bf16", "fmha_paged_fwd_d64_bf16",
                         "fmha_prefix_fwd_d64_bf16", "fmha_paged_workspace_bytes")), _fm.FmhaError)
    return mod


_binding = _load_binding()
_call_rope, _call_append, _call_attend = _binding.rope, _binding.append, _binding.attend
_LAYOUTS = {"thd": 0, "htd": 1, "bshd": 2, "bhsd": 3}


def _layout(x, layout: Optional[str]) -> int:
    if layout is None:
        return 0 if getattr(x, "ndim", 4) == 3 else 2  # (what is no tensor is refused by the call)
    try:
        return _LAYOUTS[layout]
    except KeyError:
        raise _bad(f"unknown layout {layout!r}") from None


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


def _operand(g):
    """A gradient as the operators take it: autograd also hands out expanded ones."""
    ok = g.stride(-1) == 1 and all(s % 8 == 0 for s in g.stride()[:-1]) and g.data_ptr() % 16 == 0
    return g if ok else g.contiguous()


class _Rope(torch.autograd.Function):
    """rope under autograd: the map is linear, and its transpose the rotation back."""

    @staticmethod
    def forward(ctx, q, k, cos_sin, positions, sections, axis_of, interleaved, inverse, layout):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos_sin, positions)
        ctx.kw = dict(sections=sections, axis_of=axis_of, interleaved=interleaved, inverse=not inverse, layout=layout)
        both = rope(q, k, cos_sin, positions, **dict(ctx.kw, inverse=inverse))
        ctx.mark_non_differentiable(*(y for x, y in zip((q, k), both) if x is not None and not x.requires_grad))
        return both

    @staticmethod
    def backward(ctx, dq, dk):
        dq, dk = (None if g is None else _operand(g) for g in (dq, dk))
        if dq is None:
            dq, dk = (None, None) if dk is None else (None, rope(dk, None, *ctx.saved_tensors, **ctx.kw)[0])
        else:
            dq, dk = rope(dq, dk, *ctx.saved_tensors, **ctx.kw)
        return (dq, dk) + (None,) * 7


def rope(q, k, cos_sin, positions, *, sections=None, axis_of=None, interleaved: bool = False, inverse: bool = False,
         layout: Optional[str] = None, out=None, stream=None):
    """Q and K (which may be None) with their pairs rotated by the tokens' positions.

    ``positions``: int32 over q's token dimensions (``[total]`` or ``[batch,
    seqlen]``), or ``[axes, ...]`` for positions with several axes (time,
    height, width).  ``sections`` gives how many consecutive pairs each axis
    turns; ``axis_of`` names the axis of every pair instead.  ``interleaved``:
    pairs (2j, 2j+1) instead of (j, j + rot_dim/2).  Dimensions from rot_dim on
    pass through.  ``out``: the tensors to write, which may be q and k
    themselves (not while autograd records them).  Layouts: "thd", "htd", "bshd",
    "bhsd".  Differentiable in q and k.
    """
    if (getattr(q, "requires_grad", False) or getattr(k, "requires_grad", False)) and torch.is_grad_enabled():
        if out is not None:
            raise _bad("rope with out= has no gradient, and q or k requires one")
        if stream is None or not isinstance(q, torch.Tensor):
            return _Rope.apply(q, k, cos_sin, positions, sections, axis_of, interleaved, inverse, layout)
        here = torch.cuda.current_stream(q.device)
        with torch.cuda.stream(_fm.named_stream(stream, q.device)):  # the gradient runs there too
            both = _Rope.apply(q, k, cos_sin, positions, sections, axis_of, interleaved, inverse, layout)
        for x in both:
            if x is not None:
                x.record_stream(here)
        return both
    q_out, k_out = out if out is not None else (None, None)
    return _call_rope(q, k, cos_sin, positions, sections, axis_of, interleaved, inverse, _layout(q, layout), q_out,
                      k_out, stream)


def rope_bwd(dq, dk, cos_sin, positions, **kw):
    """Gradients of :func:`rope`'s inputs from its outputs', for callers that
    keep no autograd graph: the rotation back (a rotation's transpose), same
    arguments."""
    return rope(dq, dk, cos_sin, positions, inverse=True, **kw)


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
    return _call_append(k, v, k_cache, v_cache, page_table, seqlens_k, q, cos_sin, positions, sections, axis_of,
                        interleaved, cu_seqlens_q, _layout(k, layout), q_out, stream)


def paged_workspace_bytes(batch: int, seqlen_q: int, heads_q: int, heads_k: int, total_q: int = 0,
                          prefix_len: int = 0) -> int:
    """Bytes of device scratch that :func:`paged_fwd` (``prefix_len`` 0) or
    :func:`prefix_fwd` needs for these sizes (``total_q`` > 0: packed tokens, of
    which a sequence has at most ``seqlen_q``)."""
    return int(_fm.load_library().fmha_paged_workspace_bytes(batch, seqlen_q, total_q, heads_q, heads_k, prefix_len))


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
    return _call_attend(q, k_cache, v_cache, page_table, seqlens_k, None, 0, causal, cu_seqlens_q, max_seqlen_q, scale,
                        return_lse, _layout(q, layout), out, lse_out, workspace, stream)


def prefix_fwd(q, k_cache, v_cache, prefix_pages, prefix_len: int, page_table, seqlens_k, *, causal: bool = True,
               cu_seqlens_q=None, max_seqlen_q: Optional[int] = None, scale: Optional[float] = None,
               return_lse: bool = False, layout: Optional[str] = None, out=None, lse_out=None, workspace=None,
               stream=None):
    """:func:`paged_fwd` where every sequence's keys are the ``prefix_len`` keys
    in ``prefix_pages`` (int32 ``[pages]``) followed by its own ``seqlens_k[b]``
    ones in ``page_table``: the prefix is read once for the whole batch.
    ``causal`` concerns the sequences' own keys; all tokens see the prefix."""
    return _call_attend(q, k_cache, v_cache, page_table, seqlens_k, prefix_pages, prefix_len, causal, cu_seqlens_q,
                        max_seqlen_q, scale, return_lse, _layout(q, layout), out, lse_out, workspace, stream)
