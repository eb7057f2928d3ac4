"""C ABI of the serving operators (include/fmha_paged.h): layout, exports, and
the argument checks that need no GPU."""
import ctypes
import os
import re
import subprocess

import pytest

import fmha_native_b200 as fm

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exports():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "fmha_paged.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(fmha_\w+)\s*\(", text))
    assert {"fmha_rope_d64_bf16", "fmha_paged_append_d64_bf16", "fmha_paged_fwd_d64_bf16", "fmha_prefix_fwd_d64_bf16",
            "fmha_paged_workspace_bytes"} == names
    lib = fm.load_library()
    for n in names:
        assert getattr(lib, n)
    assert lib.fmha_fwd_d64_error_string(fm.FMHA_ERR_INDEX).startswith(b"a page id")


@pytest.mark.parametrize("name", ["FmhaRopeParams", "FmhaPagedParams"])
def test_layout_matches_c(tmp_path, name):
    struct = getattr(fm, name)
    fields = [f[0] for f in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fmha_paged.h"\nint main(void){\n'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + f'printf("%zu\\n", sizeof({name}));\nreturn 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


BASE = 1 << 20  # fake, 16-byte aligned device addresses (never dereferenced)


def rope_params(append=False):
    p = fm.FmhaRopeParams()
    for i, f in enumerate(("q", "k", "q_out", "k_out", "cos_sin", "positions")):
        setattr(p, f, BASE * (i + 1))
    for t in ("q", "k", "v", "qo", "ko", "vo"):
        setattr(p, f"stride_{t}", 256)
        setattr(p, f"nhead_stride_{t}", 64)
        setattr(p, f"batch_stride_{t}", 256 * 16)
    p.batch, p.seqlen_q, p.nhead_q, p.nhead_k, p.max_pos, p.n_pairs = 2, 3, 4, 2, 100, 32
    if append:
        p.v, p.v_out, p.page_table, p.seqlens_k = BASE * 7, BASE * 8, BASE * 9, BASE * 10
        p.page_size, p.num_pages, p.max_pages, p.table_stride = 16, 8, 4, 4
    return p


def paged_params():
    p = fm.FmhaPagedParams()
    for i, f in enumerate(("q", "k_cache", "v_cache", "o", "page_table", "seqlens_k", "prefix_pages", "workspace")):
        setattr(p, f, BASE * (i + 1))
    p.workspace_bytes = 1 << 40
    for t in ("q", "o"):
        setattr(p, f"stride_{t}", 256)
        setattr(p, f"nhead_stride_{t}", 64)
        setattr(p, f"batch_stride_{t}", 256)
    for t in ("k", "v"):
        setattr(p, f"stride_{t}", 128)
        setattr(p, f"nhead_stride_{t}", 64)
        setattr(p, f"page_stride_{t}", 128 * 16)
    p.batch, p.seqlen_q, p.nhead_q, p.nhead_k = 2, 1, 4, 2
    p.page_size, p.num_pages, p.max_pages, p.table_stride, p.prefix_len, p.scale = 16, 8, 4, 4, 30, 0.18
    return p


def status(entry, p):
    return getattr(fm.load_library(), entry)(ctypes.byref(p) if p is not None else None, None)


@pytest.mark.parametrize("change", [
    dict(q_out=None), dict(k_out=BASE + 2), dict(cos_sin=None), dict(positions=None), dict(n_pairs=12),
    dict(max_pos=0), dict(stride_q=100), dict(nhead_stride_ko=0), dict(seqlen_q=-1), dict(q=None, k=None),
    dict(v=BASE), dict(axis_of=(ctypes.c_uint8 * 32)(*[4] * 32)), dict(axis_stride=-1),
    dict(seqlen_q=1 << 30, batch=64),
], ids=str)
def test_rope_arguments(change):
    p = rope_params()
    for k, v in change.items():
        setattr(p, k, v)
    assert status("fmha_rope_d64_bf16", p) == fm.FMHA_ERR_ARG


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(v_out=BASE + 4), dict(page_table=None), dict(seqlens_k=None), dict(page_size=12),
    dict(page_size=4), dict(page_size=8192), dict(max_pages=-1), dict(inverse=1), dict(stride_ko=60),
    dict(batch_stride_vo=4), dict(batch=0), dict(table_stride=-4),
], ids=str)
def test_append_arguments(change):
    p = rope_params(True)
    for k, v in change.items():
        setattr(p, k, v)
    assert status("fmha_paged_append_d64_bf16", p) == fm.FMHA_ERR_ARG


@pytest.mark.parametrize("entry", ["fmha_paged_fwd_d64_bf16", "fmha_prefix_fwd_d64_bf16"])
@pytest.mark.parametrize("change", [
    dict(q=None), dict(o=BASE + 2), dict(k_cache=None), dict(page_table=None), dict(seqlens_k=None), dict(workspace=None),
    dict(workspace=BASE + 8), dict(workspace_bytes=100), dict(nhead_k=3), dict(nhead_k=0), dict(batch=0), dict(seqlen_q=-1),
    dict(page_size=24), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(stride_q=4), dict(stride_o=0),
    dict(page_stride_k=9), dict(max_pages=(1 << 31) - 1), dict(seqstart_q=BASE, total_q=5, seqlen_q=0),
], ids=str)
def test_attention_arguments(entry, change):
    p = paged_params()
    if "stride_o" in change or "stride_q" in change:
        p.seqlen_q = 2  # (a stride of one element is never used)
    for k, v in change.items():
        setattr(p, k, v)
    assert status(entry, p) == fm.FMHA_ERR_ARG


def test_prefix_arguments():
    for change in (dict(prefix_len=0), dict(prefix_len=-5), dict(prefix_pages=None)):
        p = paged_params()
        for k, v in change.items():
            setattr(p, k, v)
        assert status("fmha_prefix_fwd_d64_bf16", p) == fm.FMHA_ERR_ARG
    for entry in ("fmha_rope_d64_bf16", "fmha_paged_append_d64_bf16", "fmha_paged_fwd_d64_bf16", "fmha_prefix_fwd_d64_bf16"):
        assert status(entry, None) == fm.FMHA_ERR_ARG


def test_valid_calls_without_gpu_return_a_status():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these calls would launch on fake pointers")
    for entry, p in (("fmha_rope_d64_bf16", rope_params()), ("fmha_paged_append_d64_bf16", rope_params(True)),
                     ("fmha_paged_fwd_d64_bf16", paged_params()), ("fmha_prefix_fwd_d64_bf16", paged_params())):
        assert status(entry, p) == fm.FMHA_ERR_DEVICE


def test_workspace_bytes():
    f = fm.paged_workspace_bytes
    assert f(0, 1, 8, 2) == 0 and f(1, 1, 8, 3) == 0 and f(1, -1, 8, 2) == 0
    small, wide = f(4, 1, 8, 2), f(4, 1, 8, 2, 0, 1000)
    assert 0 < small < wide
    assert f(4, 1, 8, 2) == f(64, 1, 8, 2)  # single tokens: does not grow with the batch
    assert f(4, 100, 8, 2, 200) >= f(4, 1, 8, 2, 4)


def test_refusals_without_gpu():
    import torch

    x = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: fm.paged_fwd(x, x, x, x, x), lambda: fm.rope(x, None, x, x),
                 lambda: fm.paged_append(x, x, x, x, x, x), lambda: fm.paged_fwd(None, x, x, x, x, layout="bshd"),
                 lambda: fm.rope(x, None, x, x, layout="xyz")):
        with pytest.raises(fm.FmhaError) as e:
            call()
        assert e.value.status == fm.FMHA_ERR_ARG
