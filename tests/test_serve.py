"""The serving loop: what its operators give together, against the dense kernel
and 64 bits over the same keys."""
import pytest
import torch

import fmha_native_b200 as fm

pytestmark = pytest.mark.gpu


def test_serving_steps_match_attention_over_all_keys(cuda_device):
    from fmha_native_b200.serve import Server

    srv = Server(slots=5, prefix_len=333, max_len=400, page=16)
    lengths = [1, 40, 130, 17, 301]
    srv.prompts(lengths, [0, 16, 25, 0, 100])
    for _ in range(4):
        _, trace = srv.decode()
    assert fm.status() == fm.FMHA_OK
    kv = srv.kv
    assert kv.host_lengths == [n + 4 for n in lengths]
    for layer, (q, o) in enumerate(trace):
        prefix = srv.prefix_pages.long()
        for b, n in enumerate(kv.host_lengths):
            own = kv.table[b, : -(-n // kv.page)].long()

            def keys(cache):
                return torch.cat([cache[layer][prefix].flatten(0, 1)[:333], cache[layer][own].flatten(0, 1)[:n]])

            k, v = keys(kv.k).double(), keys(kv.v).double()
            g = q.shape[2] // k.shape[1]
            k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
            p = torch.softmax(torch.einsum("hd,khd->hk", q[b, 0].double(), k) / 8, -1)
            want, size = torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs())
            # weights and output are each rounded to bf16 once, 2^-8 of their value
            assert ((o[b, 0].double() - want).abs() <= 2.0 ** -8 * (size + want.abs()) + 2.0 ** -13 * size).all()
            # the dense kernel over the same keys (it truncates its weights to bf16: 2^-7)
            dense = fm.fmha_fwd(q[b][None], keys(kv.k)[None].contiguous(), keys(kv.v)[None].contiguous())
            assert ((dense[0, 0].double() - want).abs() <= 2.0 ** -7 * size + 2.0 ** -8 * want.abs() + 2.0 ** -13 * size).all()


def test_pages_come_back(cuda_device):
    from fmha_native_b200.serve import Server

    srv = Server(slots=2, prefix_len=20, max_len=64, page=16)
    free = len(srv.kv.free)
    srv.prompts([40, 50], [0, 0])
    assert len(srv.kv.free) == free - 7
    srv.kv.release(0)
    srv.kv.release(1)
    assert len(srv.kv.free) == free
    with pytest.raises(fm.FmhaError):
        srv.kv.pages_for(10 ** 6)


def test_command(cuda_device, capsys):
    from fmha_native_b200 import serve

    assert serve.main(["--requests", "4", "--prefix", "100", "--steps", "3"])["requests"] == 4
    assert "tokens/s" in capsys.readouterr().out
