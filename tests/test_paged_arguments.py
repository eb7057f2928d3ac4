"""Refusals of the serving operators that need no GPU."""
import pytest
import torch

import fmha_native_b200 as fm


@pytest.mark.parametrize("layout", [None, "thd", "bshd"])
def test_operands_that_are_no_tensors(layout):
    x = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: fm.rope(None, x, x, x, layout=layout), lambda: fm.rope(3, x, x, x, layout=layout),
                 lambda: fm.rope_bwd(None, x, x, x, layout=layout),
                 lambda: fm.paged_append(None, x, x, x, x, x, layout=layout),
                 lambda: fm.paged_fwd(None, x, x, x, x, layout=layout),
                 lambda: fm.prefix_fwd([1], x, x, x, 5, x, x, layout=layout)):
        with pytest.raises(fm.FmhaError) as e:
            call()
        assert e.value.status == fm.FMHA_ERR_ARG


@pytest.mark.gpu
def test_a_cache_without_heads_is_refused(cuda_device):
    """Not answered with a q that nothing wrote."""
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    k, kc = q[:, :, :0], torch.zeros(3, 16, 0, 64, dtype=torch.bfloat16, device="cuda")
    t, n = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(fm.FmhaError):
        fm.paged_append(k, k, kc, kc, t, n, q=q)


def test_no_q_beside_a_k_that_requires_a_gradient():
    x = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    for stream in (None, 12345):
        with pytest.raises(fm.FmhaError):
            fm.rope(None, x.clone().requires_grad_(), x, x, stream=stream)
