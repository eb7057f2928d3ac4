"""What the serving operators write in place: autograd learns of it."""
import pytest
import torch

import fmha_native_b200 as fm
from paged_harness import normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(cuda_device):
    fm.status()


def test_tensors_written_in_place_say_so():
    """A tensor that autograd saved may not change unnoticed."""
    q, k = normal((33, 6, 64), 1), normal((33, 2, 64), 2)
    table, pos = fm.rope_table(200), torch.randint(0, 200, (3, 33), device="cuda", dtype=torch.int32)
    kw = dict(sections=(8, 12, 12))
    x = q.clone().requires_grad_()
    y = x.exp()
    with torch.no_grad():
        fm.rope(y, None, table, pos, out=(y, None), **kw)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    kc, vc, qo = (torch.zeros(2, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    q1, k1 = q[:2, None], k[:2, None]
    t, n = torch.arange(2, device="cuda", dtype=torch.int32)[:, None], torch.ones(2, device="cuda", dtype=torch.int32)
    o, lse = torch.empty_like(q1), torch.empty(2, 6, 1, device="cuda")
    qo = torch.empty_like(q1)
    before = [w._version for w in (kc, vc, qo, o, lse)]
    fm.paged_append(k1, k1, kc, vc, t, n, q=q1, cos_sin=table, q_out=qo)
    fm.paged_fwd(qo, kc, vc, t, n, out=o, lse_out=lse, return_lse=True)
    assert all(w._version > v for w, v in zip((kc, vc, qo, o, lse), before))
    with torch.inference_mode():
        z = torch.empty_like(q)
    with torch.no_grad():
        fm.rope(q, None, table, pos, out=(z, None), **kw)  # inference tensors have no version
