"""Soft reads at the edges of their ranges."""
import pytest

from test_gpu_attention import TYPES

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ---- empty sides -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq,lk", [(0, 2000), (2000, 0), (0, 100_000), (3000, 0)])
def test_gradient_of_a_call_with_an_empty_side(fm, lq, lk, dtype):
    # long enough that the streamed rows, were there any, would be cut into ranges
    q, k, v = (torch.ones(2, n, h, 64, dtype=TYPES[dtype], device="cuda") for n, h in ((lq, 4), (lk, 2), (lk, 2)))
    out, lse = fm.attend(q, k, v, return_lse=True)
    gq, gk, gv = fm.attend_backward(q, q, k, v, out, lse)
    assert gq.shape == q.shape and gk.shape == k.shape and gv.shape == v.shape
    assert (gq == 0).all() and (gk == 0).all() and (gv == 0).all()
    fm.check_attention_status()
