"""More of the residual stream's operators on the GPU: calls and paths beside those of test_residual_gpu.py, whose helpers,
oracles in 64 bits and tolerances these tests use."""
import pytest

from tests.test_residual_gpu import BF, F16, F32, PAIRS, L, backward64, dt, gen, near, rand  # noqa: F401 (L is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,res", PAIRS)
@pytest.mark.parametrize("rows,dim", [(1, 1), (37, 640), (300, 1001), (5, 9000)])
def test_weight_gradient_without_a_gradient_of_the_norm(L, act, res, rows, dim):
    """No gradient reaches y: its weight's gradient is zeros, and the others are those of a call that does not ask for it."""
    import torch
    g = gen(rows + dim)
    total, h, dh = rand((rows, dim), act, g), rand((rows, dim), res, g), rand((rows, dim), res, g)
    w1, w2 = rand((dim,), act, g, 0.1, 1.0), rand((dim,), act, g, 0.1, 1.0)
    ds, dres, dw1, dw2 = torch.empty_like(total), torch.empty_like(h), torch.empty_like(w1), torch.full_like(w2, 3.0)
    L.reduce_norm_backward(h, None, dh, ds, dres, total=total, post_weight=w1, pre_weight=w2, post_weight_grad=dw1,
                           pre_weight_grad=dw2)
    assert bool((dw2 == 0).all())
    want, mag = backward64(total, None, None, dh, w1, None, None, 0, 1.0, 1e-6, 0.0, True, False)
    near(ds, want["send"], mag["send"], 256, "send")
    assert torch.equal(dres, dh)
    near(dw1, want["w1"], mag["w1"], 160, "w1")
    with pytest.raises(L.FlagcxError):  # the norm's input is needed for it
        L.reduce_norm_backward(None, None, dh, ds, dres, total=total, post_weight=w1, pre_weight=w2, pre_weight_grad=dw2)
