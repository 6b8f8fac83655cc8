"""(h) The 8-bit product has no gradients: whatever input asks for one, or carries a tangent, is refused, since a result without a word
would leave its part out of a loss."""
import pytest
import torch
from torch.autograd import forward_ad

from fastmd_amd.ops.int8 import Int8Rows, linear_int8


def calls(rows, scales, w_scales, bias, device="cpu"):
    """Both forms of x, with the given tensors."""
    q = Int8Rows(torch.ones(5, 32, dtype=torch.int8, device=device), scales)
    w = Int8Rows(torch.ones(6, 32, dtype=torch.int8, device=device), w_scales)
    return {"rows": lambda: linear_int8(rows, w, bias), "rounded": lambda: linear_int8(q, w, bias)}


def tensors(device="cpu"):
    return [torch.ones(s, device=device) for s in ((5, 32), (5,), (6,), (6,))]


CASES = [("rows", 0), ("rows", 2), ("rows", 3), ("rounded", 1), ("rounded", 2), ("rounded", 3)]


@pytest.mark.parametrize("form,which", CASES)
def test_inputs_that_need_a_gradient_are_refused(form, which):
    t = tensors()
    t[which].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        calls(*t)[form]()
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):  # nothing to lose there: refused for its device alone
        calls(*t)[form]()


@pytest.mark.parametrize("form,which", CASES)
def test_tangents_are_refused(form, which):
    t = tensors()
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(ValueError, match="no gradient"):
            calls(*t)[form]()


@pytest.mark.gpu
@pytest.mark.parametrize("form,which", CASES)
def test_on_the_gpu(form, which):
    t = tensors("cuda")
    want = calls(*t, "cuda")[form]()
    t[which].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        calls(*t, "cuda")[form]()
    with torch.no_grad():
        assert torch.equal(calls(*t, "cuda")[form](), want)
