"""insmos_amd.autograd.linear under what a caller's program may wrap around it: forward-mode differentiation."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from insmos_amd.autograd import linear


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", ["leaf", "plain", "no_grad"])
def test_linear_refuses_forward_mode_tangents(which, grad):
    """A tangent is refused, whether or not the tape is on: without one the product's share of a jvp would be missing without an error."""
    args = [torch.zeros(4, 8), torch.zeros(8, 6), torch.zeros(6), torch.zeros(4, 6)]
    with fwad.dual_level():
        args[which] = fwad.make_dual(args[which].requires_grad_(grad == "leaf"), torch.ones_like(args[which]))
        with torch.set_grad_enabled(grad != "no_grad"), pytest.raises(NotImplementedError, match="forward-mode"):
            linear(*args)
    with pytest.raises(ValueError, match="on the GPU"):    # outside the level there is no tangent
        linear(*[t.detach() for t in args])
