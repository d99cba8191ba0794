"""What the backward pass of insmos_amd.autograd.linear makes of the activation's slopes where they are far from 1 and where gradients are not
finite."""
import pytest
import torch

from insmos_amd.autograd import linear

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _one_each(z, t, act, residual=None, first=False):
    """The layer on inputs whose z are the given values (a product with the identity), and its leaves (x, weight, bias, residual)."""
    n = z.shape[1]
    ins = [z.to(t).cuda(), torch.eye(n, dtype=t, device="cuda"), torch.zeros(n, dtype=t, device="cuda")]
    if residual is not None:
        ins.append(residual.to(t).cuda())
    ins = [v.requires_grad_(True) for v in ins]
    return linear(*ins[:3], ins[3] if residual is not None else None, activation=act, residual_first=first), ins


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("act,z", [("gelu", -6.0), ("gelu", -5.0), ("gelu_tanh", -6.0), ("silu", -15.0), ("silu", -25.0), ("gelu", -0.75), ("gelu", 40.0)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_linear_gradients_that_are_not_finite_stay_so(dtype, act, z, bad):
    """However small the slope is, inf and NaN times it are neither finite nor lost: in dz, in its column of dw and db and in its row of dx."""
    t = DTYPES[dtype]
    zs = torch.full((40, 16), z)
    y, ins = _one_each(zs, t, act, torch.zeros(40, 16), True)
    dy = torch.ones(40, 16, dtype=t, device="cuda")
    dy[7, 3] = bad
    dx, dw, db, dr = torch.autograd.grad(y, ins, dy)
    hit = torch.zeros(40, 16, dtype=torch.bool, device="cuda")
    hit[7, 3] = True
    assert torch.equal(~dr.isfinite(), hit)
    assert torch.equal(~db.isfinite(), hit.any(0))
    assert bool((~dw.isfinite())[:, 3].all()) and bool(dw.isfinite()[:, :3].all())
    assert bool((~dx.isfinite())[7].any()) and bool(dx.isfinite()[:7].all()) and bool(dx.isfinite()[8:].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("residual", ["none", "first", "after"])
def test_linear_a_shut_relu_keeps_what_comes_from_behind(dtype, residual):
    t = DTYPES[dtype]
    z = torch.tensor([[2.0, -2.0, 0.0, 3.0]]).repeat(40, 4)
    y, ins = _one_each(z, t, "relu", None if residual == "none" else torch.zeros(40, 16), residual == "first")
    dy = torch.tensor([[1.0, float("inf"), float("nan"), -float("inf")]]).repeat(40, 4).to(t).cuda()
    db = torch.autograd.grad(y, ins[2], dy)[0]
    want = torch.tensor([40.0, 0.0, 0.0, -float("inf")]).repeat(4).to(t).cuda()
    assert torch.equal(db, want)
