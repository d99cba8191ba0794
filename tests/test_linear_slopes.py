"""What the backward pass of insmos_amd.autograd.linear makes of the activation's slopes where they are far from 1 and where gradients are not
finite."""
import math

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


U32 = 2.0 ** -24


def _slope64(z, act):
    """act'(z) in float64 without the cancellation of 1 + erf and 1 + tanh (which leave 1e-16, 1 % of gelu's slope at -12)."""
    z = z.double()
    if act == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c, d = (1.0, 0.0) if act == "silu" else (2 * math.sqrt(2 / math.pi), 0.044715)      # both are z / (1 + exp(-u)), u = c (z + d z^3)
    u = c * (z + d * z ** 3)
    s, rest = torch.sigmoid(u), torch.sigmoid(-u)
    return s + z * s * rest * c * (1 + 3 * d * z * z)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("act,least", [("silu", -22.0), ("gelu", -6.5), ("gelu_tanh", -5.5)])
def test_linear_slopes_in_the_tails_keep_their_size(dtype, act, least):
    """dz against the slope in float64, relative to the slope itself.  Its errors: the 16-bit types' code, 2^-10 of a slope below 2^-6 in size and 2^-16
    above; the exponential's, whose argument (up to z^2 / 2 or 1.6 |z| + 0.1 |z|^3) is rounded in fp32; where |z| < 3 that of terms of size 1 which
    nearly cancel; one rounding to the type (fp16: half of its smallest step at least)."""
    t = DTYPES[dtype]
    n = 64
    z = torch.linspace(least, 0.5, 40 * n).view(40, n).to(torch.bfloat16).float()      # exact in every type
    gen = torch.Generator().manual_seed(3)
    # gradients of a scaled loss: what fp16 has least of stays small against dz
    dy = (1024.0 * (1 + torch.rand(40, n, generator=gen))).to(t).cuda()
    y, ins = _one_each(z, t, act, torch.zeros(40, n), True)
    dz = torch.autograd.grad(y, ins[3], dy)[0].double()
    s = _slope64(z.cuda(), act)
    code = torch.where(s.abs() < 2.0 ** -6, 2.0 ** -10 * s.abs(), torch.full_like(s, 2.0 ** -16)) if dtype != "fp32" else 0
    arg = 8 * U32 * (1 + z.cuda().double() ** 2 + 0.1 * z.cuda().double().abs() ** 3) * (s.abs() + (z.cuda().abs() < 3))
    want, e = dy.double() * s, dy.double() * (code + arg) * (1 + 2.0 ** -10)
    half = torch.finfo(t).eps / 2
    ok = (dz - want).abs() <= half * want.abs() + (1 + half) * e + (2.0 ** -25 if dtype == "fp16" else 1e-30)
    assert bool(ok.all()), ((dz - want).abs() / want.abs())[~ok].max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act,bias", [("silu", -12.0), ("silu", -18.0), ("gelu", -5.0), ("gelu_tanh", -4.5)])
def test_linear_a_unit_that_is_far_in_the_tail_learns(dtype, act, bias):
    """A strongly negative bias: the slopes of all rows are small and of one sign.  db (a sum in fp32, rounded once) is off by 2^-10 of the sum, the
    exponentials' errors and its own rounding; dw and dx take dz rounded to the type once more each."""
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(5)
    x, w = (torch.rand(200, 32, generator=gen) * 0.1).to(t).cuda(), (torch.rand(32, 24, generator=gen) * 0.1).to(t).cuda()
    b = torch.full((24,), bias, dtype=t, device="cuda")
    dy = (1024.0 * (1 + torch.rand(200, 24, generator=gen))).to(t).cuda()
    ins = [v.requires_grad_(True) for v in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear(*ins, activation=act), ins, dy)
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    z = X @ W + bias
    dz = D * _slope64(z, act)
    half = torch.finfo(t).eps / 2
    # z itself: 34 sums and products of at most 12 + 0.4, and d log(slope) / dz of at most |z| + 1 (gelu_tanh: 1.6 + 0.22 z^2 < 8)
    rel = 2.0 ** -10 + 8 * U32 * (1 + bias ** 2 + 0.1 * abs(bias) ** 3) + 34 * U32 * (abs(bias) + 1) * 20
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0      # (dz in fp16: half of the smallest step)
    for g, ref, each in ((db, dz.sum(0), 0.0), (dw, X.t() @ dz, X.t() @ (half * dz.abs() + tiny)), (dx, dz @ W.t(), (half * dz.abs() + tiny) @ W.t())):
        off = (g.double() - ref).abs()
        assert bool((off <= (half + rel) * (1 + half) * ref.abs() + 200 * U32 * ref.abs() + each * (1 + 2.0 ** -7) + tiny).all()), float((off / ref.abs()).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_linear_slopes_of_far_values(act, dtype):
    """The gradients of values far out: slope 0 on one side and 1 on the other, finite, where a formula has 0 times infinity.  Nearer ones against
    float64 (errors as above)."""
    t = DTYPES[dtype]
    far = [50.0, -50.0, 1e4, -1e4, 6e4, -6e4] + ([] if dtype == "fp16" else [1e19, -1e19, 2e19, -2e19, 1e30, -1e30, 3e38, -3e38])
    near = [0.0, -0.0, 12.0, -12.0, 5.0, -5.0, 1.0, -1.0, 0.25, 8.0, -8.0, 20.0, -20.0]
    z = torch.tensor([far + near + [0.0] * (32 - len(far) - len(near))])
    y, ins = _one_each(z, t, act, torch.zeros(1, 32), True)
    dz = torch.autograd.grad(y, ins[3], torch.ones_like(y))[0].double()
    zs = ins[0].detach().double()
    s = (zs > 0).double() if act == "relu" else _slope64(zs.clamp(-700, 700), act)    # (from 700 on 0 and 1 to 1e-300)
    assert bool(dz.isfinite().all())
    half, arg = torch.finfo(t).eps / 2, 8 * U32 * (1 + zs.clamp(-40, 40) ** 2 + 0.1 * zs.clamp(-40, 40).abs() ** 3) * (s.abs() + (zs.abs() < 3))
    code = 0 if dtype == "fp32" or act == "relu" else torch.where(s.abs() < 2.0 ** -6, 2.0 ** -10 * s.abs() + 2.0 ** -38, torch.full_like(s, 2.0 ** -16))
    off = (dz - s).abs()
    assert bool((off <= half * s.abs() + (1 + half) * (arg + code) + (2.0 ** -25 if dtype == "fp16" else 2.0 ** -126)).all()), off.max()
