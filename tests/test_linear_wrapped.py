"""insmos_amd.autograd.linear under what a caller's program may wrap around it: forward-mode differentiation, tracers, fake tensors,
dispatch modes, subclasses and torch.func's transforms."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from insmos_amd.autograd import linear


def _layer(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).cuda() for s in ((40, 24), (24, 16), (16,), (40, 16))]


def _nodes(graph):
    return [n for n in graph.nodes if n.op == "call_function" and "insmos.linear" in str(n.target)]


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


@pytest.mark.parametrize("act,first", [("silu", True), ("relu", False), (None, False)])
@pytest.mark.parametrize("out_in", [False, True])
def test_linear_on_fake_tensors(act, first, out_in):
    """Shapes, types and layouts of what the layer and its gradients would give, without a device."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    with FakeTensorMode():
        x, w, b, r = (torch.empty(s, dtype=torch.bfloat16).requires_grad_() for s in ((5, 4, 24), (16, 24) if out_in else (24, 16), (16,), (5, 4, 16)))
        y = linear(x, w.t() if out_in else w, b, r, activation=act, residual_first=first)
        grads = torch.autograd.grad(y, (x, w, b, r), torch.empty_like(y))
        with pytest.raises(ValueError, match="weight"):
            linear(x, torch.empty((23, 16), dtype=torch.bfloat16))
    assert isinstance(y, FakeTensor) and y.shape == (5, 4, 16) and y.dtype == torch.bfloat16
    for g, t in zip(grads, (x, w, b, r)):
        assert isinstance(g, FakeTensor) and g.shape == t.shape and g.dtype == t.dtype


@pytest.mark.parametrize("grads", [False, True])
def test_linear_in_a_recorded_graph(grads):
    """make_fx over fake tensors: the layer (and its backward pass) is a node that its inputs lead to, and not the empty tensor that it fills."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x, w, b):
        y = linear(x, w, b, activation="gelu") * 2
        return torch.autograd.grad(y.sum(), (x, w, b)) if grads else y

    with FakeTensorMode() as mode:
        args = [torch.empty(s).requires_grad_(grads) for s in ((40, 24), (24, 16), (16,))]
        with mode:
            graph = make_fx(f)(*args).graph
    nodes = _nodes(graph)
    assert [str(n.target) for n in nodes] == ["insmos.linear.default"] + ["insmos.linear_backward.default"] * grads
    assert [n.name for n in nodes[0].all_input_nodes] == [n.name for n in graph.nodes if n.op == "placeholder"]


def test_linear_refuses_function_transforms():
    x, w = torch.zeros(4, 8), torch.zeros(8, 6)
    for f in (lambda: torch.func.vmap(lambda r: linear(r, w))(x), lambda: torch.func.grad(lambda r: linear(r, w).sum())(x),
              lambda: torch.func.jvp(lambda r: linear(r, w), (x,), (x,))):
        with pytest.raises(NotImplementedError, match="linear"):
            f()


class _Marked(torch.Tensor):
    """A subclass that leaves everything to torch."""


class _Counting(torch.Tensor):
    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        if func is linear:
            return "seen"
        return super().__torch_function__(func, types, args, kwargs or {})


def test_linear_asks_subclasses():
    x, w = torch.zeros(4, 8), torch.zeros(8, 6)
    assert linear(x, w.as_subclass(_Counting)) == "seen"
    with pytest.raises(ValueError, match="on the GPU"):
        linear(x.as_subclass(_Marked), w)
    with pytest.raises(ValueError, match="on the GPU"):
        linear(torch.nn.Parameter(x), torch.nn.Parameter(w))


@pytest.mark.gpu
@pytest.mark.parametrize("act,first", [("silu", True), ("relu", False), ("relu", True), (None, False)])
def test_linear_traced(act, first):
    """A traced module computes the layer of the inputs that it is called with, and its gradients."""
    x, w, b, r = _layer()
    traced = torch.jit.trace(lambda x_, r_: linear(x_, w, b, r_, activation=act, residual_first=first), (x, r))
    x2, _, _, r2 = _layer(1)
    assert torch.equal(traced(x2, r2), linear(x2, w, b, r2, activation=act, residual_first=first))
    ins, ref = [[t.clone().requires_grad_() for t in (x2, r2)] for _ in range(2)]
    dy = torch.randn(40, 16, device="cuda")
    got = torch.autograd.grad(traced(*ins), ins, dy)
    want = torch.autograd.grad(linear(ref[0], w, b, ref[1], activation=act, residual_first=first), ref, dy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("out_in", [False, True])
@pytest.mark.parametrize("act,first", [("gelu", True), ("relu", False), ("relu", True), (None, True)])
def test_linear_under_a_dispatch_mode(act, first, out_in):
    """A mode that lets everything through sees the operators, and the results are the ones without it; a second derivative raises there too."""
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, w, b, r = _layer()
    w = w.t().contiguous().t() if out_in else w
    ins = [t.detach().requires_grad_() for t in (x, w, b, r)]
    dy = torch.randn(40, 16, device="cuda")
    want_y = linear(*ins, activation=act, residual_first=first)
    want = torch.autograd.grad(want_y, ins, dy)
    with Watch():
        y = linear(*ins, activation=act, residual_first=first)
        got = torch.autograd.grad(y, ins, dy)
        again = torch.autograd.grad(linear(*ins, activation=act).sum(), ins[0], create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(again.sum(), ins[1])
    assert torch.equal(y, want_y) and all(torch.equal(a, c) and a.stride() == c.stride() for a, c in zip(got[:3], want))
    assert torch.equal(got[3], want[3])
    assert seen.count("insmos.linear.default") == 2 and seen.count("insmos.linear_backward.default") >= 2


@pytest.mark.gpu
def test_linear_keeps_plain_subclasses():
    x, w, b, r = _layer()
    y = linear(x.as_subclass(_Marked), w, b, r, activation="gelu")
    assert type(y) is _Marked and torch.equal(y.as_subclass(torch.Tensor), linear(x, w, b, r, activation="gelu"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("out_in", [False, True])
@pytest.mark.parametrize("act,first", [(0, False), (1, True), (1, False), (2, True), (4, False)])
def test_linear_operator_is_registered_soundly(act, first, out_in, dtype):
    """torch's own checks of the registered operators: schema (nothing mutated or aliased), autograd, fake results like the real ones."""
    from insmos_amd import autograd as A
    t = getattr(torch, dtype)
    x, w, b, r = (v.to(t) for v in _layer())
    w = w.t().contiguous().t() if out_in else w
    leaves = [v.detach().requires_grad_() for v in (x, w, b, r)]
    torch.library.opcheck(A._linear_op, (*leaves, act, first), test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    y, slope = A._linear_op(x, w, b, r, act, first)
    held = slope if act > 1 or not first else y
    torch.library.opcheck(A._linear_backward_op, (torch.randn_like(y), held, x, w, act, not first, [True] * 4), test_utils=("test_schema", "test_faketensor"))
