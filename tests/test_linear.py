"""insmos_amd.autograd.linear (csrc/linear*.hip, csrc/host_tensors.cpp): forward and gradients against the formulas in float64, with
element-wise bounds that follow from the roundings; layouts, alignments and sizes where a kernel can go wrong; refusals."""
import ctypes

import pytest
import torch

from insmos_amd import _lib
from insmos_amd.autograd import linear

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U32 = 2.0 ** -24          # half a step of fp32, relative


def _act(z, name):
    if name is None:
        return z
    if name == "relu":
        return torch.relu(z)
    if name == "silu":
        return torch.nn.functional.silu(z)
    return torch.nn.functional.gelu(z, approximate="tanh" if name == "gelu_tanh" else "none")


def _case(M, K, N, dtype, act, residual, layout, bias=True, pads=(0, 0, 0), seed=0):
    """Inputs on the GPU: x, residual and dy as slices of wider rows (pads), the weight in either layout.  For relu small integers and a
    bias of halves: z is exact in every type and never at relu's border, where a rounding would decide."""
    g = torch.Generator().manual_seed(seed)
    t = DTYPES[dtype]

    def rows(m, n, pad, scale=1.0, whole=False):
        v = torch.randint(-2, 3, (m, n + pad), generator=g).float() if whole else scale * torch.randn(m, n + pad, generator=g)
        v = v.to(t).cuda()
        if pad:
            v[:, n:] = float("nan")    # what lies between the rows must not be used
        return v[:, :n]

    relu = act == "relu"
    x = rows(M, K, pads[0], whole=relu)
    w = rows(K, N, 0, K ** -0.5, whole=relu) if layout == "in_out" else rows(N, K, 0, K ** -0.5, whole=relu).t()
    b = ((torch.randint(-2, 3, (N,), generator=g).float() + 0.5) if relu else 0.3 * torch.randn(N, generator=g)).to(t).cuda() if bias or relu else None
    r = rows(M, N, pads[1], whole=relu) if residual else None
    dy = rows(M, N, pads[2])
    return x, w, b, r, dy


def _check(x, w, b, r, dy, act, first, grads=True):
    half = torch.finfo(x.dtype).eps / 2
    ins = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(ins)
    xi, wi = next(it), next(it)
    bi = next(it) if b is not None else None
    ri = next(it) if r is not None else None
    y = linear(xi, wi, bi, ri, activation=act, residual_first=first)
    with torch.no_grad():
        same = linear(x, w, b, r, activation=act, residual_first=first)
    assert torch.equal(y.detach(), same)                       # with and without a tape: the same kernel and bits
    X, W, D = x.double(), w.double(), dy.double()
    z, S = X @ W, X.abs() @ W.abs()                            # S bounds the partial sums
    if b is not None:
        z, S = z + b.double(), S + b.double().abs()
    if first:
        z, S = z + r.double(), S + r.double().abs()
    z = z.detach().requires_grad_(True)
    a = _act(z, act)
    K, N, M = w.shape[0], w.shape[1], x.shape[0]
    ez = (K + 4) * U32 * S                                     # K products and sums, bias, residual: one rounding each
    ea = 1.13 * ez + (8 * U32 * (1 + z.abs()) * (1 + z.abs()) if act not in (None, "relu") else 0)   # slopes <= 1.13; exp of up to z^2: its argument's rounding
    ref, ey = a.detach(), ea
    if r is not None and not first:
        ref, ey = ref + r.double(), ey + U32 * (ref.abs() + r.double().abs())
    ok = (y.double() - ref).abs() <= half * ref.abs() + (1 + half) * ey + 1e-30 + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert bool(ok.all()), ("y", float((y.double() - ref).abs().max()))
    if not grads:
        return
    got = torch.autograd.grad(y, ins, dy)
    (slope,) = torch.autograd.grad(a, z, torch.ones_like(a))
    # the slope as used: fp32, or 16 bits in steps of 2^-15; |act''| <= 1.13 carries the error of z; relu's is exact here
    es = torch.zeros_like(slope) if act in (None, "relu") else 1.2 * ez + 16 * U32 * (1 + z.detach() ** 2) + (2.0 ** -16 if x.dtype != torch.float32 else 0)
    dz = D * slope
    edz = D.abs() * es + U32 * dz.abs()                        # before the rounding to the type
    half0 = half if act is not None or x.dtype == torch.float32 else 0.0
    edz16 = edz + half0 * (dz.abs() + edz) + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-30   # half of fp16's smallest step
    want = [(dz @ W.t(), edz16 @ W.abs().t() + (N + 2) * U32 * (dz.abs() @ W.abs().t())),
            (X.t() @ dz, X.abs().t() @ edz16 + (M + 2) * U32 * (X.abs().t() @ dz.abs()))]
    if b is not None:
        want.append((dz.sum(0), edz.sum(0) + (M + 2) * U32 * dz.abs().sum(0)))
    if r is not None:
        want.append((dz, edz) if first else (D, torch.zeros_like(D)))
    for name, g, (ref, e) in zip(("dx", "dw", "db", "dr"), got, want):
        assert g.shape == ref.shape and g.dtype == x.dtype
        ok = (g.double() - ref).abs() <= half * ref.abs() + (1 + half) * e + tiny
        assert bool(ok.all()), (name, float((g.double() - ref).abs().max()), float(e.max()))


SHAPES = [(1, 1, 1), (1, 8, 8), (1, 64, 40), (2, 1001, 33), (13, 130, 257), (32, 512, 64), (33, 64, 32), (40, 72, 24), (64, 33, 65), (100, 1, 100),
          (129, 200, 136), (130, 17, 1), (257, 96, 40), (300, 513, 515), (700, 64, 300), (16, 8192, 48), (1024, 40, 8), (5000, 24, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_against_float64(M, K, N, dtype):
    for i, (act, residual, first) in enumerate(((None, False, False), ("relu", True, True), ("gelu", True, False), ("silu", False, False),
                                                ("gelu_tanh", True, True), ("relu", True, False))):
        layout = ("in_out", "out_in")[(i + M) % 2]
        _check(*_case(M, K, N, dtype, act, residual, layout, bias=(i + K) % 2 == 0, seed=i), act, first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("pads", [(8, 8, 8), (5, 3, 1), (1, 16, 2)])
@pytest.mark.parametrize("M,K,N", [(7, 72, 40), (150, 40, 72), (260, 130, 134), (90, 33, 47), (140, 67, 129)])
def test_linear_rows_of_any_pitch(M, K, N, pads, dtype):
    """Rows as slices of wider matrices with NaN between them: pitches that are and are not multiples of 16 bytes."""
    for layout in ("in_out", "out_in"):
        _check(*_case(M, K, N, dtype, "gelu", True, layout, pads=pads, seed=3), "gelu", False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(1024, 512, 768), (513, 2048, 264), (2100, 256, 2056), (20000, 64, 128), (3000, 128, 64), (24, 3000, 96), (4096, 1, 8)])
def test_linear_every_tile(M, K, N, dtype):
    """Sizes that take the large tile, the narrow ones, several parts of k and the last, partial tiles of each."""
    for layout in ("in_out", "out_in"):
        _check(*_case(M, K, N, dtype, "silu", True, layout, seed=5), "silu", True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_linear_shapes_strides_and_broadcasts(dtype):
    t = DTYPES[dtype]
    torch.manual_seed(1)
    w = (torch.randn(24, 40) * 0.2).to(t).cuda()
    b = torch.randn(40).to(t).cuda()
    flat = torch.randn(60, 24).to(t).cuda()
    want = linear(flat, w, b, activation="silu")
    assert torch.equal(linear(flat.view(3, 4, 5, 24), w, b, activation="silu"), want.view(3, 4, 5, 40))
    assert torch.equal(linear(flat.t().contiguous().t(), w, b, activation="silu"), want)              # columns apart
    assert torch.equal(linear(flat[0], w, b, activation="silu"), linear(flat[:1], w, b, activation="silu")[0])
    assert torch.equal(linear(flat[::2], w, b, activation="silu"), linear(flat[::2].contiguous(), w, b, activation="silu"))
    wide = torch.randn(24, 80).to(t).cuda()
    assert torch.equal(linear(flat, wide[:, ::2], b), linear(flat, wide[:, ::2].contiguous(), b))     # a weight with both strides
    assert torch.equal(linear(flat, wide[:, 3:43], b), linear(flat, wide[:, 3:43].contiguous(), b))   # an address off the 16-byte grid
    one = torch.randn(1, 24).to(t).cuda()
    assert torch.equal(linear(one.expand(60, 24), w, b), linear(one.repeat(60, 1), w, b))
    # a residual of one row for all, and its gradient: the sum over the rows
    row = torch.randn(40).to(t).cuda().requires_grad_(True)
    y = linear(flat, w, b, row.expand(60, 40), activation="gelu")
    assert torch.equal(y.detach(), linear(flat, w, b, row.detach().expand(60, 40).contiguous(), activation="gelu"))
    dy = torch.randn(60, 40).to(t).cuda()
    (g,) = torch.autograd.grad(y, row, dy)
    half = torch.finfo(t).eps / 2
    ref = dy.double().sum(0)
    assert bool(((g.double() - ref).abs() <= 61 * half * dy.double().abs().sum(0)).all())             # (torch adds the rows)
    # the same tensor twice: x as its own residual
    sq = (torch.randn(40, 40) * 0.1).to(t).cuda()
    x = torch.randn(50, 40).to(t).cuda().requires_grad_(True)
    dy = torch.randn(50, 40).to(t).cuda()
    (gx,) = torch.autograd.grad(linear(x, sq, None, x), x, dy)
    ref = dy.double() @ sq.double().t() + dy.double()
    S = dy.double().abs() @ sq.double().abs().t() + dy.double().abs()
    assert bool(((gx.double() - ref).abs() <= 3 * half * S).all())
    # a gradient that is an expanded scalar
    x = flat.detach().requires_grad_(True)
    linear(x, w).sum().backward()
    ref = w.double().sum(1).expand(60, 24)
    assert bool(((x.grad.double() - ref).abs() <= half * ref.abs() + 42 * U32 * w.double().abs().sum(1)).all())


@pytest.mark.gpu
def test_linear_empty_and_partly_needed():
    w = torch.randn(8, 16, device="cuda", requires_grad=True)
    b = torch.randn(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = linear(x, w, b, activation="silu")
    assert y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.any() and not b.grad.any()
    assert linear(torch.empty(3, 0, 8, device="cuda"), w.detach()).shape == (3, 0, 16)
    assert linear(torch.randn(3, 8, device="cuda"), torch.empty(8, 0, device="cuda")).shape == (3, 0)
    x = torch.randn(50, 8, device="cuda")
    r = torch.randn(50, 16, device="cuda")
    full = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    dy = torch.randn(50, 16, device="cuda")
    want = torch.autograd.grad(linear(*full, activation="gelu", residual_first=True), full, dy)
    for i in range(4):      # one at a time
        ins = [t.detach().requires_grad_(j == i) for j, t in enumerate(full)]
        (g,) = torch.autograd.grad(linear(*ins, activation="gelu", residual_first=True), ins[i], dy)
        assert torch.equal(g, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_linear_extremes(act):
    """Far values, infinities and NaN behave as the activation's formula does, in the row and column that they are in alone."""
    for dtype in ("fp32", "bf16"):
        x = torch.zeros(40, 16, dtype=DTYPES[dtype], device="cuda")
        w = torch.eye(16, 24, dtype=DTYPES[dtype], device="cuda")
        values = torch.tensor([0.0, -0.0, 50.0, -50.0, 1e4, -1e4, 1e30, -1e30, 1e-30, 12.0, -12.0, 5.0, -5.0, 1.0, -1.0, 0.25])
        x[3] = values.to(x.dtype)
        x[5, 7] = float("nan")
        x = x.requires_grad_(True)
        y = linear(x, w, activation=act)
        z = x.detach().double() @ w.double()
        z[5] = z[6]                                                  # (NaN times zero is NaN in the whole row: checked below)
        ref = _act(z.clamp(-1e15, 1e15), act)
        ref = torch.where(z.abs() > 1e15, torch.where(z > 0, z, torch.zeros_like(z)), ref)
        rest = [i for i in range(40) if i != 5]
        got = y.detach().double()[rest]
        ok = bool(((got - ref[rest]).abs() <= torch.finfo(x.dtype).eps / 2 * ref[rest].abs() + 2e-6 * (1 + z[rest].abs().clamp(max=1))).all())
        assert ok, y[3].tolist()
        assert bool(torch.isnan(y.detach()[5, 7])) and bool(torch.isfinite(y.detach()[rest]).all())
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
        fine = [i for i in range(40) if i not in (3, 5)]
        assert bool(torch.isfinite(g[fine]).all())
    big = torch.full((4, 64), 6e4, dtype=torch.float16, device="cuda")
    assert bool(torch.isinf(linear(big, torch.ones(64, 8, dtype=torch.float16, device="cuda"))).all())   # fp16's range ends there


@pytest.mark.gpu
def test_linear_gradients_against_differences():
    """(f(p + h v) - f(p - h v)) / 2 h against <gradient, v> in fp32: the second is off by h^2 / 6 f''' and by f's rounding / h."""
    torch.manual_seed(2)
    x, w, b, r = (torch.randn(40, 20, device="cuda"), 0.3 * torch.randn(20, 24, device="cuda"), torch.randn(24, device="cuda"),
                  torch.randn(40, 24, device="cuda"))
    c = torch.randn(40, 24, device="cuda")
    for act in ("gelu", "gelu_tanh", "silu"):
        ins = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        grads = torch.autograd.grad((linear(*ins, activation=act, residual_first=True) * c).sum(), ins)
        for i in range(4):
            v = torch.randn_like(ins[i])
            v /= v.norm()
            h = 2e-2
            f = []
            for s in (1, -1):
                moved = [t.detach() + (s * h * v if j == i else 0) for j, t in enumerate(ins)]
                f.append(float((linear(*moved, activation=act, residual_first=True).double() * c.double()).sum()))
            diff, want = (f[0] - f[1]) / (2 * h), float((grads[i].double() * v.double()).sum())
            # f's terms: 960 of size |c y| ~ 1 with errors 1e-7 each; f''' h^2 / 6 with f''' ~ |c| |dz / dp|^3 ~ 100
            assert abs(diff - want) < 960 * 1e-6 / h / 30 + 100 * h * h / 6, (act, i, diff, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_linear_offsets_past_32_bits(dtype):
    """Rows whose byte offsets pass 2^31 and 2^32 in x, dy and the gradients' long sum."""
    t = DTYPES[dtype]
    es = torch.finfo(t).bits // 8
    M, pitch = 70000, (1 << 16) // es * 2          # 128 KB rows: 9 GB
    buf = torch.zeros(M, pitch, dtype=t, device="cuda")
    buf[:, :40] = torch.randn(M, 40, device="cuda").to(t)
    x = buf[:, :40]
    w = (torch.randn(40, 72, device="cuda") * 0.1).to(t)
    dy = buf[:, :72]                               # (the same memory: inputs only)
    xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = linear(xs, ws)
    gx, gw = torch.autograd.grad(y, (xs, ws), dy)
    half = torch.finfo(t).eps / 2
    for i in (0, 16383, 16384, 32767, 32768, 65535, M - 1):
        ref = x[i].double() @ w.double()
        assert bool(((y[i].double() - ref).abs() <= half * ref.abs() + 50 * U32 * (x[i].double().abs() @ w.double().abs()) + 1e-7).all()), i
        ref = dy[i].double() @ w.double().t()
        assert bool(((gx[i].double() - ref).abs() <= half * ref.abs() + 80 * U32 * (dy[i].double().abs() @ w.double().abs().t()) + 1e-7).all()), i
    ref, S = x.double().t() @ dy.double(), x.double().abs().t() @ dy.double().abs()
    # (x and dy share memory, so the diagonal sums 70 000 squares of mean 1: 70 000 is past fp16's largest number 65 504, and inf its rounding)
    over = ref.abs() > torch.finfo(t).max
    assert bool(torch.isinf(gw[over]).all()) and int(over.sum()) == (40 if dtype == "fp16" else 0)
    assert bool(((gw.double() - ref).abs() <= half * ref.abs() + M * U32 * S)[~over].all())


@pytest.mark.gpu
def test_linear_is_deterministic_on_any_stream_and_in_graphs():
    """The same bits from every run, from two streams at once, and from replays of two captured graphs (forward and backward) that do not
    share workspaces, with eager work between the replays."""
    torch.manual_seed(4)
    x = torch.randn(300, 1100, device="cuda").bfloat16()
    w = (torch.randn(1100, 64, device="cuda") * 0.03).bfloat16()     # several parts of k
    b = torch.randn(64, device="cuda").bfloat16()
    dy = torch.randn(300, 64, device="cuda").bfloat16()

    def step(x, dy):
        ins = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = linear(*ins, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, ins, dy))

    want = step(x, dy)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step(x, dy))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for g in got for a, c in zip(g, want))
    del got
    graphs, outs, ins = [], [], []
    for k in range(2):
        xi, di = x.clone(), dy.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xi, di)
        graphs.append(g)
        outs.append(out)
        ins.append((xi, di))
    for rep in range(4):
        fresh = [(torch.randn_like(x), torch.randn_like(dy)) for _ in range(2)]
        for (xi, di), (a, c) in zip(ins, fresh):
            xi.copy_(a)
            di.copy_(c)
        for g in graphs:
            g.replay()
        eager = [step(a, c) for a, c in fresh]
        torch.cuda.synchronize()
        for out, e in zip(outs, eager):
            assert all(torch.equal(p, q) for p, q in zip(out, e)), rep


@pytest.mark.gpu
def test_linear_once_differentiable():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), w)


def test_linear_refusals():
    x, w = torch.zeros(4, 8), torch.zeros(8, 6)
    for text, args, kw in (("activation", (x, w), {"activation": "tanh"}), ("activation", (x, w), {"activation": ["relu"]}),
                           ("float32, bfloat16 or float16", (x.double(), w.double()), {}), ("weight", (x, torch.zeros(7, 6)), {}),
                           ("weight", (x, torch.zeros(8)), {}), ("weight is", (x, w.half()), {}), ("bias", (x, w, torch.zeros(5)), {}),
                           ("bias is", (x, w, torch.zeros(6).half()), {}), ("residual", (x, w, None, torch.zeros(6)), {}),
                           ("residual", (x, w, None, torch.zeros(4, 5)), {}), ("widths", (torch.zeros(4, 0), torch.zeros(0, 6)), {}),
                           ("widths", (torch.zeros(1, 1 << 21), torch.zeros(1 << 21, 1)), {}), ("on the GPU", (x, w), {}),
                           ("sparse", (x, w.to_sparse()), {})):
        with pytest.raises(ValueError, match=text):
            linear(*args, **kw)
    with pytest.raises(ValueError):
        linear(x.requires_grad_(True), torch.zeros(7, 6))


def test_linear_entry_points_refuse():
    """The C entries return their codes before any launch (none of these calls reaches the device)."""
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def forward(x=p, ldx=8, w=p, ldw=16, out_in=0, bias=None, res=None, ldr=0, act=0, M=4, K=8, N=16, dt=0, y=p, ldy=16, slope=None, lds=16, ws=p, n=1024):
        return lib.insmos_linear(x, ldx, w, ldw, out_in, bias, res, ldr, 0, act, M, K, N, dt, y, ldy, slope, lds, ws, n, None)

    for bad in ({"x": None}, {"w": None}, {"y": None}, {"K": 0}, {"N": 0}, {"M": -1}, {"M": 1 << 31}, {"K": 1 << 21}, {"dt": 3}, {"act": 5}, {"act": -1},
                {"ldx": 7}, {"ldw": 15}, {"ldw": 7, "out_in": 1}, {"ldy": 15}, {"x": p + 2}, {"bias": p + 1}, {"res": p, "ldr": -1}, {"res": p + 1, "ldr": 16},
                {"slope": p}, {"slope": p + 4, "act": 2}, {"slope": p, "act": 2, "lds": 15}, {"ws": p + 8}, {"ldx": 1 << 21}):
        assert forward(**bad) == -1, bad
    assert forward(M=0) == 0
    # 16-bit rows at an odd pitch, and no room for the copy
    assert forward(M=200, ldx=9, dt=1, n=0) == -3 and forward(M=200, ldx=9, dt=2, ws=None) == -3
    assert lib.insmos_linear_ws_bytes(4, 0, 8, 0) == 0 and lib.insmos_linear_ws_bytes(4, 8, 8, 7) == 0

    def backward(dy=p, ldd=16, slope=None, lds=16, kind=0, x=p, ldx=8, w=p, ldw=16, M=4, K=8, N=16, dt=0, dx=p, lddx=8, dw=p, lddw=16, dz=None, lddz=16, ws=p, n=1024):
        return lib.insmos_linear_backward(dy, ldd, slope, lds, kind, x, ldx, w, ldw, 0, M, K, N, dt, dx, lddx, dw, lddw, None, dz, lddz, ws, n, None)

    for bad in ({"M": 0}, {"dy": None}, {"kind": 1}, {"kind": 2}, {"kind": 3}, {"kind": 2, "slope": p + 4}, {"x": None}, {"w": None}, {"lddx": 7}, {"lddw": 15},
                {"dz": p + 4}, {"dz": p, "lddz": 15}, {"dt": -1}, {"ldd": 15}):
        assert backward(**bad) == -1, bad
    assert backward(kind=1, slope=p, n=0) == -3      # dz needs room


@pytest.mark.gpu
def test_linear_captured_beside_a_live_eager_graph():
    """An eager graph on the default stream keeps its leaves' nodes: a backward pass that is captured on another stream would reach them, and is
    refused.  Once that graph is gone the same capture works and replays what an eager pass gives."""
    gen = torch.Generator().manual_seed(31)
    x, gy = torch.randn(37, 24, generator=gen).cuda(), torch.randn(37, 16, generator=gen).cuda()
    w = (torch.randn(24, 16, generator=gen) * 0.3).cuda().requires_grad_(True)
    alive = linear(x, w, activation="silu")
    (want,) = torch.autograd.grad(alive, w, gy, retain_graph=True)
    torch.cuda.synchronize()

    def capture():
        g, out = torch.cuda.CUDAGraph(), None
        with torch.cuda.graph(g):
            try:
                (out,) = torch.autograd.grad(linear(x, w, activation="silu"), w, gy)
            except RuntimeError as e:
                out = str(e)
        return g, out

    _, said = capture()
    assert isinstance(said, str) and "being captured" in said
    del alive
    g, out = capture()
    assert torch.is_tensor(out), out
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(4090, 2100, 4090), (4000, 300, 1901), (2050, 8200, 2050), (61, 700, 30002), (8200, 520, 2055)])
def test_linear_large_tiles(M, K, N, dtype):
    """Sizes that take the 256 x 256 tile (whole and with k in parts), the 128 x 128 one and 64 and 32 rows of it, each with partial last tiles."""
    for layout in ("in_out", "out_in"):
        _check(*_case(M, K, N, dtype, "gelu_tanh", True, layout, seed=8), "gelu_tanh", False)


@pytest.mark.gpu
def test_linear_negated_views():
    """The imaginary part of a conjugate: a view whose memory holds the values with the other sign, as every operand and as the gradient."""
    gen = torch.Generator().manual_seed(12)
    imag = lambda *s: torch.conj(torch.randn(*s, dtype=torch.complex64, generator=gen).cuda()).imag   # noqa: E731
    x, w, b, r, dy = imag(20, 12), imag(12, 9), imag(9), imag(20, 9), imag(20, 9)
    assert x.is_neg()
    plain = [t.resolve_neg().contiguous() for t in (x, w, b, r, dy)]
    ins, ref = [t.detach().requires_grad_(True) for t in (x, w, b, r)], [t.requires_grad_(True) for t in plain[:4]]
    y, want = linear(*ins, activation="silu"), linear(*ref, activation="silu")
    assert torch.equal(y, want)
    for g, e in zip(torch.autograd.grad(y, ins, dy), torch.autograd.grad(want, ref, plain[4])):
        assert torch.equal(g, e)


@pytest.mark.gpu
def test_linear_in_checkpoints_and_with_saved_tensor_hooks():
    """Recomputation in the backward pass and packed saved tensors give the same gradients."""
    from torch.utils.checkpoint import checkpoint
    gen = torch.Generator().manual_seed(13)
    x, w, b = (torch.randn(s, generator=gen).cuda().requires_grad_(True) for s in ((50, 24), (24, 16), (16,)))
    f = lambda x_, w_, b_: linear(x_, w_, b_, activation="gelu")   # noqa: E731
    want = torch.autograd.grad(f(x, w, b).square().sum(), (x, w, b))
    got = torch.autograd.grad(checkpoint(f, x, w, b, use_reentrant=False).square().sum(), (x, w, b))
    assert all(torch.equal(g, e) for g, e in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        y = f(x, w, b)
    got = torch.autograd.grad(y.square().sum(), (x, w, b))
    assert all(torch.equal(g, e) for g, e in zip(got, want))
    x2 = x.detach().clone().requires_grad_(True)
    y = f(x2, w, b)
    with torch.no_grad():
        x2.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y.sum(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(5, 9001, 40), (32, 4096, 160), (9, 6000, 1030), (1, 600, 9000), (31, 77, 8200), (3, 1025, 512)])
def test_linear_few_rows_both_ways(M, K, N, dtype):
    """Up to 32 rows: sizes on either side of the choice between their own kernel and tiles with parts of k, odd operands among them."""
    for layout in ("in_out", "out_in"):
        _check(*_case(M, K, N, dtype, "silu", True, layout, seed=17), "silu", True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [("bf16", (0x7FC0, 0x7FFF, 0x7F81, -0x40, -1)), ("fp16", (0x7E00, 0x7FFF, 0x7C01, 0x7D55, -1))])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_linear_nan_of_any_payload_reaches_the_gradients(dtype, bits, act):
    """NaNs with all kinds of bits in x, in the bias and in the residual: the slopes that are stored in 16 bits say so too (dz, and with it dx and the
    weight's gradient, is NaN where z is)."""
    t = DTYPES[dtype]
    x = torch.ones(len(bits) + 40, 16, dtype=t, device="cuda")
    x[:len(bits), 0] = torch.tensor(bits, dtype=torch.int16).view(t).cuda()
    w, r = torch.full((16, 24), 0.1, dtype=t, device="cuda"), torch.zeros(len(bits) + 40, 24, dtype=t, device="cuda")
    r[-1, 3] = torch.tensor(bits[1], dtype=torch.int16).view(t).cuda()
    ins = [v.requires_grad_(True) for v in (x, w, r)]
    y = linear(x, w, None, r, activation=act, residual_first=True)
    dx, dw, dr = torch.autograd.grad(y, ins, torch.ones_like(y))
    want = torch.zeros_like(y, dtype=torch.bool)
    want[:len(bits)] = True
    want[-1, 3] = True
    assert torch.equal(y.isnan(), want) and torch.equal(dr.isnan(), want)
    assert torch.equal(dx.isnan().any(1), want.any(1)) and bool(dw.isnan().all())
