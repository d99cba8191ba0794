"""insmos_amd.optim (csrc/optim.hip, csrc/host_tensors.cpp): the AdamW / Adam step against its formula in float64, with bounds from the
roundings; the 8-bit moments code for code; the clip; what must stay untouched; the Optimizer class; refusals."""
import copy
import ctypes

import numpy as np
import pytest
import torch

from insmos_amd import _lib
from insmos_amd.optim import AdamW, adamw_step, grad_norm, state_offsets

U32 = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
SIZES = [1, 3, 255, 256, 257, 5000, 0, 70001, 4096, 2]


def _layout(tensors):
    starts, total = state_offsets([t.numel() for t in tensors])
    return [(a, t.numel()) for a, t in zip(starts, tensors)], total


def _make(dtype, bits, masters, sizes=SIZES, seed=0, offset=0):
    """params, grads, m, v, step, scales, masters; offset: elements that every tensor's address is moved by."""
    g = torch.Generator().manual_seed(seed)

    def at(n, scale):
        buf = torch.empty(n + offset + 1, dtype=dtype, device="cuda")
        v = buf[offset:offset + n]
        v.copy_((scale * torch.randn(n, generator=g)).to(dtype))
        return v

    params = [at(n, 0.5) for n in sizes]
    grads = [at(n, 10.0 ** (-1 - i % 4)) for i, n in enumerate(sizes)]
    for q in grads[3:6]:
        q[::3] = 0
    lay, total = _layout(params)
    m, v = torch.zeros(total), torch.zeros(total)
    for a, n in lay:
        m[a:a + n] = 0.01 * torch.randn(n, generator=g)
        v[a:a + n] = (0.02 * torch.randn(n, generator=g)) ** 2 + 1e-8
    scales = None
    if bits == 8:
        r = torch.sqrt(v).view(-1, 256)
        scales = torch.stack([t.abs().amax(1).clamp_min(1e-30) / 448 for t in (m.view(-1, 256), r)])
        m = (m.view(-1, 256) / scales[0][:, None]).to(torch.float8_e4m3fn).view(-1)
        v = (r / scales[1][:, None]).to(torch.float8_e4m3fn).view(-1)
        scales = scales.cuda()
    w = None
    if masters:
        w = torch.zeros(total)
        for (a, n), p in zip(lay, params):
            w[a:a + n] = p.float().cpu() + 1e-4 * torch.randn(n, generator=g)
        w = w.cuda()
    step = torch.full((1,), 6, dtype=torch.int32, device="cuda")
    return params, grads, m.cuda(), v.cuda(), step, scales, w


def _decode(code, scale):
    return (code.float().view(-1, 256).double() * scale.double()[:, None]).view(-1)


def _formula(p, g, m, v, t, lr, wd, decoupled, clip):
    """(p, m, v) in float64 and bounds of what fp32 arithmetic may be off by."""
    g = g * clip
    eg = U32 * g.abs() * 2
    if not decoupled:
        eg = eg + 2 * U32 * ((wd * p).abs() + g.abs())
        g = g + wd * p
    m1, v1 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    em = 3 * U32 * ((B1 * m).abs() + ((1 - B1) * g).abs()) + (1 - B1) * eg
    ev = 5 * U32 * v1 + (1 - B2) * 2 * g.abs() * eg
    size, root = lr / (1 - B1 ** t), (1 - B2 ** t) ** -0.5
    d = torch.sqrt(v1) * root + EPS
    u = size * m1 / d
    p1 = (p * (1 - lr * wd) if decoupled else p) - u
    # sqrt halves v's relative error; division, size, sum: a rounding each
    ep = 4 * U32 * (p.abs() + u.abs()) + size * em / d + u.abs() * (0.5 * ev / v1.clamp_min(1e-300) + 6 * U32)
    return (p1, m1, v1), (ep, em, ev)


CASES = [(torch.float32, False, 0), (torch.float32, False, 1), (torch.bfloat16, False, 0), (torch.bfloat16, True, 0), (torch.float16, True, 3),
         (torch.float16, False, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("decoupled", [True, False])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e9])
@pytest.mark.parametrize("dtype,masters,offset", CASES)
def test_step_32_bits_against_float64(dtype, masters, offset, max_norm, decoupled):
    params, grads, m, v, step, _, w = _make(dtype, 32, masters, offset=offset)
    lay, _ = _layout(params)
    before = [(p.double().clone() if w is None else w[a:a + n].double().clone(), g.double().clone(), m[a:a + n].double(), v[a:a + n].double())
              for p, g, (a, n) in zip(params, grads, lay)]
    norm64 = sum(float((g ** 2).sum()) for _, g, _, _ in before) ** 0.5
    clip = 1.0 if max_norm is None else min(1.0, max_norm / (norm64 + 1e-6))
    lr, wd = 3e-3, 0.1
    norm = adamw_step(params, grads, m, v, step, lr=lr, weight_decay=wd, decoupled=decoupled, masters=w, max_grad_norm=max_norm)
    assert int(step) == 7
    if max_norm is None:
        assert norm is None
    else:
        assert norm.dtype == torch.float32 and norm.dim() == 0 and abs(float(norm) - norm64) <= 3 * U32 * norm64
    half = torch.finfo(dtype).eps / 2
    for (p0, g0, m0, v0), p, g, (a, n) in zip(before, params, grads, lay):
        assert torch.equal(g.double(), g0)
        (p1, m1, v1), (ep, em, ev) = _formula(p0, g0, m0, v0, 7, lr, wd, decoupled, clip)
        assert bool(((m[a:a + n].double() - m1).abs() <= em + 1e-38).all()) and bool(((v[a:a + n].double() - v1).abs() <= ev + 1e-38).all())
        got = p if w is None else w[a:a + n]
        tail = half * p1.abs() + (2.0 ** -25 if dtype == torch.float16 else 0) if w is None and dtype != torch.float32 else 0
        assert bool(((got.double() - p1).abs() <= ep * (1 + half) + tail).all())
        if w is not None:
            assert torch.equal(p, w[a:a + n].to(dtype))                     # the rounding of the master
        end = a + -(-n // 256) * 256
        for t in (m, v) + ((w,) if w is not None else ()):
            assert not t[a + n:end].any()


def _mix(x):
    x = x ^ (x >> np.uint32(16))
    x = (x * np.uint32(0x7FEB352D)).astype(np.uint32)
    x = x ^ (x >> np.uint32(15))
    x = (x * np.uint32(0x846CA68B)).astype(np.uint32)
    return x ^ (x >> np.uint32(16))


def _bits16(pos, t, seed):
    with np.errstate(over="ignore"):
        key = _mix(_mix(np.array([t], np.uint32)) ^ np.uint32(seed))
        h = _mix((pos & 0xFFFFFFFF).astype(np.uint32) + ((pos >> 32).astype(np.uint32) * np.uint32(0x9E3779B1)) + key)
    return (h & np.uint32(0xFFFF)).astype(np.float64) / 65536, (h >> np.uint32(16)).astype(np.float64) / 65536


def _rounded(x, ex, u, keep):
    """e4m3 values of the blocks of x in units of their scale, rounded by u in [0, 1); which of them an error of ex (and 1e-5 of the value)
    could move; scales."""
    x = x.reshape(-1, 256)
    scale = np.maximum(np.abs(x).max(1) / 448, 2.0 ** -126)
    y = np.minimum(np.abs(x) / scale[:, None], 448)
    gap = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    at = y / gap + u.reshape(-1, 256)
    q = np.minimum(np.floor(at) * gap, 448)
    near = np.abs(at - np.round(at)) < 2e-4 + ex.reshape(-1, 256) / scale[:, None] / gap
    if keep:
        q = np.where((y > 0) & (q == 0), 2.0 ** -9, q)
    return (q * np.sign(x)).reshape(-1), near.reshape(-1), scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,masters,offset", CASES)
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_step_8_bits_code_for_code(dtype, masters, offset, max_norm):
    params, grads, m, v, step, scales, w = _make(dtype, 8, masters, offset=offset, seed=1)
    lay, total = _layout(params)
    m0, r0 = _decode(m, scales[0]), _decode(v, scales[1])
    p0 = [p.double().clone() if w is None else w[a:a + n].double().clone() for p, (a, n) in zip(params, lay)]
    norm64 = sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5
    clip = 1.0 if max_norm is None else min(1.0, max_norm / (norm64 + 1e-6))
    lr, wd, seed = 3e-3, 0.1, 99
    adamw_step(params, grads, m, v, step, lr=lr, weight_decay=wd, masters=w, max_grad_norm=max_norm, scales=scales, seed=seed)
    want_m, want_v, err_m, err_v = (torch.zeros(total, dtype=torch.float64) for _ in range(4))
    half = torch.finfo(dtype).eps / 2
    for p_, p, g, (a, n) in zip(p0, params, grads, lay):
        (p1, m1, v1), (ep, em, ev) = _formula(p_, g.double(), m0[a:a + n], r0[a:a + n] ** 2, 7, lr, wd, True, clip)
        want_m[a:a + n], want_v[a:a + n] = m1.cpu(), torch.sqrt(v1).cpu()
        err_m[a:a + n] = (em + U32 * m0[a:a + n].abs()).cpu()                              # (the decoding's product)
        err_v[a:a + n] = ((0.5 * (ev / v1.clamp_min(1e-300)) + 3 * U32) * torch.sqrt(v1)).cpu()
        got = p if w is None else w[a:a + n]
        tail = half * p1.abs() + (2.0 ** -25 if dtype == torch.float16 else 0) if w is None and dtype != torch.float32 else 0
        # (m and v decoded by a multiplication in fp32: one rounding more each)
        more = 2 * U32 * (lr / (1 - B1 ** 7) * m0[a:a + n].abs() / (torch.sqrt(v1) * (1 - B2 ** 7) ** -0.5 + EPS) + (p1 - p_).abs())
        assert bool(((got.double() - p1).abs() <= (ep + more) * (1 + half) + tail).all())
        if w is not None:
            assert torch.equal(p, w[a:a + n].to(dtype))
    u = _bits16(np.arange(total, dtype=np.int64), 7, seed)
    for k, (code, want, err) in enumerate(((m, want_m.numpy(), err_m.numpy()), (v, want_v.numpy(), err_v.numpy()))):
        q, near, scale = _rounded(want, err, u[k], k == 1)
        assert near.mean() < 0.01
        got = code.float().cpu().double().numpy()
        assert np.array_equal(got[~near], q[~near])
        gap = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 2)
        assert (np.abs(got - q) <= gap).all()
        assert np.abs(scales[k].cpu().double().numpy() / scale - 1).max() < 1e-5
    for (a, n) in lay:      # padding stays zero
        end = a + -(-n // 256) * 256
        assert not m[a + n:end].float().any() and not v[a + n:end].float().any()


@pytest.mark.gpu
def test_8_bit_rounding_is_unbiased_and_reproducible():
    params, grads, m, v, step, scales, _ = _make(torch.float32, 8, False, sizes=[512], seed=2)
    runs, seeds = [], 400
    for seed in list(range(seeds)) + [0]:
        s = [t.clone() for t in (params[0], m, v, step, scales)]
        adamw_step([s[0]], grads, s[1], s[2], s[3], lr=1e-3, scales=s[4], seed=seed)
        runs.append((_decode(s[1], s[4][0]), _decode(s[2], s[4][1]), s[0]))
    assert torch.equal(runs[0][0], runs[-1][0]) and torch.equal(runs[0][1], runs[-1][1])      # the same seed: the same codes
    assert not torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][2], runs[1][2])    # another: other codes, the same parameters
    (_, m1, v1), _ = _formula(params[0].double(), grads[0].double(), _decode(m, scales[0]), _decode(v, scales[1]) ** 2, 7, 1e-3, 0.01, True, 1.0)
    for k, exact in enumerate((m1, torch.sqrt(v1))):
        mean = torch.stack([r[k] for r in runs[:seeds]]).mean(0)
        top = exact.abs().view(-1, 256).amax(1).repeat_interleave(256)
        gap = torch.exp2(torch.floor(torch.log2((exact.abs() * 448 / top).clamp_min(2.0 ** -6))) - 3) * top / 448
        # a mean of 400 draws with a deviation of at most half a gap each, 512 of them: 5 sigma (one in 1.7 million)
        big = exact.abs() > top * 2.0 ** -9 / 448                                             # (sqrt(v) below the smallest code is kept at it)
        assert bool(((mean - exact).abs()[big] <= 5 * 0.5 * gap[big] / seeds ** 0.5 + 1e-6 * top[big]).all())


@pytest.mark.gpu
def test_8_bit_zero_tiny_and_non_finite_blocks():
    n = 256 * 6
    p = torch.randn(n, device="cuda")
    g = torch.randn(n, device="cuda")
    m, v = (torch.zeros(n, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    scales = torch.zeros(2, 6, device="cuda")
    g[:256] = 0                        # nothing ever
    g[256:512] *= 1e-15
    g[512:768] *= 1e15
    g[770] = float("inf")
    g[1030] = float("nan")
    g[1280:1536] = 0
    g[1281] = 1e-3                     # one element of a block
    g[1282] = 1e-12
    p0 = p.clone()
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    adamw_step([p], [g], m, v, step, lr=1e-2, weight_decay=0.0, scales=scales)
    mf, vf = m.float(), v.float()
    assert torch.equal(p[:256], p0[:256]) and not mf[:256].any() and not vf[:256].any()
    # every finite gradient moves its parameter by lr in the first step (m = 0.1 g, sqrt(v) = sqrt(0.001) |g|; eps where g is tiny)
    for a, b in ((512, 768), (771, 1024), (1031, 1280)):
        assert bool(((p0 - p)[a:b].abs() - 1e-2).abs().max() < 1e-5)
    assert bool(torch.isnan(p[770])) and bool(torch.isnan(p[1030]))
    assert bool(torch.isnan(mf[770])) and bool(torch.isnan(vf[770])) and bool(torch.isnan(mf[1030]))
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[770, 1030]] = False
    assert bool(torch.isfinite(mf[rest]).all()) and bool(torch.isfinite(p[rest]).all()) and bool(torch.isfinite(scales).all())
    nonzero = rest & (g != 0)
    assert bool((vf[nonzero] > 0).all())            # sqrt(v) > 0 is not lost, however small beside its block's largest
    q = p.clone()                                   # ... so the next step stays a small one
    adamw_step([p], [g], m, v, step, lr=1e-2, weight_decay=0.0, scales=scales)
    assert float((p - q)[rest].abs().max()) < 0.05


@pytest.mark.gpu
def test_none_gradients_memory_order_and_misfits():
    torch.manual_seed(3)
    base = [torch.randn(40, 30, device="cuda"), torch.randn(7, device="cuda"), torch.randn(30, 40, device="cuda").t(), torch.randn(3, 5, 4, device="cuda").permute(2, 0, 1)]
    grads = [torch.randn(40, 30, device="cuda").t().contiguous().t(), None, torch.randn(40, 30, device="cuda"), torch.randn(4, 3, 5, device="cuda")]
    total = state_offsets([p.numel() for p in base])[1]
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = [torch.empty_strided(t.shape, t.stride(), device="cuda").copy_(t) for t in base]
    keep = [g.clone() if g is not None else None for g in grads]
    adamw_step(p, grads, m, v, step, lr=1e-2, weight_decay=0.0)
    assert torch.equal(p[1], base[1]) and all(a is None or torch.equal(a, b) for a, b in zip(grads, keep))
    for i in (0, 2, 3):      # element for element, whatever either tensor's memory order: the first step is lr sign(g)
        assert bool(((base[i] - p[i]) - 1e-2 * torch.sign(grads[i])).abs().max() < 1e-5)
    a = state_offsets([t.numel() for t in base])[0][1]
    assert not m[a:a + 256].any()


@pytest.mark.gpu
def test_grad_norm():
    torch.manual_seed(4)
    ts = [torch.randn(n, device="cuda") * s for n, s in ((1, 3), (8191, 1), (8192, 0.1), (8193, 2), (300000, 0.5))]
    ts += [torch.randn(5000, device="cuda").bfloat16(), torch.randn(77, 33, device="cuda").half().t(), torch.randn(50, 8, device="cuda")[:, ::2], None]
    ref = sum(float((t.double() ** 2).sum()) for t in ts if t is not None) ** 0.5
    a = grad_norm(ts)
    assert a.dim() == 0 and a.dtype == torch.float32 and abs(float(a) - ref) < 3 * U32 * ref and torch.equal(a, grad_norm(ts))
    assert abs(float(grad_norm([ts[3][1:]])) - float(ts[3][1:].double().norm())) < 3 * U32 * float(ts[3].double().norm())     # off the 16-byte grid
    for s in (1e-25, 1e25, 1e-37, 1e37):
        t = torch.full((1000,), s, device="cuda")
        assert abs(float(grad_norm([t])) / (s * 1000 ** 0.5) - 1) < 1e-5, s
    mixed = torch.cat([torch.full((10,), 1e-25, device="cuda"), torch.full((2,), 1e30, device="cuda")])
    assert abs(float(grad_norm([mixed])) / (1e30 * 2 ** 0.5) - 1) < 1e-5
    ts[1][5] = float("inf")
    assert float(grad_norm(ts)) == float("inf")
    ts[1][5] = float("nan")
    assert torch.isnan(grad_norm(ts))
    assert float(grad_norm([torch.zeros(10, device="cuda")])) == 0 and float(grad_norm([torch.zeros(0, device="cuda")])) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_skip_nonfinite_changes_nothing(bits):
    for bad in (float("inf"), float("nan")):
        params, grads, m, v, step, scales, _ = _make(torch.float32, bits, False, seed=5)
        grads[5][17] = bad
        before = [t.clone() for t in params + [m.view(torch.uint8), v.view(torch.uint8), step] + ([scales] if bits == 8 else [])]
        norm = adamw_step(params, grads, m, v, step, lr=1e-2, scales=scales, skip_nonfinite=True)
        assert not torch.isfinite(norm)
        after = params + [m.view(torch.uint8), v.view(torch.uint8), step] + ([scales] if bits == 8 else [])
        assert all(torch.equal(a, b) for a, b in zip(before, after))
        grads[5][17] = 0
        adamw_step(params, grads, m, v, step, lr=1e-2, scales=scales, skip_nonfinite=True)
        assert int(step) == 7 and not torch.equal(params[5], before[5])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_step_on_streams_and_in_graphs(bits):
    """Two lists on two streams at once, and two captured steps (with the clip and a learning rate on the device) replayed with new gradients
    and rates, against the same steps one by one."""
    def fresh(seed):
        return _make(torch.float32, bits, False, seed=seed)

    def one(s, lr):
        adamw_step(s[0], s[1], s[2], s[3], s[4], lr=lr, scales=s[5], max_grad_norm=0.3, seed=7)

    def state(s):
        return s[0] + [s[2].view(torch.uint8), s[3].view(torch.uint8), s[4]] + ([s[5]] if s[5] is not None else [])

    want = [fresh(i) for i in range(2)]
    for s in want:
        for _ in range(3):
            one(s, 1e-3)
    got, streams = [fresh(i) for i in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, st in zip(got, streams):
            with torch.cuda.stream(st):
                one(s, 1e-3)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for s, q in zip(want, got) for a, b in zip(state(s), state(q)))
    want, got = [fresh(i) for i in range(2)], [fresh(i) for i in range(2)]
    rate = torch.full((1,), 1e-3, device="cuda")
    graphs = []
    for s in got:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            one(s, rate)
        graphs.append(g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for rep in range(4):
        lr = 1e-3 * (rep + 1)
        rate.fill_(lr)
        for s, q in zip(want, got):
            for a, b in zip(s[1], q[1]):
                new = torch.randn(a.shape, generator=gen, device="cuda") * 1e-2
                a.copy_(new)
                b.copy_(new)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in want:
            one(s, torch.full((1,), lr, device="cuda"))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for s, q in zip(want, got) for a, b in zip(state(s), state(q))), rep


@pytest.mark.gpu
def test_a_tensor_past_2_to_the_30_elements():
    n = (1 << 30) + 1000
    p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    total = state_offsets([n])[1]
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    places = [0, 1, 4095, 4096, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, n - 1]
    g[places] = 0.5
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    norm = adamw_step([p], [g], m, v, step, lr=0.25, weight_decay=0.0, max_grad_norm=100.0)
    assert abs(float(norm) - 0.5 * len(places) ** 0.5) < 1e-6
    assert bool((p[places] == 0.75).all()) and int((p != 1).sum()) == len(places)
    assert bool(((m[places] - 0.05).abs() < 1e-7).all()) and int((m != 0).sum()) == len(places) and int((v != 0).sum()) == len(places)


def _network(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 0.1).to(dtype) for s in ((27, 8, 16), (16,), (64, 3), (3,), (1,), (300, 257))]


@pytest.mark.gpu
@pytest.mark.parametrize("decoupled", [True, False])
def test_optimizer_follows_torch(decoupled):
    """Six steps with a schedule and two groups against torch.optim.AdamW / Adam in float64 on the CPU."""
    ref = [t.double().requires_grad_(True) for t in _network(0)]
    own = [t.cuda().requires_grad_(True) for t in _network(0)]
    kind = torch.optim.AdamW if decoupled else torch.optim.Adam
    o_ref = kind([{"params": ref[:4]}, {"params": ref[4:], "lr": 2e-3, "weight_decay": 0.0}], lr=1e-3, weight_decay=0.1, eps=1e-6)
    o_own = AdamW([{"params": own[:4]}, {"params": own[4:], "lr": 2e-3, "weight_decay": 0.0}], lr=1e-3, weight_decay=0.1, eps=1e-6, decoupled=decoupled)
    s_ref, s_own = (torch.optim.lr_scheduler.StepLR(o, step_size=2, gamma=0.5) for o in (o_ref, o_own))
    g = torch.Generator().manual_seed(1)
    for it in range(6):
        for a, b in zip(ref, own):
            grad = torch.randn(a.shape, generator=g) * 10.0 ** -(it % 3)
            a.grad, b.grad = grad.double(), grad.cuda()
        for o in (o_ref, o_own, s_ref, s_own):
            o.step()
        for a, b in zip(ref, own):
            # an update is at most ~ lr / (1 - b1) long and known to some 40 roundings (m cancels at most between steps of equal size: x 10)
            assert float((b.detach().cpu().double() - a.detach()).abs().max()) < (it + 1) * (2e-2 * 400 * U32 + 2 * U32)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,masters", [(32, False), (8, False), (32, True), (8, True)])
def test_optimizer_state_dict_and_clip_over_groups(bits, masters):
    dtype = torch.bfloat16 if masters else torch.float32

    def build():
        ps = [t.cuda().requires_grad_(True) for t in _network(2, dtype)] + [torch.full((10,), 0.3, device="cuda", requires_grad=True)]
        return ps, AdamW([{"params": ps[:3]}, {"params": ps[3:]}], lr=1e-3, state_bits=bits, master_weights=masters, max_grad_norm=0.5, seed=3)

    def grads(ps, it):
        g = torch.Generator().manual_seed(10 + it)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()

    ps, o = build()
    for it in range(3):
        grads(ps, it)
        o.step()
        ref = sum(float((p.grad.double() ** 2).sum()) for p in ps) ** 0.5
        assert abs(float(o.last_grad_norm) - ref) < 4 * U32 * ref         # over both groups and dtypes
    saved, weights = copy.deepcopy(o.state_dict()), [p.detach().clone() for p in ps]
    for it in range(3, 5):
        grads(ps, it)
        o.step()
    qs, o2 = build()
    with torch.no_grad():
        for q, w in zip(qs, weights):
            q.copy_(w)
    o2.load_state_dict(saved)
    for it in range(3, 5):
        grads(qs, it)
        o2.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for x, y in zip(o.state.values(), o2.state.values()) for a, b in
               zip([x["exp_avg"], x["exp_avg_sq"]], [y["exp_avg"], y["exp_avg_sq"]]))
    other = AdamW(qs, lr=1e-3, state_bits=40 - bits, master_weights=masters)
    with pytest.raises(ValueError):
        other.load_state_dict({"state": saved["state"], "param_groups": other.state_dict()["param_groups"]})


@pytest.mark.gpu
def test_pointwise_layers_train_with_the_optimizer():
    """Two linear() layers and the MOS loss, three steps with clip and decay, as they are used together: parameters and losses against the same
    program in float64 on the CPU; with moments in 8 bits within their rounding of the 32-bit run."""
    from insmos_amd.autograd import linear, mos_loss
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(3000, 24, generator=gen)
    labels = torch.randint(0, 3, (3000,), generator=gen)
    init = [torch.randn(24, 40, generator=gen) * 0.3, torch.randn(40, generator=gen) * 0.1, torch.randn(40, 3, generator=gen) * 0.3, torch.zeros(3)]
    kw = dict(lr=1e-2, weight_decay=0.01, eps=1e-3)

    def run(bits):
        ps = [t.cuda().requires_grad_(True) for t in init]
        opt = AdamW(ps, max_grad_norm=0.05, state_bits=bits, **kw)
        losses = []
        for _ in range(3):
            opt.zero_grad(set_to_none=True)
            h = linear(x.cuda(), ps[0], ps[1], activation="gelu_tanh")
            loss = mos_loss(linear(h, ps[2], ps[3]), labels.cuda())
            loss.backward()
            opt.step()
            losses.append(float(loss.detach()))
        return ps, losses

    ref = [t.double().requires_grad_(True) for t in init]
    opt = torch.optim.AdamW(ref, **kw)
    want = []
    w = torch.tensor([0.0, 0.5, 0.5], dtype=torch.float64)
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        lg = torch.nn.functional.gelu(x.double() @ ref[0] + ref[1], approximate="tanh") @ ref[2] + ref[3]
        lg = torch.cat([torch.full((len(lg), 1), -float("inf"), dtype=torch.float64), lg[:, 1:]], 1)     # the ignored class
        loss = torch.nn.functional.nll_loss(torch.log(torch.softmax(lg, 1).clamp(min=1e-8)), labels, weight=w)
        loss.backward()
        torch.nn.utils.clip_grad_norm_(ref, 0.05)
        opt.step()
        want.append(float(loss.detach()))
    ps, losses = run(32)
    # eps = 1e-3 bounds an update's sensitivity: lr / eps * (a gradient's error of about 1e-6 of the norm 0.05) = 5e-7 a step, and fp32's rounding
    for a, b in zip(ps, ref):
        assert float((a.detach().cpu().double() - b.detach()).abs().max()) < 1e-5
    assert max(abs(a - b) for a, b in zip(losses, want)) < 1e-5
    ps8, losses8 = run(8)
    # codes are 1/8 of their value apart at most (sqrt(v) too): an update of at most 3 lr moves by less than 3 lr * 2 / 8 in each step behind the first
    for a, b in zip(ps8, ps):
        assert float((a.detach() - b.detach()).abs().max()) < 2 * 3e-2 * 0.25
    assert losses8[0] == losses[0]


@pytest.mark.gpu
def test_trainer_makes_its_optimizer():
    from insmos_amd import params as P
    from insmos_amd.train_unet import InsMOSTrainer
    cfg = P.default_cfg()
    tr = InsMOSTrainer(cfg, P.random_state_dict(cfg, 0))
    ref = [p.detach().cpu().double().requires_grad_(True) for p in tr.params.values()]
    o_ref = torch.optim.Adam(ref, lr=float(cfg["TRAIN"]["LR"]), weight_decay=float(cfg["TRAIN"]["WEIGHT_DECAY"]))
    opt = tr.make_optimizer()
    for p, q in zip(tr.params.values(), ref):
        g = torch.randn(p.shape, device="cuda")
        p.grad, q.grad = g, g.cpu().double()
    opt.step()
    o_ref.step()
    for p, q in zip(tr.params.values(), ref):   # one step: lr (1 + a few roundings), p's rounding
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) < 1e-4 * 40 * U32 + 2 * U32 * (1 + float(q.detach().abs().max()))
    assert tr.make_optimizer(state_bits=8, decoupled=True, lr=1e-3).param_groups[0]["lr"] == 1e-3


def _cpu_args(n=2):
    ps, gs = [torch.zeros(10) for _ in range(n)], [torch.zeros(10) for _ in range(n)]
    total = state_offsets([10] * n)[1]
    return ps, gs, torch.zeros(total), torch.zeros(total), torch.zeros(1, dtype=torch.int32)


def test_step_refusals():
    ps, gs, m, v, step = _cpu_args()
    x = torch.zeros(20)
    for text, args, kw in (("on the GPU", (ps, gs, m, v, step), {}), ("parameters and", (ps, gs[:1], m, v, step), {}), ("no parameters", ([], [], m, v, step), {}),
                           ("betas", (ps, gs, m, v, step), {"betas": (1.0, 0.9)}), ("betas", (ps, gs, m, v, step), {"betas": (0.9, -0.1)}),
                           ("eps", (ps, gs, m, v, step), {"eps": -1e-8}), ("eps", (ps, gs, m, v, step), {"weight_decay": float("nan")}),
                           ("max_grad_norm", (ps, gs, m, v, step), {"max_grad_norm": 0.0}), ("max_grad_norm", (ps, gs, m, v, step), {"max_grad_norm": float("nan")}),
                           ("float32, bfloat16 or float16", ([p.double() for p in ps], [g.double() for g in gs], m, v, step), {}),
                           ("parameter 1 is", ([ps[0], ps[1].half()], [gs[0], gs[1].half()], m, v, step), {}),
                           ("gradient 1 is", (ps, [gs[0], gs[1].half()], m, v, step), {}), ("another shape", (ps, [gs[0], torch.zeros(2, 5)], m, v, step), {}),
                           ("gaps", ([ps[0], torch.zeros(10, 2)[:, 0]], gs, m, v, step), {}), ("share memory", ([ps[0], ps[0]], gs, m, v, step), {}),
                           ("share memory", ([x[:10], x[5:15]], gs, m, v, step), {}), ("sparse", (ps, [gs[0], gs[1].to_sparse()], m, v, step), {}),
                           ("no tensor", ([ps[0], 3], gs, m, v, step), {})):
        with pytest.raises(ValueError, match=text):
            adamw_step(*args, lr=1e-3, **kw)
    with pytest.raises(ValueError, match="no gradients"):
        grad_norm([None])
    with pytest.raises(ValueError, match="on the GPU"):
        grad_norm([torch.zeros(3)])
    for bad in ({"state_bits": 16}, {"lr": -1.0}, {"lr": float("inf")}, {"max_grad_norm": -1.0}):
        with pytest.raises(ValueError):
            AdamW(ps, **bad)


def test_the_table_of_a_list():
    """What the step is given: entries in order with their place in the state, None gradients left out, reordered gradients named."""
    from insmos_amd import _host
    ps = [torch.zeros(300), torch.zeros(5, 4), torch.zeros(0), torch.zeros(4, 6).t()]
    gs = [torch.zeros(300), None, torch.zeros(0), torch.zeros(6, 4)]
    buf = bytearray(32 * 4)
    assert _host.opt_table("x", ps, gs, buf, True) == (3, 0, 1024, [3])
    rows = np.frombuffer(buf, np.int64).reshape(4, 4)
    assert rows[0].tolist() == [ps[0].data_ptr(), gs[0].data_ptr(), 300, 0] and rows[2, 2:].tolist() == [24, 768]
    assert state_offsets([300, 20, 0, 24]) == ([0, 512, 768, 768], 1024)
    with pytest.raises(ValueError, match="too short"):
        _host.opt_table("x", ps, gs, bytearray(32), True)


def test_entry_points_refuse():
    """The C entries return their codes before any launch (none of these calls reaches the device)."""
    lib = _lib.load()
    buf = (ctypes.c_char * 65536)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def table(*rows):
        t = np.array(rows, np.int64).reshape(-1, 4)
        return t, t.ctypes.data

    def step(rows=((p, p, 100, 0),), dtype=0, bits=32, m=p, v=p, scales=None, n=256, w=None, st=p, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, norm=0.0, ws=p, ws_bytes=65536):
        t, at = table(*rows)
        return lib.insmos_adamw_step(at, len(t), dtype, bits, m, v, scales, n, w, st, 1e-3, None, b1, b2, eps, wd, 1, norm, None, 0, 0, None, ws, ws_bytes, None)

    for bad in ({"dtype": 3}, {"bits": 16}, {"m": None}, {"v": None}, {"bits": 8}, {"n": 255}, {"n": 0}, {"w": p}, {"st": None}, {"ws": None}, {"m": p + 4}, {"ws": p + 8},
                {"b1": 1.0}, {"b2": -0.5}, {"eps": -1.0}, {"eps": float("nan")}, {"wd": -1.0}, {"norm": float("nan")}, {"rows": ((0, p, 100, 0),)}, {"rows": ((p, 0, 100, 0),)},
                {"rows": ((p + 2, p, 100, 0),)}, {"rows": ((p, p + 1, 100, 0),)}, {"rows": ((p, p, -1, 0),)}, {"rows": ((p, p, 100, 128),)}, {"rows": ((p, p, 100, 256),)},
                {"rows": ((p, p, 257, 0),)}, {"rows": ((p, p, 100, -256),)}, {"rows": ((p, p, 100, 0), (p, 0, 5, 0))}):
        assert step(**bad) == -1, bad
    assert step(ws_bytes=8, norm=1.0) == -3
    t, at = table((0, p, 20000, 0))
    assert lib.insmos_grad_sumsq_partials(at, 1) == 3
    assert lib.insmos_grad_sumsq(at, 1, 0, p, 2, None) == -3 and lib.insmos_grad_sumsq(at, 1, 0, None, 3, None) == -1 and lib.insmos_grad_sumsq(at, 1, 9, p, 3, None) == -1
    assert lib.insmos_grad_norm(None, 1, p, None) == -1 and lib.insmos_grad_norm(p, 1, None, None) == -1


@pytest.mark.gpu
def test_a_norm_beyond_float32_is_not_finite():
    """Two gradients of 3e38: their norm, 4.2e38, is above float32's largest number (3.4e38), so norm_out says inf and the step is left out."""
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        g = torch.zeros(600, device="cuda")
        g[:2] = 3e38
        m, v = (torch.zeros(768, device="cuda").to(torch.float32 if bits == 32 else torch.float8_e4m3fn) for _ in range(2))
        step = torch.zeros(1, dtype=torch.int32, device="cuda")
        norm = adamw_step([p], [g], m, v, step, lr=0.1, skip_nonfinite=True, scales=None if bits == 32 else torch.zeros(2, 3, device="cuda"))
        assert norm.item() == float("inf") and step.item() == 0 and torch.equal(p, torch.ones_like(p))
        g[1] = 0.0
        assert adamw_step([p], [g], m, v, step, lr=0.1, skip_nonfinite=True, max_grad_norm=1.0,
                          scales=None if bits == 32 else torch.zeros(2, 3, device="cuda")).item() == torch.tensor(3e38).item()
        assert step.item() == 1 and p[0].item() != 1.0


@pytest.mark.gpu
def test_moments_in_one_buffer_are_refused():
    p, g, m = (torch.ones(300, device="cuda") for _ in range(3))
    buf, step = torch.zeros(1024, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for a, b in ((buf[:512], buf[:512]), (buf[:512], buf[256:768]), (buf[256:768], buf[:512])):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step([p], [g], a, b, step, lr=0.1)
    adamw_step([p], [g], buf[:512], buf[512:], step, lr=0.1)
    assert step.item() == 1


@pytest.mark.gpu
def test_optimizer_refuses_changed_parameters_and_a_captured_first_step():
    p = torch.nn.Parameter(torch.randn(4, 8, 3, 3, device="cuda"))
    p.grad = torch.randn_like(p)
    o = AdamW([p], lr=0.1)
    said, stream = None, torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        try:
            o.step()
        except RuntimeError as e:
            said = str(e)
    assert "captured" in said and not o.state
    o.step()
    p.data = p.data.to(memory_format=torch.channels_last)
    with pytest.raises(RuntimeError, match="order in memory"):
        o.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_copies_and_pickles(bits):
    """A copy (deepcopy, pickle) with its parameters goes on as the original does, and its state entries are views of its own buffers."""
    import copy
    import pickle
    gen = torch.Generator().manual_seed(5)
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).cuda()) for s in ((7, 5), (300,), (3, 4, 2))]
    o = AdamW(ps, lr=0.01, state_bits=bits, max_grad_norm=1.0, seed=9)
    gs = [[torch.randn(p.shape, generator=gen).cuda() for p in ps] for _ in range(4)]

    def go(opt, its):
        for it in its:
            for p, g in zip(opt.param_groups[0]["params"], gs[it]):
                p.grad = g.clone()
            opt.step()
        return [p.detach().clone() for p in opt.param_groups[0]["params"]]

    go(o, range(2))
    copies = [copy.deepcopy(o), pickle.loads(pickle.dumps(o))]
    want = go(o, range(2, 4))
    for c in copies:
        assert all(torch.equal(a, b) for a, b in zip(go(c, range(2, 4)), want))
        for p, q in zip(c.param_groups[0]["params"], ps):
            assert all(torch.equal(c.state[p][k].float(), o.state[q][k].float()) for k in o.state[q])


@pytest.mark.gpu
def test_negated_views_are_refused_and_inference_tensors_taken():
    neg = torch.conj(torch.ones(300, dtype=torch.complex64, device="cuda")).imag
    m, v, step = torch.zeros(512, device="cuda"), torch.zeros(512, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert neg.is_neg()
    with pytest.raises(ValueError, match="negated"):
        adamw_step([torch.ones(300, device="cuda")], [neg], m, v, step, lr=0.1)
    with torch.inference_mode():
        p = torch.ones(300, device="cuda")
    assert step.item() == 0 and not bool(m.any())
    adamw_step([p], [torch.ones(300, device="cuda")], m, v, step, lr=0.25, weight_decay=0.0, eps=0.0)   # (m / sqrt(v) = 1 in the first step)
    assert step.item() == 1 and bool(((p - 0.75).abs() < 1e-6).all())
