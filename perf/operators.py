"""What the framework's optimiser step and pointwise layer cost: their cases, inputs, plain forms and definitions in 64 bits.

Two operators:

  linear   y = act(x W + b [+ r]) [+ r], forward alone or with its gradients (insmos_amd.autograd.linear)
  adamw    one AdamW / Adam step over a list of tensors, moments in 32 or in 8 bits, optionally with the clip by the gradients'
           global norm (insmos_amd.optim.adamw_step)

The moments of `adamw` lie in flat buffers: tensor i starts at 256 * sum_{j<i} ceil(numel_j / 256).  In 8 bits they are e4m3 codes of m
and of s = sqrt(v), each in units of an fp32 scale per 256 elements (largest / 448), rounded up or down by 16 bits of a hash of the
element's position, the step and the seed.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"
BLOCK = 256
BETAS, EPS = (0.9, 0.999), 1e-8


# ---------------------------------------------------------------------------------------------------------------------- cases
def _linear(name, m, k, n, dtype, act="none", bias=True, residual="none", layout="in_out", pad=0, train=False):
    return dict({"op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual,
                 "layout": layout, "pad": pad, "train": train}, **({"name": name} if name else {}))


def _adamw(name, tensors, elements, dtype, bits, masters=False, decoupled=True, clip=False):
    return dict({"op": "adamw", "tensors": tensors, "elements": elements, "dtype": dtype, "bits": bits, "masters": masters,
                 "decoupled": decoupled, "clip": clip}, **({"name": name} if name else {}))


def listed():
    return [
        # one token of a served model through a wide layer: the weights' bytes are everything
        _linear("one token bf16", 1, 2048, 8192, "bf16", act="silu"),
        # a handful of rows and odd widths, weights as nn.Linear keeps them (cout, cin)
        _linear("few rows odd fp16", 13, 1001, 2057, "fp16", act="gelu", residual="after", layout="out_in"),
        # a 1x1 layer over the points of one scan (119 817 of them), residual block form, rows of a wider matrix
        _linear("points train fp32", 119817, 64, 128, "fp32", act="relu", residual="first", pad=32, train=True),
        # many rows served at once: the matrix units are the bound
        _linear("rows forward bf16", 8192, 4096, 8192, "bf16", act="gelu_tanh", residual="after"),
        # a training step of the wide layer
        _linear("rows train bf16", 8192, 2048, 8192, "bf16", act="silu", train=True),
        # ragged: no size is a multiple of a tile, one is odd
        _linear("ragged train fp16", 4099, 1000, 1533, "fp16", act="gelu", residual="after", layout="out_in", train=True),
        # a head's few vectors: latency
        _adamw("few tensors fp32", 8, 20000, "fp32", 32),
        # the size and tensor count of this framework's network, Adam as it trains (weight decay in the gradient), clipped
        _adamw("network fp32", 250, 6500000, "fp32", 32, decoupled=False, clip=True),
        # the same with moments in 8 bits
        _adamw("network 8 bits", 250, 6500000, "fp32", 8, clip=True),
        # a large model in bf16 with fp32 master weights, clipped
        _adamw("large bf16 masters", 90, 120000007, "bf16", 32, masters=True, clip=True),
        # a large model in bf16, moments in 8 bits: the smallest footprint
        _adamw("large bf16 8 bits", 90, 200000011, "bf16", 8),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        dtype, train = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5
        m, k, n = _between(rng, 1, 131072), _between(rng, 8, 8192), _between(rng, 8, 8192)
        if rng.random() < 0.5:   # widths as most layers have them
            k, n = max(8, k // 8 * 8), max(8, n // 8 * 8)
        most = 8e11 if dtype != "fp32" else 1e11
        per_row = (6 if train else 2) * k * n + 2000 * (k + n)
        m = max(1, min(m, int(most / per_row)))
        return _linear(None, m, k, n, dtype, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.75,
                       residual=rng.choice(["none", "first", "after"]), layout=rng.choice(["in_out", "out_in"]),
                       pad=rng.choice([0, 0, 8, 5]), train=train)
    dtype, bits = rng.choice(["fp32", "bf16", "fp16"]), rng.choice([32, 8])
    return _adamw(None, _between(rng, 1, 400), _between(rng, 2000, 100000000), dtype, bits,
                  masters=dtype != "fp32" and rng.random() < 0.5, decoupled=rng.random() < 0.7, clip=rng.random() < 0.5)


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        r = case["residual"] != "none"
        values = m * k + k * n + m * n * (1 + r) + (n if case["bias"] else 0)
        if case["train"]:
            values += m * n + m * k + k * n + (m * n if r else 0) + (n if case["bias"] else 0)
        return {"bytes": values * size, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    n = case["elements"]
    state = 16 * n if case["bits"] == 32 else 4 * n + 16 * (n // BLOCK)
    params = (2 if case["masters"] else 3) * size * n + (8 * n if case["masters"] else 0)
    return {"bytes": state + params, "flops": 16 * n}


# --------------------------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    """Sizes of the tensors: weights of very different sizes among small vectors, as in a network; their sum is `elements`."""
    t, total = case["tensors"], case["elements"]
    share = [((i * 7919 + 13) % 97 + 1) ** 2 if i % 3 == 0 else 0.02 * ((i * 31) % 17 + 1) for i in range(t)]
    unit = total / sum(share)
    sizes = [max(1, int(s * unit)) for s in share]
    big = sizes.index(max(sizes))
    sizes[big] = max(1, sizes[big] + total - sum(sizes))
    return sizes


def _lay(sizes):
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = normal(m, k + case["pad"])
        x *= torch.exp(0.5 * normal(1, k + case["pad"]))   # some channels are much larger than others
        w = normal(k, n) / math.sqrt(k) if case["layout"] == "in_out" else (normal(n, k) / math.sqrt(k))
        s = {"case": case, "x": x.to(dtype)[:, :k], "w": w.to(dtype) if case["layout"] == "in_out" else w.to(dtype).t(),
             "b": (0.1 * normal(n)).to(dtype) if case["bias"] else None,
             "r": normal(m, n).to(dtype) if case["residual"] != "none" else None,
             "dy": (0.05 * normal(m, n)).to(dtype) if case["train"] else None}
        if case["train"]:
            for name in ("x", "w", "b", "r"):
                if s[name] is not None:
                    s[name] = s[name].detach().requires_grad_(True)
        return s
    sizes = _sizes(case)
    starts, total = _lay(sizes)
    lay = [(a, n) for a, n in zip(starts, sizes)]
    # storage of the parameters and gradients: one buffer each, of which every tensor is a slice (aligned as an allocator aligns)
    params, grads = torch.zeros(total, device=DEV, dtype=dtype), torch.zeros(total, device=DEV, dtype=dtype)
    spread = torch.exp(1.5 * normal(total // BLOCK)).repeat_interleave(BLOCK)
    g32 = 1e-3 * spread * normal(total)
    g32 = torch.where(torch.rand(total, generator=g, device=DEV) < 0.05, torch.zeros_like(g32), g32)   # rows that no sample touched
    p32 = 0.05 * normal(total)
    avg, rms = 3e-4 * spread * normal(total), 1e-3 * spread * (0.3 + normal(total).abs())
    inside = torch.cat([(torch.arange(-(-n // BLOCK) * BLOCK, device=DEV) < n) for n in sizes]).float()
    params.copy_(p32 * inside)
    grads.copy_(g32 * inside)
    avg, rms, p32 = avg * inside, rms * inside, p32 * inside
    s = {"case": case, "flat": params, "params": [params[a:a + n] for a, n in lay], "grads": [grads[a:a + n] for a, n in lay],
         "step": torch.full((1,), 41, dtype=torch.int32, device=DEV), "masters": p32 if case["masters"] else None, "scales": None,
         "hyper": {"lr": 2e-4, "betas": BETAS, "eps": EPS, "weight_decay": 0.01, "decoupled": case["decoupled"],
                   "max_grad_norm": 1.0 if case["clip"] else None, "seed": 1234}}
    if case["bits"] == 32:
        s["m"], s["v"] = avg, rms * rms
    else:
        top = [t.view(-1, BLOCK).abs().amax(1, keepdim=True).clamp_min(2.0 ** -126) / 448 for t in (avg, rms)]
        s["m"] = (avg.view(-1, BLOCK) / top[0]).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)
        s["v"] = (rms.view(-1, BLOCK) / top[1]).clamp(0, 448).to(torch.float8_e4m3fn).view(-1)
        s["scales"] = torch.stack([top[0].view(-1), top[1].view(-1)])
    return s


# -------------------------------------------------------------------------------------------------------------- the plain forms
def _act(z, act):
    if act == "relu":
        return torch.clamp_min(z, 0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


def _linear_formula(s, wide):
    """The layer and its gradients with every intermediate in `wide`."""
    c = s["case"]
    x, w = s["x"].detach().to(wide), s["w"].detach().to(wide)
    r = s["r"].detach().to(wide) if s["r"] is not None else None
    z = x @ w
    if s["b"] is not None:
        z = z + s["b"].detach().to(wide)
    if c["residual"] == "first":
        z = z + r
    y = _act(z, c["act"])
    if c["residual"] == "after":
        y = y + r
    out = {"y": y}
    if c["train"]:
        dy = s["dy"].to(wide)
        dz = dy * _act_slope(z, c["act"])
        out["dx"], out["dw"] = dz @ w.t(), x.t() @ dz
        if s["b"] is not None:
            out["db"] = dz.sum(0)
        if r is not None:
            out["dr"] = dz if c["residual"] == "first" else dy
    return out


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits16(n, step, seed, device):
    """Two times 16 random bits for each of n positions at a step (int32 device tensor), as integers."""
    key = _mix(_mix(step.to(torch.int64)) ^ (seed & 0xFFFFFFFF))
    pos = torch.arange(n, device=device)
    h = _mix(((pos & 0xFFFFFFFF) + (pos >> 32) * 0x9E3779B1 + key) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def _codes(x, u, keep):
    """e4m3 codes of the rows of x (blocks of 256, fp32) in units of their scale, rounded by the 16 bits u; (codes, scales).
    keep: what is not zero does not become zero."""
    a = x.abs()
    fine = a <= 3.4028234663852886e38
    scale = (torch.where(fine, a, torch.zeros_like(a)).amax(1, keepdim=True) * (1.0 / 448)).clamp_min(2.0 ** -126)
    y = (a * (1.0 / scale)).clamp_max(448.0)
    # e4m3's smallest normal number 2^-6 taken to fp32's 2^-126: exponent and three bits of the mantissa then are the code
    bits = (y * 2.0 ** -120).view(torch.int32).to(torch.int64)
    code = (bits + (u << 4)) >> 20
    if keep:
        code = torch.where((a > 0) & (code == 0), torch.ones_like(code), code)
    code = torch.where(fine, code, torch.full_like(code, 0x7F)) | torch.where(torch.signbit(x), 0x80, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _adamw_plain(s):
    c, h = s["case"], s["hyper"]
    (b1, b2), lr, wd = h["betas"], h["lr"], h["weight_decay"]
    sizes = [t.numel() for t in s["params"]]
    rounded = [-(-n // BLOCK) * BLOCK for n in sizes]

    def flat(ts):
        return torch.cat([torch.nn.functional.pad(t.float(), (0, r - n)) for t, n, r in zip(ts, sizes, rounded)])

    g, p = flat(s["grads"]), s["masters"] if s["masters"] is not None else flat(s["params"])
    s["step"] += 1
    t = s["step"].double()
    size = torch.tensor(lr, dtype=torch.float64, device=g.device) / (1 - torch.pow(torch.tensor(b1, dtype=torch.float64, device=g.device), t))
    root = 1 / torch.sqrt(1 - torch.pow(torch.tensor(b2, dtype=torch.float64, device=g.device), t))
    norm = None
    if h["max_grad_norm"] is not None:
        norm = torch.sqrt(g.double().square().sum())
        g = g * torch.clamp_max(h["max_grad_norm"] / (norm + 1e-6), 1.0).float()
    if not c["decoupled"]:
        g = g + wd * p
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["scales"][0][:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["scales"][1][:, None]).view(-1)
        v = v * v
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    root_v = torch.sqrt(v)
    p = p * ((1 - lr * wd) if c["decoupled"] else 1.0) - size.float() * (m / (root_v * root.float() + EPS))
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        u = _bits16(g.numel(), s["step"], h["seed"], g.device)
        for k, (name, x) in enumerate((("m", m), ("v", root_v))):
            codes, scale = _codes(x.view(-1, BLOCK), u[k].view(-1, BLOCK), keep=name == "v")
            s[name].copy_(codes.view(-1))
            s["scales"][k].copy_(scale.view(-1))
    if s["masters"] is not None:
        s["masters"].copy_(p)
    [t.copy_(q[:n]) for t, q, n in zip(s["params"], p.split(rounded), sizes)]
    return _adamw_outputs(s, norm.float() if norm is not None else None)


def _adamw_outputs(s, norm):
    out = {"params": s["flat"], "m": s["m"], "v": s["v"], "step": s["step"]}
    for name, t in (("scales", s["scales"]), ("masters", s["masters"]), ("norm", norm)):
        if t is not None:
            out[name] = t
    return out


def run(s):
    c = s["case"]
    if c["op"] == "linear":
        if own:
            from insmos_amd.autograd import linear
            act, first = None if c["act"] == "none" else c["act"], c["residual"] == "first"
            if not c["train"]:
                with torch.no_grad():
                    return {"y": linear(s["x"], s["w"], s["b"], s["r"], activation=act, residual_first=first)}
            y = linear(s["x"], s["w"], s["b"], s["r"], activation=act, residual_first=first)
            names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
            grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
            return dict({"d" + n: t for n, t in zip(names, grads)}, y=y)
        return {name: t.to(s["x"].dtype) for name, t in _linear_formula(s, torch.float32).items()}
    if own:
        from insmos_amd.optim import adamw_step
        norm = adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], scales=s["scales"], masters=s["masters"], **s["hyper"])
        return _adamw_outputs(s, norm if c["clip"] else None)
    return _adamw_plain(s)


# ------------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_linear(s):
    c = s["case"]
    x, w = s["x"].detach().double(), s["w"].detach().double()
    pre = torch.zeros(c["m"], c["n"], dtype=torch.float64, device=x.device)
    if s["b"] is not None:
        pre += s["b"].detach().double()[None, :]
    if c["residual"] == "first":
        pre += s["r"].detach().double()
    pre = torch.addmm(pre, x, w).requires_grad_(c["train"])
    post = {"none": lambda v: v * 1.0, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu,
            "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[c["act"]](pre)
    out = {"y": (post + s["r"].detach().double() if c["residual"] == "after" else post).detach()}
    if c["train"]:
        dy = s["dy"].double()
        (d,) = torch.autograd.grad(post, pre, dy)
        out["dx"] = torch.mm(d, w.t())
        out["dw"] = torch.mm(x.t(), d)
        if s["b"] is not None:
            out["db"] = torch.mv(d.t(), torch.ones(c["m"], dtype=torch.float64, device=x.device))
        if s["r"] is not None:
            out["dr"] = d if c["residual"] == "first" else dy
    return out


def _exact_codes(x, u, keep):
    a = x.abs()
    scale = torch.clamp_min(a.max(dim=1).values / 448, 2.0 ** -126)
    y = torch.clamp_max(a / scale[:, None], 448)
    # the distance of neighbouring e4m3 numbers around y: an eighth of the power of two below it, at least 2^-9
    gap = torch.exp2(torch.floor(torch.log2(torch.clamp_min(y, 2.0 ** -6))) - 3)
    q = torch.floor(y / gap + u.double() / 65536) * gap
    q = torch.clamp_max(q, 448)
    if keep:
        q = torch.where((a > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return q * torch.sign(x), scale


def _exact_adamw(s):
    c, h = s["case"], s["hyper"]
    (b1, b2), lr, wd = h["betas"], h["lr"], h["weight_decay"]
    t = int(s["step"].item()) + 1
    starts, total = _lay([q.numel() for q in s["params"]])
    g, p = (torch.zeros(total, dtype=torch.float64, device=DEV) for _ in range(2))
    for at, q, d in zip(starts, s["params"], s["grads"]):
        g[at:at + q.numel()] = d.double()
        p[at:at + q.numel()] = q.double()
    if s["masters"] is not None:
        p = s["masters"].double()
    out = {"step": s["step"] + 1}
    if h["max_grad_norm"] is not None:
        norm = float(torch.dot(g, g)) ** 0.5
        g *= min(1.0, h["max_grad_norm"] / (norm + 1e-6))
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
    if not c["decoupled"]:
        g += wd * p
    if c["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        each = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        m, v = s["m"].to(torch.float32).double() * each[0], (s["v"].to(torch.float32).double() * each[1]) ** 2
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    update = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    p = (p - lr * wd * p if c["decoupled"] else p) - lr * update
    # (the padding between tensors keeps its zeros: m = v = 0 there, and 0 / eps = 0)
    out["params"] = p
    if s["masters"] is not None:
        out["masters"] = p
    if c["bits"] == 32:
        out["m"], out["v"] = m, v
    else:
        u = _bits16(total, s["step"] + 1, h["seed"], g.device)
        both = [_exact_codes(x.view(-1, BLOCK), u[k].view(-1, BLOCK), k == 1) for k, x in enumerate((m, torch.sqrt(v)))]
        out["m"], out["v"] = both[0][0].view(-1), both[1][0].view(-1)
        out["scales"] = torch.stack([both[0][1], both[1][1]])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_linear(s) if case["op"] == "linear" else _exact_adamw(s)
