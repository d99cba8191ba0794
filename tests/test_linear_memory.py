"""What insmos_amd.autograd.linear allocates and keeps."""
import pytest
import torch

from insmos_amd import _lib
from insmos_amd.autograd import linear

F32, BF16, F16 = 0, 1, 2
A = 1 << 20      # an address on 16 bytes (none of these calls reads it)


def test_workspace_is_counted_for_the_call():
    """A copy for the operands that need one and for no other, parts of k where the call has them, nothing for few rows; never more than what is
    reserved for any operands of these sizes."""
    lib = _lib.load()

    def need(m, k, n, dt, x=A, ldx=None, w=A, ldw=None, out_in=0):
        got = lib.insmos_linear_ws_bytes_for(x, ldx or k, w, ldw or (k if out_in else n), out_in, m, k, n, dt)
        assert got <= lib.insmos_linear_ws_bytes(m, k, n, dt)
        return got

    pad = lambda b: (b + 255) // 256 * 256                                  # noqa: E731
    for dt in (F32, BF16, F16):
        assert need(1, 1024, 8192, dt) == need(8192, 4096, 8192, dt) == need(1000000, 256, 1024, dt) == 0
        assert need(0, 8, 8, dt) == 0
    assert lib.insmos_linear_ws_bytes(1000000, 256, 1024, F32) == 0         # fp32 is read as it lies, at any address and pitch
    assert lib.insmos_linear_ws_bytes(1, 2048, 8192, BF16) == 0             # few rows: so is everything
    m, k, n = 8192, 4096, 8192
    x_copy, w_copy = pad(m * k * 2), pad(k * n * 2)
    assert need(m, k, n, BF16, x=A + 2) == x_copy == need(m, k, n, BF16, ldx=k + 1)
    assert need(m, k, n, BF16, w=A + 2) == w_copy == need(m, k, n, F16, ldw=k + 3, out_in=1)
    assert lib.insmos_linear_ws_bytes(m, k, n, BF16) == x_copy + w_copy
    assert need(300, 8192, 64, BF16) > 0 and need(300, 8192, 64, BF16) % (pad(300 * 64 * 4)) == 0   # parts of k

    def back(m, k, n, dt, kind=0, dy=A, lddy=None, x=A, ldx=None, w=A, ldw=None, out_in=0, dx=1, dw=1, db=1, dz=0):
        got = lib.insmos_linear_backward_ws_bytes_for(dy, lddy or n, kind, x, ldx or k, w, ldw or (k if out_in else n), out_in, m, k, n, dt, dx, dw, db, dz)
        assert got <= lib.insmos_linear_backward_ws_bytes(m, k, n, dt)
        return got

    m, k, n = 8192, 2048, 8192
    dz = pad(m * n * 2)
    plain = back(m, k, n, BF16)                                             # sums and parts
    assert plain < dz
    assert back(m, k, n, BF16, kind=2) == plain + dz and back(m, k, n, BF16, kind=2, dz=1) == plain
    assert back(m, k, n, BF16, lddy=n + 1) == plain + dz                    # dy that cannot be loaded becomes dz
    assert back(m, k, n, BF16, x=A + 2) == plain + pad(m * k * 2) and back(m, k, n, BF16, w=A + 2) == plain + pad(k * n * 2)
    assert back(m, k, n, BF16, x=A + 2, dw=0) <= plain and back(m, k, n, BF16, w=A + 2, dx=0) <= plain
    assert back(m, k, n, BF16, dx=0, dw=0, db=0, kind=2, dz=1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,k,n", [(torch.bfloat16, 1, 4096, 8192), (torch.bfloat16, 4096, 4096, 4096), (torch.float32, 200000, 64, 128)])
def test_a_call_allocates_its_result_alone(dtype, m, k, n):
    x, w = torch.ones(m, k, dtype=dtype, device="cuda"), torch.ones(k, n, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = linear(x, w)
    torch.cuda.synchronize()
    # (torch takes memory in whole 2 MiB and splits no rest of 1 MiB or less off: 200 000 x 128 fp32 values, 102 400 000 bytes, count as 49 x 2 MiB,
    # 360 448 more)
    assert torch.cuda.max_memory_allocated() - before <= y.numel() * y.element_size() + (1 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("m,k,n", [(3, 40, 24), (300, 130, 72), (300, 4100, 66), (5000, 64, 130)])
def test_the_reserve_for_any_operands_is_enough(dtype, m, k, n):
    """The C entries with a workspace of insmos_linear*_ws_bytes for operands at odd addresses and pitches, in either weight layout; one byte less
    than the call's own count is refused before anything is written."""
    lib, t = _lib.load(), getattr(torch, dtype)
    code = {"float32": F32, "bfloat16": BF16, "float16": F16}[dtype]
    gen = torch.Generator().manual_seed(m + n)
    whole = lambda r, c: torch.randint(-2, 3, (r, c), generator=gen).to(t).cuda()   # noqa: E731
    st = torch.cuda.current_stream().cuda_stream
    for out_in in (0, 1):
        for off, pad in ((0, 0), (1, 1)):
            wr, wc = (n, k) if out_in else (k, n)
            hold = [torch.cat([torch.zeros(off, dtype=t, device="cuda"), whole(r, c + pad).flatten()]) for r, c in ((m, k), (wr, wc), (m, n))]
            x, w, dy = (h[off:].view(r, c + pad)[:, :c] for h, (r, c) in zip(hold, ((m, k), (wr, wc), (m, n))))
            y, dx, dw, db = (torch.full(s, 7.0, dtype=t, device="cuda") for s in ((m, n), (m, k), (wr, wc), (n,)))
            args = (x.data_ptr(), k + pad, w.data_ptr(), wc + pad, out_in)
            exact = lib.insmos_linear_ws_bytes_for(*args, m, k, n, code)
            for size in ([exact - 1] if exact else []) + [exact, lib.insmos_linear_ws_bytes(m, k, n, code)]:
                ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
                rc = lib.insmos_linear(*args, None, None, 0, 0, 0, m, k, n, code, y.data_ptr(), n, None, 0, ws.data_ptr(), size, st)
                assert rc == (-3 if size < exact else 0)
                z = x.double() @ (w.double().t() if out_in else w.double())
                assert bool((y == 7).all()) if size < exact else torch.equal(y, z.to(t))     # (whole numbers: exact sums)
            back = (dy.data_ptr(), n + pad, None, 0, 0, *args)
            exact = lib.insmos_linear_backward_ws_bytes_for(dy.data_ptr(), n + pad, 0, *args, m, k, n, code, 1, 1, 1, 0)
            for size in ([exact - 1] if exact else []) + [exact, lib.insmos_linear_backward_ws_bytes(m, k, n, code)]:
                ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
                rc = lib.insmos_linear_backward(*back, m, k, n, code, dx.data_ptr(), k, dw.data_ptr(), wc, db.data_ptr(), None, 0, ws.data_ptr(), size, st)
                assert rc == (-3 if size < exact else 0)
                X, W, D = x.double(), w.double(), dy.double()
                want = (D @ (W if out_in else W.t()), D.t() @ X if out_in else X.t() @ D, D.sum(0))
                for g, r in zip((dx, dw, db), want):
                    assert bool((g == 7).all()) if size < exact else torch.equal(g, r.to(t))


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("out_in", [False, True])
def test_the_tape_keeps_what_the_needed_gradients_read(act, out_in):
    """x for the weight's gradient, the weight for x's, slopes (relu: y) for any; the gradients are those of the whole set."""
    gen = torch.Generator().manual_seed(2)
    x, b, r, dy = (torch.randn(s, generator=gen).cuda() for s in ((40, 24), (16,), (40, 16), (40, 16)))
    w = torch.randn(16, 24, generator=gen).cuda().t() if out_in else torch.randn(24, 16, generator=gen).cuda()

    def run(needed):
        kept, ins = [], [t.detach().requires_grad_(i in needed) for i, t in enumerate((x, w, b, r))]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t.data_ptr()), t)[1], lambda t: t):
            y = linear(*ins, activation=act, residual_first=True)
        grads = torch.autograd.grad(y, [ins[i] for i in needed], dy)
        return kept, dict(zip(needed, grads)), [t.stride() for t in grads]

    _, want, _ = run((0, 1, 2, 3))
    for needed in ((0,), (1,), (2,), (3,), (0, 2), (1, 3), (0, 1)):
        kept, got, strides = run(needed)
        assert (x.data_ptr() in kept) == (1 in needed) and (w.data_ptr() in kept) == (0 in needed)
        assert len(kept) == (0 in needed) + (1 in needed) + (act is not None)
        assert all(torch.equal(got[i], want[i]) for i in needed)
        if 1 in needed:
            assert got[1].stride() == w.stride()


@pytest.mark.gpu
def test_the_profiler_sees_the_layer_and_the_optimiser():
    import ctypes

    from insmos_amd.optim import AdamW
    lib = _lib.load()
    x, w = torch.randn(300, 40, device="cuda"), torch.randn(40, 24, device="cuda", requires_grad=True)
    opt = AdamW([w], lr=1e-3, max_grad_norm=1.0)
    torch.cuda.synchronize()
    lib.insmos_prof_reset()
    lib.insmos_prof_enable(1)
    try:
        linear(x, w, activation="gelu").sum().backward()
        opt.step()
        ids, ms, counts = (ctypes.c_int * 64)(), (ctypes.c_double * 64)(), (ctypes.c_int64 * 64)()
        n = lib.insmos_prof_read(64, ids, ms, counts)
    finally:
        lib.insmos_prof_enable(0)
    seen = {lib.insmos_prof_name(ids[i]).decode(): counts[i] for i in range(n) if counts[i]}
    lib.insmos_prof_reset()
    assert set(seen) == {"linear", "linear_slope", "adamw"}
    assert seen["linear"] in (2, 3, 4) and seen["linear_slope"] == 1 and seen["adamw"] == 3     # products and joins; dz; norm, values, update


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 24), (5, 130, 33), (33, 64, 40), (300, 72, 65), (300, 520, 514), (1000, 40, 8), (61, 700, 2050), (2100, 264, 72), (4100, 2050, 30)])
def test_what_lies_around_the_operands_is_not_used(dtype, m, k, n):
    """Every operand as a block of a larger matrix of NaN: rows before and behind it, columns on both sides.  Whole numbers, so results are exact."""
    t, gen = getattr(torch, dtype), torch.Generator().manual_seed(m)

    def block(rows, cols, left, right):
        hold = torch.full((rows + 200, cols + left + right), float("nan"), dtype=t, device="cuda")
        v = hold[100:100 + rows, left:left + cols]
        v.copy_(torch.randint(-2, 3, (rows, cols), generator=gen))
        return v

    for left, right in ((8, 8), (2, 6), (1, 2)):
        for out_in in (False, True):
            x, r, dy = block(m, k, left, right), block(m, n, left, right), block(m, n, left, right)
            w = block(n, k, left, right).t() if out_in else block(k, n, left, right)
            ins = [v.detach().requires_grad_(True) for v in (x, w, r)]
            y = linear(ins[0], ins[1], None, ins[2])
            dx, dw, dr = torch.autograd.grad(y, ins, dy)
            X, W, R, D = (v.double() for v in (x, w, r, dy))
            for got, want in ((y, X @ W + R), (dx, D @ W.t()), (dw, X.t() @ D), (dr, D)):
                assert torch.equal(got.detach(), want.to(t)), (left, right, out_in)
