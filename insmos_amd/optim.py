"""The optimiser step on MI355X: AdamW (or Adam with coupled weight decay, which models/models.py:185-190 trains with) over a whole
list of tensors in one short chain of HIP launches (csrc/optim.hip), moments in 32 or in 8 bits, with the clip by the gradients'
global norm inside the step.

  * AdamW: a torch.optim.Optimizer (learning-rate schedulers, param_groups, state_dict work as usual).
  * adamw_step(): the step itself on flat state buffers.
  * grad_norm(): the global 2-norm of a list of gradients, on the device.

State layout: the moments of a list (and its fp32 master weights) lie in one buffer each; tensor i starts at
256 * sum_{j<i} ceil(numel_j / 256) (state_offsets()), in the tensor's own memory order, and what lies behind its end is zero.
In 8 bits exp_avg holds e4m3 codes of m and exp_avg_sq those of sqrt(v), in units of scales[0] / scales[1], one fp32 value per 256
elements; codes are rounded stochastically by a hash of (element, step, seed), so a step is reproducible.

Nothing is read back from the device and no memory is kept between calls of the functions, so a step can be captured in a graph; a
captured step repeats with the addresses of the tensors it was captured with and the learning rate it was captured with unless that
is a tensor.
"""
import collections
import ctypes
import math

import torch

from . import _lib

STATE_BLOCK = 256     # elements per scale; a tensor's start in the state buffers is a multiple of it
_ENTRY = 32           # bytes of an InsmosOptTensor


def state_offsets(sizes):
    """Starts of tensors of these sizes in the state buffers, and the buffers' length."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-int(n) // STATE_BLOCK) * STATE_BLOCK
    return starts, at


def _table(what, params, grads):
    """(table, its entries, dtype code, length of the state buffers, tensors that the table points into beside the caller's)"""
    from . import _host
    table, extra = bytearray(_ENTRY * max(1, len(grads))), None
    used, dtype, total, reorder = _host.opt_table(what, params, grads, table, False)
    if reorder:
        extra = list(grads)
        for i in reorder:      # gradients in their parameter's memory order (or, alone, any dense one)
            p = grads[i] if params is None else params[i]
            extra[i] = p.contiguous() if params is None else torch.empty_strided(p.shape, p.stride(), dtype=p.dtype,
                                                                                 device=p.device).copy_(grads[i])
        used, dtype, total, _ = _host.opt_table(what, params, extra, table, False)
    return (ctypes.c_char * len(table)).from_buffer(table), used, dtype, total, extra


def grad_norm(grads):
    """The 2-norm over all elements of the tensors (None entries are left out) as a 0-dim float32 tensor on their device; several
    dtypes may be mixed.  Summed in fp64, in a fixed order: the same gradients give the same bits."""
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grad_norm: no gradients")
    lib = _lib.load()
    lists = {}
    for g in grads:
        lists.setdefault(g.dtype, []).append(g)
    dev = grads[0].device
    tables = [_table("grad_norm", None, ts) for ts in lists.values()]
    if any(ts[0].device != dev for ts in lists.values()):
        raise ValueError("grad_norm: all tensors on one device")
    with torch.cuda.device(dev):
        st = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        counts = [int(lib.insmos_grad_sumsq_partials(t[0], t[1])) for t in tables]
        partials = torch.empty(max(1, sum(counts)), dtype=torch.float64, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        at = 0
        for (table, used, dtype, _, _extra), n in zip(tables, counts):
            _lib.check(lib.insmos_grad_sumsq(table, used, dtype, partials.data_ptr() + 8 * at, n, st), "insmos_grad_sumsq")
            at += n
        _lib.check(lib.insmos_grad_norm(partials.data_ptr(), at, norm.data_ptr(), st), "insmos_grad_norm")
    return norm


def _flat(what, t, dtype, n, dev):
    if t.dtype != dtype or t.device != dev or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"adamw_step: {what} is a contiguous {dtype} tensor of {n} elements on {dev}, "
                         f"not {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.data_ptr() % 16:
        raise ValueError(f"adamw_step: {what} starts on a 16-byte boundary")


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, decoupled=True,
               scales=None, masters=None, max_grad_norm=None, grad_norm=None, skip_nonfinite=False, seed=0):
    """One step over `params` (in place) with `grads` (None entries: that tensor and its state stay as they are).

    params, grads: lists of the same length, float32, bfloat16 or float16 (one dtype and device), dense in memory; a parameter may
      appear once.  exp_avg, exp_avg_sq: the moments in the state layout above, both float32, or both torch.float8_e4m3fn with
      scales = float32 (2, length / 256).  step: int32 tensor of one element, the steps done so far; it is advanced.
    lr: a number, or a float32 tensor of one element on the device.  decoupled: AdamW; False: the decay is added to the gradient.
    masters: float32 weights in the state layout (bfloat16 / float16 params only): they are updated, params become their rounding.
    max_grad_norm: the gradients count as scaled by min(1, max_grad_norm / (norm + 1e-6)); they are not changed.
    grad_norm: the norm to clip by, a float32 tensor of one element (grad_norm() of more than this list); None: this list's.
    skip_nonfinite: where the norm is inf or NaN nothing changes, the counter neither.
    Returns the norm as a 0-dim float32 tensor where it was taken or given, else None."""
    params, grads = list(params), list(grads)
    b1, b2 = (float(b) for b in betas)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"adamw_step: betas in [0, 1), not {tuple(betas)}")
    eps, weight_decay = float(eps), float(weight_decay)
    if not 0.0 <= eps < math.inf or not 0.0 <= weight_decay < math.inf:
        raise ValueError(f"adamw_step: eps and weight_decay at least 0, not {eps}, {weight_decay}")
    if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
        raise ValueError(f"adamw_step: max_grad_norm above 0 or None, not {max_grad_norm}")
    table, used, dtype, total, _extra = _table("adamw_step", params, grads)
    dev = params[0].device
    bits = 8 if exp_avg.dtype == torch.float8_e4m3fn else 32
    state = torch.float8_e4m3fn if bits == 8 else torch.float32
    _flat("exp_avg", exp_avg, state, total, dev)
    _flat("exp_avg_sq", exp_avg_sq, state, total, dev)
    if total and abs(exp_avg.data_ptr() - exp_avg_sq.data_ptr()) < total * exp_avg.element_size():
        raise ValueError("adamw_step: exp_avg and exp_avg_sq share memory")
    if bits == 8:
        if scales is None:
            raise ValueError("adamw_step: moments in 8 bits need scales")
        _flat("scales", scales, torch.float32, 2 * total // STATE_BLOCK, dev)
    elif scales is not None:
        raise ValueError("adamw_step: scales belong to moments in 8 bits")
    if masters is not None:
        if dtype == 0:
            raise ValueError("adamw_step: masters belong to bfloat16 or float16 parameters")
        _flat("masters", masters, torch.float32, total, dev)
    if step.dtype != torch.int32 or step.numel() != 1 or step.device != dev:
        raise ValueError(f"adamw_step: step is one int32 on {dev}, not {step.dtype} {tuple(step.shape)} on {step.device}")
    lr_dev = None
    if torch.is_tensor(lr) and lr.device == dev:
        if lr.dtype != torch.float32 or lr.numel() != 1:
            raise ValueError(f"adamw_step: lr is a number or one float32, not {lr.dtype} {tuple(lr.shape)}")
        lr_dev, lr_host = lr.data_ptr(), 0.0
    else:
        lr_host = float(lr)
        if not 0.0 <= lr_host < math.inf:
            raise ValueError(f"adamw_step: lr at least 0, not {lr_host}")
    norm_in = None
    if grad_norm is not None:
        if grad_norm.dtype != torch.float32 or grad_norm.numel() != 1 or grad_norm.device != dev:
            raise ValueError(f"adamw_step: grad_norm is one float32 on {dev}, not {grad_norm.dtype} on {grad_norm.device}")
        norm_in = grad_norm.data_ptr()
    lib = _lib.load()
    with torch.cuda.device(dev):
        norm_out = None
        if grad_norm is None and (max_grad_norm is not None or skip_nonfinite):
            norm_out = torch.empty((), dtype=torch.float32, device=dev)
        need = int(lib.insmos_adamw_ws_bytes(table, used))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.insmos_adamw_step(
            table, used, dtype, bits, exp_avg.data_ptr(), exp_avg_sq.data_ptr(),
            scales.data_ptr() if scales is not None else None, total, masters.data_ptr() if masters is not None else None,
            step.data_ptr(), lr_host, lr_dev, b1, b2, eps, weight_decay, 1 if decoupled else 0,
            float(max_grad_norm) if max_grad_norm is not None else 0.0, norm_in, 1 if skip_nonfinite else 0, int(seed) & 0xFFFFFFFF,
            norm_out.data_ptr() if norm_out is not None else None, ws.data_ptr(), need,
            ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "insmos_adamw_step")
    written = params if used == len(params) else [p for p, g in zip(params, grads) if g is not None]
    torch.autograd.graph.increment_version(written + [exp_avg, exp_avg_sq, step] + [t for t in (scales, masters) if t is not None])
    return grad_norm if grad_norm is not None else norm_out


class _Bucket:
    """The state of one group's parameters of one dtype and device."""

    def __init__(self, params, state_bits, master_weights):
        self.params = params
        dev, dtype = params[0].device, params[0].dtype
        from . import _host
        self.order = _host.opt_order(params)
        self.starts, total = state_offsets([p.numel() for p in params])
        state = torch.float8_e4m3fn if state_bits == 8 else torch.float32
        self.exp_avg, self.exp_avg_sq = (torch.zeros(total, dtype=torch.float32, device=dev).to(state) for _ in range(2))
        self.scales = torch.zeros((2, total // STATE_BLOCK), dtype=torch.float32, device=dev) if state_bits == 8 else None
        # one counter of steps for the parameters that have had gradients in the same steps
        self.steps, self.counter = [torch.zeros(1, dtype=torch.int32, device=dev)], [0] * len(params)
        self.masters = None
        if master_weights and dtype != torch.float32:
            self.masters = torch.zeros(total, dtype=torch.float32, device=dev)
            for i in range(len(params)):
                self.view(self.masters, i).copy_(params[i].detach())

    def __getstate__(self):     # (the codes as bytes: torch pickles no 8-bit floats)
        return {k: v.view(torch.uint8) if torch.is_tensor(v) and v.dtype == torch.float8_e4m3fn else v for k, v in self.__dict__.items()}

    def __setstate__(self, state):
        self.__dict__.update({k: v.view(torch.float8_e4m3fn) if torch.is_tensor(v) and v.dtype == torch.uint8 else v for k, v in state.items()})

    def view(self, flat, i):
        """Tensor i's part of a state buffer, shaped and ordered as the parameter."""
        p = self.params[i]
        return torch.as_strided(flat, p.shape, p.stride(), self.starts[i])

    def entries(self, i):
        """What a state_dict holds of parameter i (views of the buffers; the scales are the blocks' that the tensor covers)."""
        out = {"step": self.steps[self.counter[i]], "exp_avg": self.view(self.exp_avg, i), "exp_avg_sq": self.view(self.exp_avg_sq, i)}
        if self.scales is not None:
            a = self.starts[i] // STATE_BLOCK
            out["scales"] = self.scales[:, a:a + -(-self.params[i].numel() // STATE_BLOCK)]
        if self.masters is not None:
            out["master"] = self.view(self.masters, i)
        return out


    def shares(self, grads, missing):
        """[(counter, gradients of its parameters)] for the parameters that have a gradient, and which parameters' counter has changed: where only some
        of a counter's parameters have one, the others go on with a copy of it.  missing: how many have none."""
        if len(self.steps) == 1 and not missing:     # (the usual step)
            return [(self.steps[0], grads)], []
        lists, moved = [], []
        for k in range(len(self.steps)):
            members = [i for i, c in enumerate(self.counter) if c == k]
            without = [i for i in members if grads[i] is None]
            if len(without) == len(members):
                continue
            if without:
                if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: other parameters have gradients than in the steps before, whose counters part here; that cannot be "
                                       "captured (take one such step before the capture)")
                self.steps.append(self.steps[k].clone())
                for i in without:
                    self.counter[i] = len(self.steps) - 1
                moved += without
            lists.append((self.steps[k], grads if len(members) == len(grads) else [g if c == k else None for g, c in zip(grads, self.counter)]))
        return lists, moved

    def set_steps(self, values):
        """Counters that stand at these numbers, one per parameter."""
        kinds = sorted(set(values))
        self.steps = [torch.full((1,), v, dtype=torch.int32, device=self.exp_avg.device) for v in kinds]
        self.counter = [kinds.index(v) for v in values]


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled=False: Adam with the decay in the gradient) whose step() is adamw_step() on every parameter group.

    state_bits: 32, or 8 (two bytes of moments per parameter and 8 more per 256, instead of eight per parameter).  master_weights: keep fp32 weights of
    bfloat16 / float16 parameters.  max_grad_norm: clip by the norm over ALL gradients of the optimiser.  skip_nonfinite: a step whose
    gradients' norm is inf or NaN changes nothing.  seed: of the 8-bit rounding.  lr may be a float32 tensor on the device (a captured
    step then follows it).  After step(), last_grad_norm holds the norm (None where it was not taken).

    A parameter without a gradient keeps its value, its moments and its count of steps; parameters that have had gradients in the same steps
    share a counter and a call of adamw_step().  The state is made at the first step (or load_state_dict) from the parameters as they are
    then; a group's list, its shapes and their order in memory are fixed from then on.  A captured step needs one that was taken before the
    capture, with gradients of the same parameters."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, decoupled=True, state_bits=32,
                 master_weights=False, max_grad_norm=None, skip_nonfinite=False, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, not {state_bits}")
        if not torch.is_tensor(lr) and not 0.0 <= float(lr) < math.inf:
            raise ValueError(f"AdamW: lr at least 0, not {lr}")
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError(f"AdamW: max_grad_norm above 0 or None, not {max_grad_norm}")
        self.state_bits, self.master_weights = int(state_bits), bool(master_weights)
        self.max_grad_norm, self.skip_nonfinite, self.seed = max_grad_norm, bool(skip_nonfinite), int(seed)
        self.last_grad_norm = None
        self._buckets = {}      # group index -> list of _Bucket
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled=decoupled))

    def _group_buckets(self, gi):
        if gi not in self._buckets:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: the state is made by the first step, which cannot be captured (a replay would clear it)")
            lists = {}
            for p in self.param_groups[gi]["params"]:
                lists.setdefault((p.device, p.dtype), []).append(p)
            self._buckets[gi] = [_Bucket(ps, self.state_bits, self.master_weights) for ps in lists.values()]
            for b in self._buckets[gi]:
                for i, p in enumerate(b.params):
                    self.state[p] = b.entries(i)
        return self._buckets[gi]

    @torch.no_grad()
    def step(self, closure=None):
        from . import _host
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for gi, group in enumerate(self.param_groups):
            for b in self._group_buckets(gi):
                order, grads, missing = _host.opt_grads(b.params)
                if order != b.order:
                    raise RuntimeError("AdamW: a parameter's shape or order in memory has changed since its state was made")
                lists, moved = b.shares(grads, missing)
                for i in moved:
                    self.state[b.params[i]]["step"] = b.steps[b.counter[i]]
                work += [(group, b, counter, grads) for counter, grads in lists]
        norm = None
        wanted = self.max_grad_norm is not None or self.skip_nonfinite
        if wanted and len(work) > 1:
            norm = grad_norm([g for _, _, _, grads in work for g in grads])
        for group, b, counter, grads in work:
            norm_b = adamw_step(b.params, grads, b.exp_avg, b.exp_avg_sq, counter, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                                weight_decay=group["weight_decay"], decoupled=group["decoupled"], scales=b.scales, masters=b.masters,
                                max_grad_norm=self.max_grad_norm, grad_norm=norm, skip_nonfinite=self.skip_nonfinite, seed=self.seed)
        self.last_grad_norm = norm_b if work and wanted else None
        return loss

    _KEPT = ("state_bits", "master_weights", "max_grad_norm", "skip_nonfinite", "seed", "last_grad_norm", "_buckets")

    def __getstate__(self):     # (copies and pickles; the entries of self.state are views of the buffers, made again)
        return {**super().__getstate__(), **{k: getattr(self, k) for k in self._KEPT}, "state": collections.defaultdict(dict)}

    def __setstate__(self, state):
        super().__setstate__(state)
        for bs in self._buckets.values():
            for b in bs:
                for i, p in enumerate(b.params):
                    self.state[p] = b.entries(i)

    def _check_entries(self, what, got, p):
        """`got` is a state_dict's state of a parameter like p."""
        bits = torch.float8_e4m3fn if self.state_bits == 8 else torch.float32
        want = {"step": (torch.int32, (1,)), "exp_avg": (bits, p.shape), "exp_avg_sq": (bits, p.shape)}
        if self.state_bits == 8:
            want["scales"] = (torch.float32, (2, -(-p.numel() // STATE_BLOCK)))
        if self.master_weights and p.dtype != torch.float32:
            want["master"] = (torch.float32, p.shape)
        if set(got) != set(want) or any(not torch.is_tensor(got[k]) or got[k].dtype != t or got[k].shape != torch.Size(s) for k, (t, s) in want.items()):
            raise ValueError(f"AdamW.load_state_dict: the state of parameter {what} is of another kind or shape "
                             f"(state_bits {self.state_bits}, master_weights {self.master_weights} here)")

    def load_state_dict(self, state_dict):
        """A state_dict() of an AdamW with the same state_bits and master_weights over parameters of the same shapes.  One that is refused changes nothing."""
        state = state_dict["state"]
        lists = [[state.get(j) for j in group["params"]] for group in state_dict["param_groups"]]      # (as the groups' parameters)
        for group, ids, got in zip(self.param_groups, state_dict["param_groups"], lists):
            for p, j, entries in zip(group["params"], ids["params"], got):
                if entries is not None:
                    self._check_entries(j, entries, p)
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})     # (refuses groups of other sizes)
        self._buckets.clear()
        self.state.clear()
        for gi, (group, got) in enumerate(zip(self.param_groups, lists)):
            if all(entries is None for entries in got):
                continue
            entries_of = {id(p): entries for p, entries in zip(group["params"], got)}
            for b in self._group_buckets(gi):
                steps = [0] * len(b.params)
                for i, p in enumerate(b.params):
                    entries = entries_of[id(p)]
                    if entries is None:
                        continue
                    steps[i] = int(entries["step"])
                    for k, t in b.entries(i).items():
                        if k != "step":
                            t.copy_(entries[k])
                b.set_steps(steps)
                for i, p in enumerate(b.params):
                    self.state[p]["step"] = b.steps[b.counter[i]]
