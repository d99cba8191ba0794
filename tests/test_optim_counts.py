"""insmos_amd.optim.AdamW where not every parameter has a gradient in every step."""
import copy

import pytest
import torch

from insmos_amd.optim import AdamW

U32 = 2.0 ** -24
# steps in which a parameter has a gradient: always, late, in turns, never, in the first alone
PATTERN = [lambda it: True, lambda it: it >= 3, lambda it: it % 2 == 0, lambda it: it % 2 == 1, lambda it: False, lambda it: it == 0, lambda it: True]
SHAPES = [(40, 30), (257,), (5, 5, 5), (300,), (17,), (64,), (9,)]


def _grads(params, it, scale=1.0):
    gen = torch.Generator().manual_seed(100 + it)
    for p, has in zip(params, PATTERN):
        g = scale * torch.randn(p.shape, generator=gen)
        p.grad = g.to(p.dtype).to(p.device) if has(it) else None


@pytest.mark.gpu
@pytest.mark.parametrize("decoupled", [True, False])
@pytest.mark.parametrize("clip", [None, 3.0])
def test_late_gradients_follow_torch(decoupled, clip):
    """Every parameter's bias corrections count its own steps, as torch's do (counted by the list's, a first gradient in the fourth step would make an
    update of lr (1 - b1) / (1 - b1^4) sqrt((1 - b2^4) / (1 - b2)) = 0.58 lr, and one in the thousandth of 2.5 lr)."""
    gen = torch.Generator().manual_seed(0)
    start = [torch.randn(s, generator=gen) for s in SHAPES]
    ref, own = [t.double().requires_grad_(True) for t in start], [t.cuda().requires_grad_(True) for t in start]
    o_ref = (torch.optim.AdamW if decoupled else torch.optim.Adam)(ref, lr=1e-2, weight_decay=0.1, eps=1e-6)
    o_own = AdamW(own, lr=1e-2, weight_decay=0.1, eps=1e-6, decoupled=decoupled, max_grad_norm=clip)
    for it in range(8):
        _grads(ref, it)
        _grads(own, it)
        if clip:
            norm = float(torch.nn.utils.clip_grad_norm_([p for p in ref if p.grad is not None], clip))
        o_ref.step()
        o_own.step()
        if clip:
            assert abs(float(o_own.last_grad_norm) - norm) < 4 * U32 * norm
        for a, b in zip(ref, own):
            # an update is at most ~ lr / (1 - b1) long and known to some 40 roundings (m cancels at most between steps of equal size: x 10)
            assert float((b.detach().cpu().double() - a.detach()).abs().max()) < (it + 1) * (0.1 * 400 * U32 + 4 * U32), it
        for p, q in zip(ref, own):
            assert int(o_own.state[q]["step"]) == int(o_ref.state[p]["step"] if o_ref.state[p] else 0)
    assert torch.equal(own[4].detach().cpu(), start[4])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_counts_survive_state_dicts_and_copies(bits):
    gen = torch.Generator().manual_seed(1)
    start = [torch.randn(s, generator=gen) for s in SHAPES]

    def go(params, o, its):
        for it in its:
            _grads(params, it)
            o.step()
        return [p.detach().clone() for p in params]

    ps = [t.cuda().requires_grad_(True) for t in start]
    o = AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=4)
    half = go(ps, o, range(4))
    saved, copied = copy.deepcopy(o.state_dict()), copy.deepcopy(o)
    want = go(ps, o, range(4, 8))
    qs = [t.clone().requires_grad_(True) for t in half]
    o2 = AdamW(qs, lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=4)
    o2.load_state_dict(saved)
    assert [int(o2.state[q]["step"]) for q in qs] == [4, 1, 2, 2, 0, 1, 4]
    assert all(torch.equal(a, b) for a, b in zip(go(qs, o2, range(4, 8)), want))
    assert all(torch.equal(a, b) for a, b in zip(go(copied.param_groups[0]["params"], copied, range(4, 8)), want))
    assert [int(o.state[p]["step"]) for p in ps] == [int(o2.state[q]["step"]) for q in qs]


@pytest.mark.gpu
def test_a_captured_step_counts_for_its_parameters():
    """A set of gradients that has been stepped with can be captured and replays advance its counter alone; another set cannot."""
    gen = torch.Generator().manual_seed(2)
    start = [torch.randn(s, generator=gen) for s in SHAPES[:3]]
    runs = []
    for captured in (True, False):
        ps = [t.cuda().requires_grad_(True) for t in start]
        o = AdamW(ps, lr=1e-2)
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        o.step()
        ps[1].grad = None
        if captured:
            said, empty = None, torch.cuda.CUDAGraph()
            with torch.cuda.graph(empty):
                try:
                    o.step()
                except RuntimeError as e:
                    said = str(e)
            assert "counters part" in said and [int(o.state[p]["step"]) for p in ps] == [1, 1, 1]
        o.step()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o.step()
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
        else:
            for _ in range(3):
                o.step()
        assert [int(o.state[p]["step"]) for p in ps] == [5, 1, 5]
        runs.append([p.detach().clone() for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def _state(params, bits, steps):
    """A state_dict's state of these parameters with recognisable values."""
    out, at = {}, 0
    for i, p in enumerate(params):
        m = torch.full(p.shape, float(i + 1))
        out[i] = {"step": torch.tensor([steps[i]], dtype=torch.int32), "exp_avg": m, "exp_avg_sq": m * 2}
        if bits == 8:
            out[i] = {**{k: v.to(torch.float8_e4m3fn) if k != "step" else v for k, v in out[i].items()},
                      "scales": torch.full((2, -(-p.numel() // 256)), 0.5)}
    return out


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_state_dict_changes_nothing(bits):
    """Whatever is wrong with a state_dict is found before the state that is there is touched: the last parameter's shape, its kind of state, a missing
    entry, another optimiser's state, groups of other sizes."""
    ps = [torch.zeros(s, requires_grad=True) for s in SHAPES]
    o = AdamW([{"params": ps[:4]}, {"params": ps[4:]}], lr=1e-3, state_bits=bits)
    groups = o.state_dict()["param_groups"]
    good = _state(ps, bits, [3, 1, 3, 0, 7, 7, 2])
    o.load_state_dict({"state": good, "param_groups": groups})

    def same():
        have = o.state_dict()
        return have["param_groups"] == groups and all(torch.equal(have["state"][i][k].view(torch.uint8), t.view(torch.uint8)) for i in good for k, t in good[i].items())

    assert same() and [int(o.state[p]["step"]) for p in ps] == [3, 1, 3, 0, 7, 7, 2]
    last, other = len(ps) - 1, _state(ps, 40 - bits, [5] * 7)
    shape = _state([*ps[:-1], torch.zeros(10)], bits, [5] * 7)
    missing = {**_state(ps, bits, [5] * 7), last: {k: t for k, t in good[last].items() if k != "exp_avg_sq"}}
    foreign = {**_state(ps, bits, [5] * 7), last: {**good[last], "step": torch.tensor(3.0)}}
    warmer = [{**g, "lr": 9.0} for g in groups]
    for state in (other, shape, missing, foreign):
        with pytest.raises(ValueError):
            o.load_state_dict({"state": state, "param_groups": warmer})
        assert same()
    for bad in (warmer[:1], [warmer[0], {**warmer[1], "params": [4, 5]}]):
        with pytest.raises(ValueError):
            o.load_state_dict({"state": _state(ps, bits, [5] * 7), "param_groups": bad})
        assert same()


def test_a_state_dict_goes_by_the_numbers_of_its_groups():
    """Parameters are matched through the groups' lists, as torch.optim does, and ones without state start anew."""
    ps = [torch.zeros(4, requires_grad=True) for _ in range(3)]
    o = AdamW(ps, lr=1e-3)
    state = _state(ps, 32, [1, 2, 3])
    del state[1]
    o.load_state_dict({"state": state, "param_groups": [{**o.state_dict()["param_groups"][0], "params": [2, 1, 0]}]})
    assert [int(o.state[p]["step"]) for p in ps] == [3, 0, 1] and [float(o.state[p]["exp_avg"][0]) for p in ps] == [3.0, 0.0, 1.0]
