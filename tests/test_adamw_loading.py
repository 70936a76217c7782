"""What FusedAdamW takes over from checkpoints, torch's among them, and what it refuses."""
import copy

import pytest
import torch
import training_refs as T

from ccfuser_b200.ops import optim as O
from ccfuser_b200.ops.optim import FusedAdamW, adamw_step, state_values


def _params(dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(shape, generator=g).to(dtype)) for shape in ((90, 60), (9,))]


def _train(opt, params, seed, steps):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype)
        opt.step()


def _all_of(opt):
    """Groups and state as plain values, tensors copied."""
    copied = copy.deepcopy(opt.state_dict())
    return copied["param_groups"], copied["state"]


def _assert_same(a, b):
    assert a[0] == b[0] and a[1].keys() == b[1].keys()
    for i, state in a[1].items():
        assert state.keys() == b[1][i].keys()
        for name, t in state.items():
            u = b[1][i][name]
            assert torch.equal(t, u) and t.dtype == u.dtype if torch.is_tensor(t) else t == u


@pytest.mark.parametrize("flag", ["maximize", "amsgrad"])
def test_what_it_cannot_do_is_refused_and_nothing_changes(flag):
    params, theirs = _params(), _params()
    ref = torch.optim.AdamW(theirs, lr=0.5, **{flag: True})
    _train(ref, theirs, 1, 2)
    opt = FusedAdamW(params, lr=1e-2, state_bits=8, seed=3)
    _train(opt, params, 2, 2)
    before, weights = _all_of(opt), [p.detach().clone() for p in params]
    with pytest.raises(ValueError, match=flag):
        opt.load_state_dict(ref.state_dict())
    _assert_same(_all_of(opt), before)
    assert all(torch.equal(p, w) for p, w in zip(params, weights))
    # and it loads on
    plain = torch.optim.AdamW(theirs, lr=0.5)
    _train(plain, theirs, 1, 2)
    opt.load_state_dict(plain.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and opt.state[params[0]]["step"] == 2


@pytest.mark.parametrize("option", [dict(maximize=True), dict(amsgrad=True), dict(state_bits=4), dict(state_bits=16)])
def test_options_of_a_group_are_refused_like_the_constructors(option):
    a, b = _params()
    with pytest.raises(ValueError):
        FusedAdamW([{"params": [a], **option}])
    opt = FusedAdamW([a])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [b], **option})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [b], "state_bits": 8, "maximize": False})
    assert [g["state_bits"] for g in opt.param_groups] == [32, 8]


@pytest.mark.parametrize("piece", [256, 1024, 1 << 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("capturable", [False, True])
def test_torchs_checkpoint_in_8_bits(dtype, capturable, piece, monkeypatch):
    """Groups keep what torch's know nothing of; moments come into 8 bits as a step would round them, in pieces of any size, and train on."""
    monkeypatch.setattr(O, "_PIECE", piece)
    g = torch.Generator().manual_seed(4)
    make = lambda: [torch.nn.Parameter(torch.ones(s, dtype=dtype)) for s in ((3, 1500), (70, 70), (9,), (4, 1100))]  # noqa: E731
    theirs, params = make(), make()
    params[0].skip_allreduce = True      # an expert's: exponents by row
    ref = torch.optim.AdamW([{"params": theirs[:1], "lr": 0.1}, {"params": theirs[1:], "lr": 0.2}])
    for _ in range(3):
        for p in theirs[:3]:             # the last has no gradient yet
            p.grad = torch.randn(p.shape, generator=g).to(dtype)
        ref.step()
    opt = FusedAdamW([{"params": params[:1]}, {"params": params[1:], "seed": 11}], state_bits=8, seed=7, capturable=capturable)
    opt.load_state_dict(ref.state_dict())
    assert [(q["lr"], q["state_bits"], q["seed"], q["capturable"]) for q in opt.param_groups] == [(0.1, 8, 7, capturable), (0.2, 8, 11, capturable)]
    for p, q, rows, seed, number in ((params[0], theirs[0], 3, 7, 0), (params[1], theirs[1], 1, 11 + (1 << 32), 0)):
        state = opt.state[p]
        assert state["exponents"].shape[0] == rows and state["exp_avg"].dtype == torch.uint8 and int(state["step"]) == 3
        bits = T.rounding_bits(seed, 3, number, p.numel())
        for k, (name, these) in enumerate((("exp_avg", [b & 0xFFFFF for b in bits]), ("exp_avg_sq", [b >> 12 for b in bits]))):
            got = state_values(state[name], state["exponents"], k == 1, torch.float32)
            assert torch.equal(got.double(), T.stored(ref.state[q][name], rows, these, k == 1)), name
    small = opt.state[params[2]]
    assert "exponents" not in small and torch.equal(small["exp_avg"], ref.state[theirs[2]]["exp_avg"].float())
    # the next step is one on these codes, and what starts later has 8 bits
    want = {n: t.clone() for n, t in opt.state[params[1]].items() if n != "step"}
    weight, grads = params[1].detach().clone(), [torch.randn(p.shape, generator=g).to(dtype) for p in params]
    for p, grad in zip(params, grads):
        p.grad = grad
    opt.step()
    adamw_step([weight], [grads[1]], [want["exp_avg"]], [want["exp_avg_sq"]], 4, lr=0.2, exponents=[want["exponents"]], seed=11 + (1 << 32))
    assert torch.equal(weight, params[1]) and all(torch.equal(t, opt.state[params[1]][n]) for n, t in want.items())
    assert opt.state[params[3]]["exp_avg"].dtype == torch.uint8 and int(opt.state[params[0]]["step"]) == 4


def test_own_options_come_from_the_checkpoint():
    params, others = _params(), _params()
    a = FusedAdamW(params, state_bits=8, seed=3)
    _train(a, params, 1, 2)
    b = FusedAdamW(others, seed=5)
    b.load_state_dict(a.state_dict())
    assert (b.param_groups[0]["state_bits"], b.param_groups[0]["seed"]) == (8, 3) and torch.equal(a.state[params[0]]["exponents"], b.state[others[0]]["exponents"])


def test_values_that_are_not_finite_come_into_8_bits_as_in_a_step():
    p, q = torch.nn.Parameter(torch.ones(80, 64)), torch.nn.Parameter(torch.ones(80, 64))
    ref = torch.optim.AdamW([p])
    p.grad = torch.ones_like(p)
    ref.step()
    ref.state[p]["exp_avg"][0, 0] = torch.inf
    opt = FusedAdamW([q], state_bits=8)
    opt.load_state_dict(ref.state_dict())
    first = state_values(opt.state[q]["exp_avg"], opt.state[q]["exponents"], dtype=torch.float32).reshape(-1)
    assert first[:256].isnan().all() and first[256:].isfinite().all()


class _Made(torch.utils._python_dispatch.TorchDispatchMode):
    """The bytes an element of the largest tensors that operations make."""

    def __init__(self, numel):
        super().__init__()
        self.numel, self.widest = numel, 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if torch.is_tensor(out) and out.numel() >= self.numel:
            self.widest = max(self.widest, out.element_size())
        return out


@pytest.mark.parametrize("dtype,bits,widest", [(torch.bfloat16, 8, 1), (torch.float32, 8, 1), (torch.bfloat16, 32, 4)])
def test_loading_makes_nothing_wider_than_what_it_keeps(dtype, bits, widest):
    params, others = _params(dtype), _params(dtype)
    a, b = FusedAdamW(params, state_bits=bits), FusedAdamW(others)
    _train(a, params, 1, 2)
    saved = a.state_dict()
    with _Made(params[0].numel()) as made:
        b.load_state_dict(saved)
    assert made.widest == widest
    _assert_same(_all_of(a), _all_of(b))


def test_hooks_of_a_load_see_the_dictionary_and_what_came_of_it():
    params, others = _params(torch.bfloat16), _params(torch.bfloat16)
    a, b = FusedAdamW(params, state_bits=8), FusedAdamW(others)
    _train(a, params, 1, 2)
    seen = []
    b.register_load_state_dict_pre_hook(lambda _, d: {**d, "param_groups": [{**g, "lr": 0.25} for g in d["param_groups"]]})
    b.register_load_state_dict_post_hook(lambda opt: seen.append({n: t for n, t in opt.state[others[0]].items()}))
    b.load_state_dict(a.state_dict())
    assert b.param_groups[0]["lr"] == 0.25 and seen[0].keys() == a.state[params[0]].keys()
    assert seen[0]["exp_avg"].dtype == torch.uint8 and torch.equal(seen[0]["exp_avg"], a.state[params[0]]["exp_avg"])


def test_a_load_that_fails_changes_nothing():
    params, theirs = _params(), _params()
    opt, ref = FusedAdamW(params, state_bits=8, lr=1e-2), torch.optim.AdamW(theirs, lr=0.5)
    _train(opt, params, 1, 2)
    _train(ref, theirs, 1, 2)
    before = _all_of(opt)
    broken = copy.deepcopy(ref.state_dict())
    del broken["state"][1]["exp_avg_sq"]
    cut = copy.deepcopy(ref.state_dict())
    cut["state"][0]["exp_avg"] = cut["state"][0]["exp_avg"][1:]
    for bad in (broken, cut, torch.optim.SGD(theirs).state_dict(), torch.optim.AdamW(theirs[:1]).state_dict()):
        with pytest.raises((KeyError, ValueError)):
            opt.load_state_dict(bad)
        _assert_same(_all_of(opt), before)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5


@pytest.mark.parametrize("capturable", [False, True])
def test_rates_that_torch_keeps_in_tensors(capturable):
    params, theirs = _params(), _params()
    ref = torch.optim.AdamW(theirs, lr=torch.tensor(0.1, dtype=torch.float64), betas=(torch.tensor(0.8), torch.tensor(0.99)))
    opt = FusedAdamW(params, capturable=capturable)
    opt.load_state_dict(ref.state_dict())
    lr = opt.param_groups[0]["lr"]
    assert torch.is_tensor(lr) == capturable and (not capturable or lr.dtype == torch.float32)
    want, weights = copy.deepcopy(params), [p.detach().clone() for p in params]
    _train(FusedAdamW(want, lr=float(lr), betas=tuple(float(torch.tensor(b)) for b in (0.8, 0.99))), want, 1, 2)
    _train(opt, params, 1, 2)
    assert all(torch.equal(p, q) and not torch.equal(p, w) for p, q, w in zip(params, want, weights))


def test_a_group_without_parameters():
    params, theirs = _params(), _params()
    make = lambda cls, p: cls([{"params": p}, {"params": []}], lr=torch.tensor(0.1), capturable=True)  # noqa: E731
    a, b = make(FusedAdamW, params), make(FusedAdamW, theirs)
    _train(a, params, 1, 1)
    b.load_state_dict(a.state_dict())
    _assert_same(_all_of(a), _all_of(b))
