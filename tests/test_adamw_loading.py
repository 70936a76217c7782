"""What FusedAdamW takes over from checkpoints, torch's among them, and what it refuses."""
import copy

import pytest
import torch

from ccfuser_b200.ops.optim import FusedAdamW


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
