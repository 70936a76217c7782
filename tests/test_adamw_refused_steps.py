"""A step of FusedAdamW that is refused: step numbers, moments and weights stay, and the next one goes on as if it had not been."""
import copy

import pytest
import torch

from ccfuser_b200.ops.optim import FusedAdamW

SHAPES = ((70, 60), (9,), (65, 64), (3, 3))


def _params():
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(shape, generator=g)) for shape in SHAPES]


def _set_gradients(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=g)


def _make(bits, groups, capturable):
    params = _params()
    split = [{"params": params[:2]}, {"params": params[2:]}] if groups == 2 else params
    return FusedAdamW(split, lr=1e-2, state_bits=bits, capturable=capturable), params


def _all_of(opt, params):
    return copy.deepcopy([{**opt.state[p]} if p in opt.state else None for p in params]), [p.detach().clone() for p in params]


def _assert_same(a, b):
    for s, t, p, q in zip(a[0], b[0], a[1], b[1]):
        assert torch.equal(p, q) and (s is None) == (t is None)
        for name in s or ():
            assert torch.equal(s[name], t[name]) if torch.is_tensor(s[name]) else s[name] == t[name], name


@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("where", range(4))
@pytest.mark.parametrize("bits,groups,capturable", [(32, 1, False), (8, 1, False), (8, 2, False), (32, 1, True), (8, 1, True), (32, 2, True)])
def test_a_sparse_gradient_anywhere(bits, groups, capturable, where, steps):
    (a, params), (b, others) = (_make(bits, groups, capturable) for _ in range(2))
    for i in range(steps):
        for opt, mine in ((a, params), (b, others)):
            _set_gradients(mine, i)
            opt.step()
    before = _all_of(a, params)
    _set_gradients(params, 10)
    params[where].grad = params[where].grad.to_sparse()
    with pytest.raises(TypeError):
        a.step()
    _assert_same(_all_of(a, params), before)
    for i in range(20, 22):
        for opt, mine in ((a, params), (b, others)):
            _set_gradients(mine, i)
            opt.step()
    _assert_same(_all_of(a, params), _all_of(b, others))


@pytest.mark.parametrize("capturable", [False, True])
def test_a_later_call_that_is_refused_leaves_the_counts_of_those_before_it(capturable):
    """Moments of another shape in the last batch: the batch before it has taken its step, is counted, and goes on rightly."""
    opt, params = _make(8, 1, capturable)
    for i in range(2):
        _set_gradients(params, i)
        opt.step()
    small, whole = opt.state[params[1]], opt.state[params[1]]["exp_avg"]
    small["exp_avg"] = whole[:5]
    _set_gradients(params, 2)
    with pytest.raises(ValueError):
        opt.step()
    assert int(opt.state[params[0]]["step"]) == 3 and int(small["step"]) == (3 if capturable else 2)
    small["exp_avg"] = whole
    _set_gradients(params, 3)
    opt.step()
    assert int(opt.state[params[0]]["step"]) == 4 and int(small["step"]) == (4 if capturable else 3)
