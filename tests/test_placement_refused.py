"""``rebalance_experts`` that is refused leaves every tensor where it was, whichever parameter the refusal is about; on one rank and between two."""
import pytest
import torch
import torch.nn as nn

from ccfuser_b200 import MoEConfig, MoELayer
from ccfuser_b200.ops.optim import FusedAdamW, state8
from ccfuser_b200.parallel.placement import rebalance_experts

PLACEMENT = [2, 0, 3, 1]


def _layer(world=1):
    torch.manual_seed(5)
    return MoELayer(MoEConfig(d_model=1100, d_ffn=70, num_experts=4, dtype=torch.float32, backend="cpu", ep_size=world, max_tokens=16))


def _step(layer, opt, rank=0):
    opt.zero_grad()
    layer(torch.randn(16, 1100, generator=torch.Generator().manual_seed(7 + rank))).square().sum().backward()
    opt.step()


def _all_of(layer, opt):
    found = {n: [p.detach().clone()] + [t.clone() for t in opt.state.get(p, {}).values() if torch.is_tensor(t)] for n, p in layer.named_parameters()}
    return found, getattr(layer, "placement_history", None)


def _assert_refused(layer, opt, error):
    before = _all_of(layer, opt)
    with pytest.raises(error):
        rebalance_experts(layer, PLACEMENT, opt)
    after = _all_of(layer, opt)
    assert before[1] == after[1]
    for name, tensors in before[0].items():
        assert all(torch.equal(a, b) for a, b in zip(tensors, after[0][name])), name


def _replace_router(layer):
    """A router put in behind the layer's making, without its marks."""
    old = layer.gate.gate
    layer.gate.gate = nn.Linear(old.in_features, old.out_features, bias=old.bias is not None)


def _break(layer, opt, which):
    p = dict(layer.named_parameters())[which]
    opt.state[p]["exponents"] = state8(p)[2]


@pytest.mark.parametrize("which", ["experts.htoh4.weight", "experts.h4toh.weight", "gate.gate.weight", "router", "no router"])
def test_on_one_rank(which):
    layer = _layer()
    if which == "router":
        _replace_router(layer)
    opt = FusedAdamW(layer.parameters(), lr=1e-2, state_bits=8)
    _step(layer, opt)
    assert "exponents" in opt.state[layer.gate.gate.weight]
    error = ValueError
    if which == "no router":
        layer.gate.gate, error = nn.Linear(1100, 3), TypeError
    elif which != "router":
        _break(layer, opt, which)
    _assert_refused(layer, opt, error)


def test_a_gate_that_refuses_by_itself():
    layer = _layer()
    opt = FusedAdamW(layer.parameters(), lr=1e-2, state_bits=8)
    _step(layer, opt)

    def refuse(placement, optimizer):
        raise RuntimeError("not now")

    layer.gate.permute_experts = refuse
    _assert_refused(layer, opt, RuntimeError)


def _ranks(rank, world):
    for which in ("router", "experts.h4toh.weight"):
        layer = _layer(world)
        if which == "router":
            torch.manual_seed(6)
            _replace_router(layer)
        opt = FusedAdamW(layer.parameters(), lr=1e-2, state_bits=8)
        _step(layer, opt, rank)
        if which != "router":
            _break(layer, opt, which)
        _assert_refused(layer, opt, ValueError)
    return True


def test_between_two_ranks():
    from mp_util import run_ranks
    assert run_ranks(_ranks, 2) == [True, True]
