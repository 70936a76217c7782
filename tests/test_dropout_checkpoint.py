"""Seed, step and call number of dropouts in checkpoints. No GPU."""
import json

import pytest
import torch
from test_token_models import _txl

from ccfuser_b200.ops.dropout import Dropout, DropoutState
from ccfuser_b200.utils.checkpoint import load_ep_checkpoint, save_ep_checkpoint


def _steps(m, n, first):
    torch.manual_seed(first)
    out = []
    for _ in range(n):
        x, y = torch.randint(0, 50, (2, 8)), torch.randint(0, 50, (2, 8))
        out.append(m(x, y)[0].detach())
    return out


@pytest.mark.parametrize("seed", [5, None])
def test_a_resumed_run_goes_on_with_its_masks(tmp_path, seed):
    m = _txl(dropout=0.3, dropout_seed=seed)
    first = _steps(m, 2, 1)
    save_ep_checkpoint(m, str(tmp_path / "c"), 0, 1)
    want = _steps(m, 3, 2)
    torch.manual_seed(99)                            # a new process draws another seed
    again = type(m)(m.config)
    assert load_ep_checkpoint(again, str(tmp_path / "c"), 0, 1)["dropout_restored"]
    assert all(torch.equal(a, b) for a, b in zip(want, _steps(again, 3, 2)))
    fresh = _txl(dropout=0.3, dropout_seed=seed)
    assert all(torch.equal(a, b) for a, b in zip(first, _steps(fresh, 2, 1)))


def test_a_checkpoint_without_dropout_states(tmp_path):
    m = _txl(dropout=0.3, dropout_seed=5)
    save_ep_checkpoint(m, str(tmp_path / "c"), 0, 1)
    manifest = json.loads((tmp_path / "c.manifest.json").read_text())
    del manifest["dropout"]                          # as earlier ones are
    (tmp_path / "c.manifest.json").write_text(json.dumps(manifest))
    _steps(m, 1, 1)
    assert not load_ep_checkpoint(m, str(tmp_path / "c"), 0, 1)["dropout_restored"]
    assert m.drop.state.tensor.tolist() == [5, 1]
    plain = _txl()
    assert load_ep_checkpoint(plain, str(tmp_path / "c"), 0, 1)["dropout_restored"]      # none in either


def test_states_across_ranks():
    """One rank's state serves all: each draws with the seed of its own."""
    a, b = DropoutState(7, rank=0), DropoutState(1, rank=3)
    for _ in range(4):
        a.advance()
    a.next_call()
    before = b.tensor
    b.load_state_dict(a.state_dict())
    assert b.tensor is before and b.tensor.tolist() == [10, 4] and b.calls == 1
    a.load_state_dict(b.state_dict())
    assert a.tensor.tolist() == [7, 4]
    top = DropoutState(2 ** 63 - 1, rank=2)
    assert top.tensor.tolist() == [-2 ** 63 + 1, 0] and top.state_dict()["seed"] == 2 ** 63 - 1
    drop = torch.nn.Sequential(Dropout(0.5, a), Dropout(0.1, a), Dropout(0.1, b))
    from ccfuser_b200.utils.checkpoint import dropout_states
    assert dropout_states(drop) == [a, b]
