"""An id or label outside its table stops training before it reaches the weights."""
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(m):
    return [p.detach().clone() for p in m.parameters()]


@pytest.mark.parametrize("fuse", [False, True])
@pytest.mark.parametrize("where", ["ids", "labels"])
def test_a_training_step_raises(fuse, where):
    from ccfuser_b200 import TokenIndexError
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.train import TrainStep
    torch.manual_seed(0)
    m = GPTMoE(GPTMoEConfig(vocab_size=1000, n_layer=2, n_head=4, d_model=256, d_ffn=512, seq_len=128, num_experts=8, max_tokens=512, backend="fused"),
               device="cuda")
    trainer = TrainStep(m, lr=1e-2, fuse_expert_sgd=fuse)
    ids = torch.randint(0, 1000, (4, 128)).pin_memory()
    trainer.step(ids)
    before = _weights(m)
    bad = ids.clone().pin_memory()
    bad[2, 5] = 70_000
    with pytest.raises(TokenIndexError, match="training step.*token 261"):
        trainer.step(*((bad, ids) if where == "ids" else (ids, bad)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, _weights(m)))
    loss = trainer.step(ids)                 # the status word is clear again
    assert loss == loss and not all(torch.equal(a, b) for a, b in zip(before, _weights(m)))
    for layer in m.moe_layers():
        layer.release()


@pytest.mark.parametrize("model", ["gpt", "bert", "txl"])
def test_the_training_example_stops(monkeypatch, model):
    from ccfuser_b200 import TokenIndexError
    from ccfuser_b200.examples import train
    made, build = [], train.build

    def with_a_bad_id(*args):
        m, batch, tokens = build(*args)
        batch["ids"][1, 3] = 10 ** 6
        made.append((m, _weights(m)))
        return m, batch, tokens
    monkeypatch.setattr(train, "build", with_a_bad_id)
    monkeypatch.setattr(sys, "argv", ["train", "--model", model, "--variant", "dense", "--layers", "1", "--batch", "2", "--seq", "32", "--steps", "2"])
    with pytest.raises(TokenIndexError, match="step 0.*token 35"):
        train.main()
    torch.cuda.synchronize()
    (m, before), = made
    assert all(torch.equal(a, b) for a, b in zip(before, _weights(m)))


@pytest.mark.parametrize("at", [3, 2 ** 23 - 2, 2 ** 23 - 1, 2 ** 23 + 1])
def test_the_number_of_a_late_token(at):
    """The status word has 23 bits for it: behind them no other token is named."""
    from ccfuser_b200 import TokenIndexError
    from ccfuser_b200.ops.embedding import embedding, embedding_grad
    from ccfuser_b200.ops.gemm import Workspace
    from ccfuser_b200.ops.logprobs import token_logprobs
    n = 2 ** 23 + 2
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    ids[at] = 2
    w = torch.ones(2, 8, device="cuda", dtype=torch.bfloat16)
    calls = [lambda: embedding(ids, w), lambda: token_logprobs(w[:1].expand(n, 8)[:, :2], ids), lambda: embedding_grad(w[:1].expand(n, 8), ids, 2)]
    for call in calls:
        call()
        with pytest.raises(TokenIndexError, match=f"token {at} lies" if at < 2 ** 23 - 1 else "token 8388607 or a later one"):
            Workspace.get("cuda").check("test")
