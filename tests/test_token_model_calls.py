"""Calls that the models took while their embeddings and losses were torch's. No GPU."""
import pytest
import torch
import torch.nn.functional as F
from test_token_models import _gpt, _txl

from ccfuser_b200.models.bert_moe import BertMoEConfig, BertMoEForQuestionAnswering


@pytest.mark.parametrize("shape", [(48,), (48, 1), (2, 24)])
def test_labels_of_another_shape(shape):
    ids, labels = torch.randint(0, 200, (3, 16)), torch.randint(0, 200, (3, 16))
    m = _gpt()
    assert torch.equal(m(ids, labels.reshape(shape)), m(ids, labels))
    x, y = torch.randint(0, 50, (6, 8)), torch.randint(0, 50, (6, 8))
    m = _txl()
    assert torch.equal(m(x, y.reshape(shape))[0], m(x, y)[0])


@pytest.mark.parametrize("ids_shape,types_shape", [((1, 9), (3, 9)), ((3, 9), (1, 9)), ((3, 9), (9,)), ((3, 9), (3, 9))])
def test_bert_token_types_broadcast(ids_shape, types_shape):
    torch.manual_seed(0)
    m = BertMoEForQuestionAnswering(BertMoEConfig(vocab_size=60, n_layer=1, n_head=2, d_model=32, d_ffn=64, max_position=20, moe_layers=(),
                                                  dtype=torch.float32))
    ids, tt = torch.randint(0, 60, ids_shape), torch.randint(0, 2, types_shape)
    seen = []
    m.ln_emb.register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
    start, _ = m(ids, None, tt)
    want = F.embedding(ids, m.word.weight) + F.embedding(torch.arange(9), m.position.weight) + F.embedding(tt, m.token_type.weight)
    torch.testing.assert_close(seen[0], want)
    assert start.shape == (3, 9)


def test_the_embedding_factor_of_transformer_xl():
    m, ids = _txl(), torch.randint(0, 50, (2, 8))
    assert m.emb_scale == 32 ** 0.5
    seen = []
    m.layers[0].register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
    m.emb_scale = 2.0
    m(ids)
    torch.testing.assert_close(seen[0], F.embedding(ids, m.word_emb.weight) * 2.0)


class _Adapter(torch.nn.Module):
    """A low-rank addition to a table, which keeps the table's name for its weight."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.a, self.b = torch.nn.Parameter(torch.randn(base.num_embeddings, 2)), torch.nn.Parameter(torch.randn(2, base.embedding_dim))

    @property
    def weight(self):
        return self.base.weight

    def forward(self, ids):
        return self.base(ids) + F.embedding(ids, self.a) @ self.b


def _tables(name):
    """A model, the call that runs it, its embedding modules and what the sum of their outputs goes through."""
    torch.manual_seed(0)
    ids, tt = torch.randint(0, 40, (2, 8)), torch.randint(0, 2, (2, 8))
    if name == "gpt":
        m = _gpt()
        return m, lambda: m(ids), {"wte": ids, "wpe": torch.arange(8)}, m.h[0], 1.0
    if name == "bert":
        m = BertMoEForQuestionAnswering(BertMoEConfig(vocab_size=60, n_layer=1, n_head=2, d_model=32, d_ffn=64, max_position=20, moe_layers=(),
                                                      dtype=torch.float32))
        return m, lambda: m(ids, None, tt), {"word": ids, "position": torch.arange(8), "token_type": tt}, m.ln_emb, 1.0
    m = _txl()
    return m, lambda: m(ids), {"word_emb": ids}, m.layers[0], 32 ** 0.5


@pytest.mark.parametrize("name,table", [("gpt", "wte"), ("gpt", "wpe"), ("bert", "word"), ("bert", "position"), ("bert", "token_type"), ("txl", "word_emb")])
@pytest.mark.parametrize("change", ["replaced", "adapter", "hook", "pre_hook"])
def test_replaced_and_hooked_tables(name, table, change):
    """An embedding module is what it does when called: another module, an adapter around it or a hook counts as it did."""
    m, call, places, first, scale = _tables(name)
    calls = []
    if change == "replaced":
        old = getattr(m, table)
        setattr(m, table, torch.nn.Embedding(old.num_embeddings, old.embedding_dim))
    elif change == "adapter":
        setattr(m, table, _Adapter(getattr(m, table)))
    elif change == "hook":
        getattr(m, table).register_forward_hook(lambda mod, args, out: calls.append(1) or out * 3.0)
    else:
        getattr(m, table).register_forward_pre_hook(lambda mod, args: calls.append(1))
    want = 0.0
    for i, (n, at) in enumerate(places.items()):
        part = getattr(m, n)(at)
        want = want + (part * scale if i == 0 else part)
    del calls[:]
    seen = []
    first.register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
    call()
    torch.testing.assert_close(seen[0], want)
    assert len(calls) == ("hook" in change)


def test_a_step_of_its_own_in_a_subclass():
    from ccfuser_b200.train import TrainStep

    class Counted(TrainStep):
        steps = 0

        def step_device(self, ids, labels):
            self.steps += 1
            return super().step_device(ids, labels)
    trainer = Counted(_gpt())
    ids = torch.randint(0, 200, (2, 16))
    before = [p.detach().clone() for p in trainer.raw_model.parameters()]
    assert trainer.step(ids) > 0 and trainer.steps == 1
    assert not all(torch.equal(a, b) for a, b in zip(before, trainer.raw_model.parameters()))
    before = [p.detach().clone() for p in trainer.raw_model.parameters()]
    with pytest.raises(IndexError):
        trainer.step(ids + 256)
    assert all(torch.equal(a, b) for a, b in zip(before, trainer.raw_model.parameters()))
