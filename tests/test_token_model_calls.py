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
