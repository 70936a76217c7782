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
