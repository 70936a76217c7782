"""The models' ends on the host: embedding, dropout and loss as the library's operators against what they are made of. No GPU."""
import pytest
import torch
import torch.nn.functional as F

from ccfuser_b200.models.bert_moe import BertMoEConfig, BertMoEForQuestionAnswering
from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig


def _gpt(**kw):
    torch.manual_seed(0)
    return GPTMoE(GPTMoEConfig(vocab_size=200, n_layer=2, n_head=2, d_model=32, d_ffn=64, seq_len=16, moe_every=0, dtype=torch.float32, **kw))


def _txl(**kw):
    torch.manual_seed(0)
    return TransformerXLMoE(TransformerXLMoEConfig(n_token=50, n_layer=2, n_head=2, d_model=32, d_head=16, d_inner=64, tgt_len=8, mem_len=8, moe=False,
                                                   dtype=torch.float32, **kw))


def test_gpt_loss_and_scores():
    m = _gpt()
    ids = torch.randint(0, 200, (3, 16))
    labels = ids.roll(-1, 1)
    labels[1, 5:] = -100
    with torch.no_grad():
        logits = m(ids)
        assert logits.shape == (3, 16, 200) and m.vocab_padded == 256
        torch.testing.assert_close(m(ids, labels), F.cross_entropy(logits.reshape(-1, 200), labels.reshape(-1)))
        out = m.score(ids, top_k=3, temperature=2.0)
        lp = torch.log_softmax(logits[:, :-1] / 2.0, dim=-1)
        torch.testing.assert_close(out.logprobs, lp.gather(2, ids[:, 1:, None])[..., 0])
        torch.testing.assert_close(out.entropy, -(lp.exp() * lp).sum(-1))
        torch.testing.assert_close(out.top_logprobs, lp.topk(3).values)
        assert out.top_ids.shape == (3, 15, 3) and m.score(ids).top_ids is None
    assert not any(k.startswith("drop") for k in m.state_dict())


def test_a_sequence_longer_than_the_position_table_is_refused():
    with pytest.raises(ValueError):
        _gpt()(torch.zeros(1, 17, dtype=torch.long))


def test_bert_embeddings():
    torch.manual_seed(0)
    m = BertMoEForQuestionAnswering(BertMoEConfig(vocab_size=60, n_layer=1, n_head=2, d_model=32, d_ffn=64, max_position=20, moe_layers=(),
                                                  dtype=torch.float32))
    ids, tt = torch.randint(0, 60, (2, 9)), torch.randint(0, 2, (2, 9))
    seen = []
    m.ln_emb.register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
    m(ids, None, tt)
    want = F.embedding(ids, m.word.weight) + F.embedding(torch.arange(9), m.position.weight) + F.embedding(tt, m.token_type.weight)
    torch.testing.assert_close(seen[0], want)


@pytest.mark.parametrize("pre_lnorm", [False, True])
def test_transformer_xl_dropout(pre_lnorm):
    """No dropout: the model as it was. With it: masks by seed and step, none in evaluation, parameters and state dict unchanged."""
    x, y = torch.randint(0, 50, (2, 8)), torch.randint(0, 50, (2, 8))
    plain, m, again = _txl(pre_lnorm=pre_lnorm), _txl(dropout=0.3, dropout_seed=5, pre_lnorm=pre_lnorm), _txl(dropout=0.3, dropout_seed=5, pre_lnorm=pre_lnorm)
    assert list(plain.state_dict()) == list(m.state_dict())
    for other in (m, again):
        other.load_state_dict(plain.state_dict())
    with torch.no_grad():
        want = plain(x, y)[0]
        first, second = m(x, y)[0], m(x, y)[0]
        assert first != second and first != want
        assert again(x, y)[0] == first and again(x, y)[0] == second
        assert m.drop.state.tensor.tolist() == [5, 2] and m.drop.state.calls == 2 + 2 * 2      # embedding, two branches a layer, output
        torch.testing.assert_close(m.eval()(x, y)[0], want)
    loss, mems = m.train()(x, y)
    loss.backward()
    assert all(p.grad is not None for n, p in m.named_parameters()) and mems[0].shape == (2, 8, 32)
    seeds = {_txl(dropout=0.1).drop.state.tensor[0].item() for _ in range(2)}
    assert len(seeds) == 1       # drawn from torch's generator


def test_transformer_xl_loss_is_the_cross_entropy():
    m = _txl()
    x, y = torch.randint(0, 50, (2, 8)), torch.randint(0, 50, (2, 8))
    hidden, _ = m(x)
    torch.testing.assert_close(m(x, y)[0], F.cross_entropy(F.linear(hidden, m.word_emb.weight).reshape(-1, 50), y.reshape(-1)))
