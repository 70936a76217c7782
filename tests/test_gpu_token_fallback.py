"""Models on a GPU whose embeddings and losses the kernels do not take: torch's operations serve them, as before the kernels."""
import pytest
import torch
from test_gpu_token_step import _step

pytestmark = pytest.mark.gpu


def _models(dtype, device, dropout=0.0):
    """Each model with the arguments of a step."""
    from ccfuser_b200.models.bert_moe import BertMoEConfig, BertMoEForQuestionAnswering
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    torch.manual_seed(0)
    ids, labels, two = torch.randint(0, 50, (3, 8)), torch.randint(0, 50, (3, 8)), torch.randint(0, 2, (3, 8))
    labels[1, 5:] = -100
    gpt = GPTMoE(GPTMoEConfig(vocab_size=50, n_layer=1, n_head=2, d_model=32, d_ffn=64, seq_len=8, moe_every=0, dtype=dtype))
    bert = BertMoEForQuestionAnswering(BertMoEConfig(vocab_size=60, n_layer=1, n_head=2, d_model=32, d_ffn=64, max_position=40, moe_layers=(), dtype=dtype))
    txl = TransformerXLMoE(TransformerXLMoEConfig(n_token=50, n_layer=1, n_head=2, d_model=32, d_head=16, d_inner=64, tgt_len=8, mem_len=8, moe=False,
                                                  dtype=dtype, dropout=dropout, dropout_seed=3))
    args = {"gpt": (gpt, (ids, labels)), "bert": (bert, (ids, torch.ones_like(ids), two, ids[:, 0] % 8, ids[:, 1] % 8)), "txl": (txl, (ids, ids.roll(1, 1)))}
    return {k: (m.to(device), [a.to(device) for a in v]) for k, (m, v) in args.items()}


@pytest.mark.parametrize("name", ["gpt", "bert", "txl"])
def test_fp64_models(name):
    """Against the same on the host. In fp32 on both sides are BERT's span loss and Transformer-XL's sines and cosines of positions, which differ by up to two steps
    (2^-22) between the host's functions and the GPU's and enter its scores through weights of 0.02; all else is in fp64."""
    m, args = _models(torch.float64, "cuda", 0.25)[name]
    ref, ref_args = _models(torch.float64, "cpu", 0.25)[name]
    ref.load_state_dict(m.state_dict())
    loss, grads = _step(m, args)
    want, wants = _step(ref, ref_args)
    tol = 1e-12 if name == "gpt" else 2.0 ** -20
    assert abs(float(loss) - float(want)) <= tol * abs(float(want))
    largest = max(float(w.norm()) for w in wants)
    for g, w in zip(grads, wants):
        assert g.dtype == torch.float64 and float((g.cpu() - w).norm()) <= tol * largest


def test_more_tokens_than_the_kernels_take(monkeypatch):
    from ccfuser_b200.ops import embedding as E
    torch.manual_seed(0)
    m = E.Embedding(30, 16, padding_idx=3, scale=2.0, device="cuda")
    p = torch.randn(9, 16, device="cuda", requires_grad=True)
    ids = torch.randint(0, 30, (5, 7), device="cuda")
    want = m(ids, position_weight=p)
    grads = torch.autograd.grad(want.sum(), [m.weight, p])
    monkeypatch.setattr(E, "MAX_TOKENS", 34)
    got = m(ids, position_weight=p)
    assert "Ccf" not in got.grad_fn.name()
    # a product and a sum, each rounded, against one rounding of both: half a step of each
    torch.testing.assert_close(got, want, rtol=2.0 ** -22, atol=2.0 ** -22)
    for a, b in zip(torch.autograd.grad(got.sum(), [m.weight, p]), grads):
        assert torch.equal(a, b)                 # sums of ones, times two
    with pytest.raises(ValueError):              # refusals stand in front
        m(ids, position_weight=p[:6])
