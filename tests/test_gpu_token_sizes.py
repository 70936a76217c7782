"""Offsets that pass 32 bits: logits, tables and activations of more than 2^31 elements, looked at where they end. About 15 GB on the GPU."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def test_logits_beyond_32_bits():
    from ccfuser_b200.ops.logprobs import token_logprobs
    rows, width, last = 43_000, 50_001, 5
    assert rows * width > 2 ** 31
    x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(0)
    x[-last:] = torch.randn(last, width, generator=g, device="cuda").bfloat16()
    x.requires_grad_(True)
    t = torch.full((rows,), 7, device="cuda")
    t[-1] = width - 1
    out = token_logprobs(x, t, top_k=2)
    ref = R.Scores(x[-last:], t[-last:], width, 2)
    R.assert_close(out.logprobs[-last:], ref.picked, ref.of_lp(ref.picked))
    R.assert_close(out.entropy[-last:], ref.h, ref.of_h())
    assert torch.equal(out.top_ids[-last:].cpu(), ref.top_ids) and out.top_ids[0].tolist() == [0, 1]
    up = torch.zeros(rows, device="cuda")
    up[-last:] = 1.0
    dx, = torch.autograd.grad(out.logprobs, [x], up)
    want, off = ref.grad(up[-last:])
    R.assert_close(dx[-last:], want, off)
    assert not bool(dx[:-last].any())


def test_a_table_beyond_32_bits():
    from ccfuser_b200.ops.embedding import embedding
    rows, d = 70_000, 32_768
    assert rows * d > 2 ** 31
    w = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
    w[-3:] = torch.arange(3, device="cuda").bfloat16()[:, None] + 1
    w.requires_grad_(True)
    ids = torch.tensor([rows - 1, 0, rows - 3, rows - 1, rows - 2], device="cuda")
    y = embedding(ids, w, 2.0)
    assert y[:, 0].tolist() == y[:, -1].tolist() == [6, 0, 2, 6, 4]
    dw, = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert dw[-3:, -1].tolist() == dw[-3:, 0].tolist() == [2, 2, 4] and float(dw[0].float().sum()) == 2 * d
    assert not bool(dw[1:-3].any())


def test_activations_beyond_32_bits():
    from ccfuser_b200.ops.dropout import dropout
    n = 2 ** 31 + 2 ** 20 + 5
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = dropout(x, 0.5, torch.tensor([3, 4], device="cuda"), 6)
    first = (n // 8 - 100) * 8
    bits = R.philox_bits(3, 4, 6, n - first, first // 8)
    assert torch.equal(y[first:].cpu() != 0, bits >= 32768)
    bits = R.philox_bits(3, 4, 6, 800, 2 ** 28 - 50)       # around 2^31 elements
    assert torch.equal(y[2 ** 31 - 400:2 ** 31 + 400].cpu() != 0, bits >= 32768)


def test_the_widest_rows():
    from ccfuser_b200.ops.embedding import embedding, embedding_grad
    w = (torch.arange(2 ** 25, device="cuda") % 251).bfloat16().view(2, 2 ** 24)
    ids = torch.tensor([1, 0, 1], device="cuda")
    y = embedding(ids, w)
    assert torch.equal(y, w[ids])
    grad = embedding_grad(y, ids, 3)
    assert torch.equal(grad[0], w[0]) and torch.equal(grad[1], w[1] + w[1]) and not grad[2].any()
