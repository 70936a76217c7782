"""Gradients of tables whose ids need 64-bit keys in the sort (2^22 - 1 rows and more) and of more tokens than have their launches overlap (32768)."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(ids, dy, rows, scale, skip=None):
    """The rows that have tokens against 64 bits on the host, all others against zero."""
    from ccfuser_b200.ops.embedding import embedding_grad
    dw = embedding_grad(dy, ids, rows, scale, skip)
    again = embedding_grad(dy, ids, rows, scale, skip)
    used, place = torch.unique(ids.cpu().long(), return_inverse=True)
    ref, size, count = R.table_grad(place, dy, len(used), scale, None if skip is None else int((used == skip).nonzero()))
    assert torch.equal(dw, again)
    R.assert_close(dw[used.cuda()], ref, R.U * (count + 4) * size, "gradient")
    dw[used.cuda()] = 0
    assert not bool(dw.any())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [8, 7])
@pytest.mark.parametrize("rows", [2 ** 22 - 2, 2 ** 22 - 1, 2 ** 22 + 100])
@pytest.mark.parametrize("tokens", [5, 1000, 3000, 9500])
def test_ids_beyond_22_bits(dtype, d, rows, tokens):
    """Ids at both ends of the table, in its last rows often, and beside the number that stands for no row; one row is skipped."""
    g = torch.Generator(device="cuda").manual_seed(tokens + d)
    ids = torch.randint(0, rows, (tokens,), generator=g, device="cuda")
    ids[1::3] = rows - 1 - torch.randint(0, 3, (len(ids[1::3]),), generator=g, device="cuda")
    ids[0], ids[4] = rows - 2, 2 ** 22 - 3
    dy = torch.randn(tokens, d, generator=g, device="cuda").to(TYPES[dtype])
    _check(ids, dy, rows, 1.5)
    _check(ids, dy, rows, 1.5, rows - 2)


@pytest.mark.parametrize("tokens", [32768, 32769, 70001])
@pytest.mark.parametrize("kind", ["uniform", "one", "few", "padded"])
def test_many_tokens(tokens, kind):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    ids = torch.randint(0, {"uniform": 5000, "one": 1, "few": 7, "padded": 900}[kind], (tokens,), generator=g, device="cuda").int()
    if kind == "padded":
        ids[tokens // 4:] = 3
    dy = torch.randn(tokens, 40, generator=g, device="cuda").bfloat16()
    _check(ids, dy, 5003, 0.5, 3 if kind == "padded" else None)


@pytest.mark.parametrize("batch,seq", [(33, 1024), (3, 20000), (40000, 1)])
def test_many_tokens_in_three_tables(batch, seq):
    from ccfuser_b200.ops.embedding import embedding
    g = torch.Generator(device="cuda").manual_seed(seq)
    w, p, t = ((torch.randn(r, 16, generator=g, device="cuda") * 0.1).half().requires_grad_(True) for r in (300, seq, 2))
    ids, kinds = torch.randint(0, 300, (batch, seq), generator=g, device="cuda"), torch.randint(0, 2, (batch, seq), generator=g, device="cuda")
    dy = torch.randn(batch, seq, 16, generator=g, device="cuda").half()
    y = embedding(ids, w, 3.0, position_weight=p, type_weight=t, type_ids=kinds)
    at = torch.arange(seq).expand(batch, seq)
    ref, size = R.embedding_sum([(ids, w, 3.0), (at, p, 1.0), (kinds, t, 1.0)])
    R.assert_close(y, ref, 6 * R.U * size)
    for (i, table, s), dw in zip([(ids, w, 3.0), (at, p, 1.0), (kinds, t, 1.0)], torch.autograd.grad(y, [w, p, t], dy)):
        want, size, count = R.table_grad(i, dy, table.shape[0], s)
        R.assert_close(dw, want, R.U * (count + 4) * size, "gradient")
