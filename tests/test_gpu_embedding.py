"""Embedding sums and their gradients (csrc/embedding.cu) against sums in 64 bits, at the edges of vectors, sorted chunks, pieces and joined runs."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _status_is_clear():
    from ccfuser_b200.ops.gemm import Workspace
    yield
    Workspace.get("cuda").check("test")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dt, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)


def _check(ids, w, scale, dy, y, dw, skip=None):
    ref, size, count = R.table_grad(ids, dy, w.shape[0], scale, skip)
    R.assert_close(dw, ref, R.U * (count + 4) * size, "gradient")


def _run(ids, w, scale=1.0, dy=None, padding_idx=None, **kw):
    from ccfuser_b200.ops.embedding import embedding
    tables = [w] + [kw[k] for k in ("position_weight", "type_weight") if k in kw]
    for t in tables:
        t.requires_grad_(True)
    y = embedding(ids, w, scale, padding_idx=padding_idx, **kw)
    return y, torch.autograd.grad(y, tables, dy)


# tokens: one, a piece and around it, a sorted chunk and around it, several chunks; d: off and on 16 bytes, beyond one slice of a warp
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,rows,d", [(1, 1, 1), (1, 40, 8), (7, 3, 17), (8, 3, 64), (9, 100, 200), (33, 2, 1000), (1023, 5, 24), (1024, 700, 256), (1025, 1, 8),
                                           (2049, 33, 264), (5000, 64, 513), (6145, 6145, 40),
                                           (8192, 90, 16), (8193, 5, 24), (17000, 3000, 8)])
def test_sizes(dtype, tokens, rows, d):
    g, dt = _gen(tokens + d), TYPES[dtype]
    w, dy = _randn(g, dt, rows, d, std=0.05), _randn(g, dt, tokens, d)
    ids = torch.randint(0, rows, (tokens,), generator=g, device="cuda")
    y, (dw,) = _run(ids, w, 3.7, dy)
    ref, size = R.embedding_sum([(ids, w, 3.7)])
    R.assert_close(y, ref, 4 * R.U * size)
    _check(ids, w, 3.7, dy, y, dw)


@pytest.mark.parametrize("kind", ["one", "two", "first_and_last", "sorted", "reversed", "runs"])
@pytest.mark.parametrize("tokens", [31, 640, 4500, 9000])
def test_orders_of_ids(kind, tokens):
    """One word for all tokens, runs that begin and end inside, at and across pieces."""
    g, rows = _gen(tokens), 65
    place = torch.arange(tokens, device="cuda")
    ids = {"one": place * 0 + 64, "two": (place % 2) * 40, "first_and_last": torch.where(place % 3 == 0, 0, 64),
           "sorted": place * rows // tokens, "reversed": rows - 1 - place * rows // tokens, "runs": (place // 13) % rows}[kind].int()
    w, dy = _randn(g, torch.bfloat16, rows, 72), _randn(g, torch.bfloat16, tokens, 72)
    y, (dw,) = _run(ids, w, 0.5, dy)
    _check(ids, w, 0.5, dy, y, dw)
    again = _run(ids, w, 0.5, dy)[1][0]
    assert torch.equal(dw, again)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("batch,seq,d,given", [(1, 1, 8, False), (5, 37, 136, False), (3, 700, 33, True), (40, 3, 768, False), (2100, 1, 16, False)])
def test_three_tables(dtype, batch, seq, d, given):
    """Word, position and type table, the padding word without a gradient; positions by place and given (also one row for all)."""
    g, dt = _gen(seq), TYPES[dtype]
    w, p, t = (_randn(g, dt, r, d, std=0.1) for r in (50, max(seq, 64), 2))
    ids = torch.randint(0, 50, (batch, seq), generator=g, device="cuda")
    ids[:, seq // 2:] = 7
    types = (torch.rand(batch, seq, generator=g, device="cuda") < 0.3).long()
    places = torch.arange(seq, device="cuda")
    pos = torch.randperm(max(seq, 64), generator=g, device="cuda")[:seq] if given else None
    dy = _randn(g, dt, batch, seq, d)
    y, grads = _run(ids, w, 22.6, dy, padding_idx=7, position_weight=p, position_ids=pos, type_weight=t, type_ids=types)
    at = (pos if given else places).expand(batch, seq)
    ref, size = R.embedding_sum([(ids, w, 22.6), (at, p, 1.0), (types, t, 1.0)])
    R.assert_close(y, ref, 6 * R.U * size)
    for (i, table, s, skip), dw in zip([(ids, w, 22.6, 7), (at, p, 1.0, None), (types, t, 1.0, None)], grads):
        _check(i, table, s, dy, y, dw, skip)
    assert not bool(grads[0][7].any())


def test_a_table_without_a_gradient_and_hooks():
    from ccfuser_b200.ops.embedding import Embedding, embedding, embedding_grad
    g = _gen(3)
    w, p = _randn(g, torch.bfloat16, 40, 64), _randn(g, torch.bfloat16, 9, 64).requires_grad_(True)
    ids, dy = torch.randint(0, 40, (6, 9), generator=g, device="cuda"), _randn(g, torch.bfloat16, 6, 9, 64)
    y = embedding(ids, w, position_weight=p)
    dp, = torch.autograd.grad(y, [p], dy)
    _check(torch.arange(9).expand(6, 9), p, 1.0, dy, y, dp)
    m = Embedding(40, 64, padding_idx=3, scale=2.0, device="cuda", dtype=torch.bfloat16)
    m.load_state_dict({"weight": w})
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        z = m(ids)
    z.backward(dy)
    assert torch.equal(m.weight.grad, embedding_grad(dy, ids, 40, 2.0, 3))
    assert torch.equal(z, embedding(ids, w, 2.0))
    with torch.no_grad():
        assert not embedding(ids, m.weight).requires_grad


@pytest.mark.parametrize("d", [64, 63])
def test_strides_and_alignment(d):
    """Rows of a wider table, a table that is a transposed matrix, ids and gradients with strides, memory off a 16-byte boundary."""
    from ccfuser_b200.ops.embedding import embedding, embedding_grad
    g = _gen(d)
    wide = _randn(g, torch.bfloat16, 30, 100)
    ids = torch.randint(0, 30, (14, 10), generator=g, device="cuda").t()[::2]
    dy = _randn(g, torch.bfloat16, 14, 5, d + 1).transpose(0, 1)[..., 1:]
    for w in (wide[:, :d], wide[::3, 5:5 + d], _randn(g, torch.bfloat16, d, 30).t(), wide.reshape(-1)[1:1 + 30 * d].view(30, d)):
        i = ids % w.shape[0]
        w.requires_grad_(True)
        y = embedding(i, w, 1.5)
        ref, size = R.embedding_sum([(i, w, 1.5)])
        R.assert_close(y, ref, 4 * R.U * size)
        dw, = torch.autograd.grad(y, [w], dy)
        _check(i, w, 1.5, dy, y, dw)
        assert torch.equal(dw, embedding_grad(dy, i, w.shape[0], 1.5))
    same = torch.ones(1, 1, d, device="cuda", dtype=torch.bfloat16).expand(5, 14, d)       # what .sum() hands back
    dw = embedding_grad(same, ids, 30)
    assert torch.equal(dw.float(), torch.bincount(ids.reshape(-1), minlength=30)[:, None].float().expand(30, d).bfloat16().float())


def test_rows_behind_the_last_token_and_many_rows():
    """A vocabulary of more rows than any block writes, of which the tokens use the first, the last and one between; every other row is zero."""
    from ccfuser_b200.ops.embedding import embedding_grad
    rows = 100_003
    ids = torch.tensor([0, rows - 1, 51_234, rows - 1], device="cuda", dtype=torch.int32)
    dy = torch.ones(4, 8, device="cuda", dtype=torch.float16)
    dw = embedding_grad(dy, ids, rows, 2.0)
    ref = torch.zeros(rows, 8, device="cuda", dtype=torch.float16)
    ref[0], ref[rows - 1], ref[51_234] = 2, 4, 2
    assert torch.equal(dw, ref)


def test_ids_out_of_range_are_reported():
    from ccfuser_b200 import TokenIndexError
    from ccfuser_b200.ops.embedding import embedding
    from ccfuser_b200.ops.gemm import Workspace
    w = torch.ones(10, 16, device="cuda").requires_grad_(True)
    for bad in (-1, 10, 2 ** 40, -2 ** 63):
        ids = torch.tensor([1, 2, bad, 3], device="cuda")
        y = embedding(ids, w)
        with pytest.raises(TokenIndexError, match="token 2"):
            Workspace.get("cuda").check("test")
        assert bool(torch.isnan(y[2]).all()) and bool((y[[0, 1, 3]] == 1).all())
        dw, = torch.autograd.grad(y, [w], torch.ones_like(y))
        with pytest.raises(IndexError, match="token 2"):
            Workspace.get("cuda").check("test")
        assert dw.sum(dim=1).tolist() == [0, 16, 16, 16] + [0] * 6
    with pytest.raises(ValueError):
        embedding(torch.zeros(1, 11, dtype=torch.long, device="cuda"), w, position_weight=w)
    with pytest.raises(ValueError):
        embedding(torch.zeros(1, 3, dtype=torch.long), w)


def test_a_gradient_is_not_differentiated_again():
    from ccfuser_b200.ops.embedding import embedding
    w = torch.ones(10, 16, device="cuda").requires_grad_(True)
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(embedding(torch.arange(4, device="cuda"), w).square().sum(), [w], create_graph=True)
        d.sum().backward()


def test_python_function_gives_the_same_bits(monkeypatch):
    from ccfuser_b200 import native as N
    g = _gen(5)
    w, p, t = (_randn(g, torch.float16, r, 96) for r in (300, 50, 2))
    ids, types = torch.randint(0, 300, (60, 50), generator=g, device="cuda"), torch.randint(0, 2, (60, 50), generator=g, device="cuda").int()
    dy = _randn(g, torch.float16, 60, 50, 96)
    kw = dict(position_weight=p, type_weight=t, type_ids=types)
    before = N.LAUNCHES[0]
    y, grads = _run(ids, w, 2.0, dy, **kw)
    launches = N.LAUNCHES[0] - before
    monkeypatch.setattr(N, "torch_module", lambda: None)
    before = N.LAUNCHES[0]
    z, others = _run(ids, w, 2.0, dy, **kw)
    assert launches == N.LAUNCHES[0] - before == 4
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(grads, others))


def test_other_streams_and_a_captured_step():
    from ccfuser_b200.ops.embedding import embedding
    g = _gen(6)
    w, ids = _randn(g, torch.bfloat16, 200, 128).requires_grad_(True), torch.randint(0, 200, (4000,), generator=g, device="cuda")
    dy = _randn(g, torch.bfloat16, 4000, 128)

    def step(i):        # nothing of the eager graph stays alive: it would tie a captured backward pass of the same leaf to its stream
        y = embedding(i, w)
        return y.detach(), torch.autograd.grad(y, [w], dy)[0]
    ref_y, ref_d = step(ids)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step(ids))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref_y) and torch.equal(d, ref_d) for y, d in got)
    static = ids.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, d = step(static)
        graphs.append((graph, y, d))
    for shift in (0, 1, 7):
        static.copy_(ids.roll(shift))
        want = step(static)[1]
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, y, d in graphs:
            assert torch.equal(d, want) and torch.equal(y, ref_y.roll(shift, 0))
