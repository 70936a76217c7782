"""Log probabilities, entropy, alternatives and their gradient (csrc/logprobs.cu) against 64 bits, at the edges of rows, pieces, blocks and clusters."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


@pytest.fixture(autouse=True)
def _status_is_clear():
    from ccfuser_b200.ops.gemm import Workspace
    yield
    Workspace.get("cuda").check("test")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _check(x, t, vocab=None, top_k=0, temperature=1.0, seed=0, gradient=True):
    from ccfuser_b200.ops.logprobs import token_logprobs
    vocab = x.shape[-1] if vocab is None else vocab
    x = x.detach().requires_grad_(gradient)
    out = token_logprobs(x, t, top_k=top_k, temperature=temperature, vocab_size=vocab)
    ref = R.Scores(x.reshape(-1, x.shape[-1]), t.reshape(-1), vocab, top_k, temperature)
    n = t.numel()
    R.assert_close(out.logprobs.reshape(-1), ref.picked, ref.of_lp(ref.picked), "log probability")
    R.assert_close(out.entropy.reshape(-1), ref.h, ref.of_h(), "entropy")
    if top_k:
        assert torch.equal(out.top_ids.reshape(n, top_k).cpu(), ref.top_ids)
        R.assert_close(out.top_logprobs.reshape(n, top_k), torch.where(ref.top_ids < 0, -INF, ref.top), ref.of_lp(ref.top), "alternatives")
    if not gradient:
        return out, None
    g = _gen(seed + 1)
    ups = [_randn(g, *t.shape), _randn(g, *t.shape)] + ([_randn(g, *t.shape, top_k)] if top_k else [])
    dx, = torch.autograd.grad([out.logprobs, out.entropy] + ([out.top_logprobs] if top_k else []), [x], ups)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    want, off = ref.grad(ups[0].reshape(-1), ups[1].reshape(-1), ups[2].reshape(n, top_k) if top_k else None)
    R.assert_close(dx.reshape(n, -1), want, off, "gradient")
    return out, dx


# rows of one element, around a piece, at both sides of a warp's, a small and a large block's rows
SIZES = [(1, 1), (3, 2), (9, 7), (5, 8), (17, 9), (33, 100), (8, 1023), (7, 1024), (5, 1025), (3, 1031), (4, 8192), (3, 8193), (2, 50257), (1, 131072)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_sizes(dtype, rows, vocab):
    g = _gen(rows + vocab)
    x = (_randn(g, rows, vocab) * 3).to(TYPES[dtype])
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    _check(x, t)
    _check(x, t, top_k=min(vocab, 5), temperature=0.7)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,top_k", [(300, 60, 32), (2, 32, 32), (3, 3000, 32), (2, 30000, 32), (1, 30001, 20), (600, 9000, 1)])
def test_many_alternatives(dtype, rows, vocab, top_k):
    g = _gen(vocab)
    x = (_randn(g, rows, vocab) * 2).to(TYPES[dtype])
    _check(x, torch.randint(0, vocab, (rows,), generator=g, device="cuda").int(), top_k=top_k)


@pytest.mark.parametrize("vocab", [90, 1024, 4000, 20000])
@pytest.mark.parametrize("kind", ["equal", "two_values", "rising", "falling", "blocks", "zeros"])
def test_ties_go_to_the_lowest_index(kind, vocab):
    """Many equal elements, more than a block lists; whole stretches of large ones with one thread's share full of candidates; zeros of both signs."""
    place = torch.arange(vocab, device="cuda")
    row = {"equal": place * 0.0 + 1.5, "two_values": (place % 3 == 1) * 1.0, "rising": place / 64.0, "falling": -place / 64.0,
           "blocks": ((place // 8) % 512 == 5) * 2.0 + (place % 7) / 64.0, "zeros": torch.where(place % 2 == 0, -0.0, 0.0)}[kind]
    x = row.expand(3, vocab).bfloat16().contiguous()
    t = torch.tensor([0, vocab // 2, vocab - 1], device="cuda")
    _check(x, t, top_k=20)
    _check(x.float(), t, top_k=3)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [50, 1000, 5000, 40000])
def test_masks(dtype, vocab):
    """Rows masked with -inf or the type's lowest value down to three, one and no columns; targets in masked places; +inf and NaN."""
    from ccfuser_b200.ops.logprobs import token_logprobs
    dt = TYPES[dtype]
    g = _gen(vocab)
    x = _randn(g, 8, vocab).to(dt)
    allowed = torch.zeros(8, vocab, dtype=torch.bool, device="cuda")
    allowed[0, [3, vocab // 2, vocab - 1]] = True
    allowed[1, vocab // 3] = True
    allowed[3, [3, vocab // 2, vocab - 1]] = True
    allowed[4, vocab // 3] = True
    allowed[6] = True
    lowest = torch.finfo(dt).min
    fill = torch.tensor([-INF, -INF, -INF, lowest, lowest, lowest, -INF, lowest], device="cuda")[:, None]
    x = torch.where(allowed, x.float(), fill).to(dt)
    t = torch.tensor([3, vocab // 3, 1, 3, vocab // 3, 1, -100, 2], device="cuda")
    out, dx = _check(x, t, top_k=5)
    assert out.top_ids[0, 3:].tolist() == [-1, -1] and out.top_ids[1, 1:].tolist() == [-1] * 4 and out.top_ids[2].tolist() == [-1] * 5
    assert out.logprobs[2] == -INF and out.entropy[2] == 0 and not bool(dx[2].any()) and out.logprobs[6] == 0
    assert out.top_ids[5].tolist() == [0, 1, 2, 3, 4]      # nothing but the lowest value: all equal
    masked, _ = _check(x, torch.tensor([4, 0, 0, 4, 0, 0, 0, 0], device="cuda"), gradient=False)
    assert masked.logprobs[0] == -INF and masked.logprobs[1] == -INF
    x[0, vocab // 2], x[1, 7], x[3, 0] = INF, float("nan"), -float("nan")
    x.requires_grad_(True)
    out = token_logprobs(x, t, top_k=2)
    assert out.top_ids[0, 0] == vocab // 2 and out.top_ids[1, 0] == 7 and out.top_ids[3, 0] == 0
    dx, = torch.autograd.grad(out.logprobs.sum(), [x])
    for r in range(8):
        bad = r in (0, 1, 3)
        assert bool(torch.isnan(out.logprobs[r])) == bad and bool(torch.isnan(out.entropy[r])) == bad
        assert bool(torch.isnan(out.top_logprobs[r]).all()) == bad
        assert bool(torch.isnan(dx[r]).all()) == bad and bool(torch.isnan(dx[r]).any()) == bad


@pytest.mark.parametrize("vocab,width", [(3, 40), (97, 128), (1000, 1003), (9000, 9001), (50257, 50304)])
def test_columns_behind_the_vocabulary(vocab, width):
    """They hold what they like, count for nothing and get a zero."""
    g = _gen(width)
    x = _randn(g, 6, width).bfloat16()
    x[:, vocab:] = torch.tensor([INF, float("nan"), 1e30, -INF, 5.0, 0.0], device="cuda").bfloat16()[:, None]
    out, dx = _check(x, torch.randint(0, vocab, (6,), generator=g, device="cuda"), vocab=vocab, top_k=3)
    assert not bool(dx[:, vocab:].any())


def test_shapes_strides_and_alignment():
    from ccfuser_b200.ops.logprobs import token_logprobs
    g = _gen(1)
    base = _randn(g, 4, 10, 1203).bfloat16()
    t = torch.randint(0, 1100, (10, 4), generator=g, device="cuda").t()
    for x in (base, base[..., :1101], base[..., 3:], base[..., ::1].transpose(0, 1).contiguous().transpose(0, 1), base[..., 1:]):
        _check(x, t, top_k=3)
    _check(base[:, :-1], t[:, 1:])
    _check(base[::2, 0], t[::2, 0])
    _check(base[0, 0, ::3], torch.tensor(400, device="cuda"), top_k=2)
    _check(base[0, 0].expand(5, 1203), t[0, :5])
    empty = token_logprobs(base[:0], t[:0], top_k=2)
    assert empty.logprobs.shape == (0, 10) and empty.top_ids.shape == (0, 10, 2)


@pytest.mark.parametrize("function", ["C++", "Python"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_far_apart(monkeypatch, dtype, function):
    """The logits of one place of every sequence: a gradient of their own size, not of the sequences'."""
    from ccfuser_b200 import native as N
    if function == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)
    g = _gen(5)
    for seq, width, vocab in ((7, 1001, 1001), (50, 1004, 990), (3, 9003, 9000), (200, 57, 57)):
        base = (_randn(g, 5, seq, width) * 2).to(TYPES[dtype])
        t = torch.randint(0, vocab, (5,), generator=g, device="cuda")
        _, dx = _check(base[:, 0], t, vocab, top_k=2)
        assert dx.stride(0) < width + 8 and dx.untyped_storage().nbytes() <= 5 * (width + 7) * dx.element_size()


def test_each_gradient_alone_and_rows_without_one():
    from ccfuser_b200.ops.logprobs import token_logprobs
    g = _gen(2)
    x = _randn(g, 5, 3000).requires_grad_(True)
    t = torch.tensor([3, -100, 2999, 0, 8], device="cuda")
    ref = R.Scores(x, t, 3000, 4)
    ups = [_randn(g, 5), _randn(g, 5), _randn(g, 5, 4)]
    ups[0][3] = ups[1][3] = 0
    ups[2][3] = 0
    for i, name in enumerate(("logprobs", "entropy", "top_logprobs")):
        dx, = torch.autograd.grad(getattr(token_logprobs(x, t, top_k=4), name), [x], ups[i])
        want, off = ref.grad(*[ups[i] if j == i else None for j in range(3)])
        R.assert_close(dx, want, off, name)
        assert not bool(dx[3].any())
    dx, = torch.autograd.grad(token_logprobs(x, t).logprobs.mean(), [x])
    want, off = ref.grad(torch.full((5,), 0.2))
    R.assert_close(dx, want, off)
    assert not bool(dx[1].any())


def test_a_kernel_gradient_is_that_of_differences():
    from ccfuser_b200.ops.logprobs import token_logprobs
    x, t = torch.randn(2, 40, generator=torch.Generator().manual_seed(0)).cuda(), torch.tensor([3, 39], device="cuda")
    x.requires_grad_(True)

    def value(y):
        r = token_logprobs(y, t, temperature=2.0)
        return (r.logprobs.double() * 2 - r.entropy.double()).sum()
    dx, = torch.autograd.grad(value(x), [x])
    step = 2.0 ** -6      # fp32 values of about 8 with 2^-20: differences good to 2^-20 / 2^-5, and the third derivative's part below 2^-12 / 6
    for i, j in ((0, 3), (0, 0), (1, 39), (1, 7)):
        up, down = x.detach().clone(), x.detach().clone()
        up[i, j] += step
        down[i, j] -= step
        assert abs(float(value(up) - value(down)) / (2 * step) - float(dx[i, j])) < 2.0 ** -12


def test_targets_out_of_range_are_reported():
    from ccfuser_b200 import TokenIndexError
    from ccfuser_b200.ops.gemm import Workspace
    from ccfuser_b200.ops.logprobs import token_logprobs
    x = torch.zeros(4, 2000, device="cuda").requires_grad_(True)
    for bad in (-1, 1990, 2 ** 40):
        out = token_logprobs(x, torch.tensor([1, bad, 5, -100], device="cuda"), vocab_size=1990)
        with pytest.raises(TokenIndexError, match="token 1"):
            Workspace.get("cuda").check("test")
        assert torch.isnan(out.logprobs).tolist() == [False, True, False, False]
        dx, = torch.autograd.grad(out.logprobs, [x], torch.ones(4, device="cuda"))
        assert not bool(dx[[1, 3]].any()) and bool(dx[0].any())


def test_python_function_gives_the_same_bits(monkeypatch):
    from ccfuser_b200 import native as N
    g = _gen(4)
    x, t = _randn(g, 50, 1234).half(), torch.randint(0, 1200, (50,), generator=g, device="cuda")
    one = _check(x, t, vocab=1201, top_k=7, temperature=1.7)
    monkeypatch.setattr(N, "torch_module", lambda: None)
    two = _check(x, t, vocab=1201, top_k=7, temperature=1.7)
    assert all(torch.equal(a, b) for a, b in zip(one[0], two[0])) and torch.equal(one[1], two[1])


def test_a_gradient_is_not_differentiated_again():
    from ccfuser_b200.ops.logprobs import token_logprobs
    x = torch.randn(3, 50, device="cuda").requires_grad_(True)
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(token_logprobs(x, torch.arange(3, device="cuda")).logprobs.square().sum(), [x], create_graph=True)
        d.sum().backward()


def test_an_input_changed_in_between_is_noticed():
    from ccfuser_b200.ops.logprobs import token_logprobs
    w = torch.randn(3, 50, device="cuda").requires_grad_(True)
    x = w * 2
    out = token_logprobs(x, torch.arange(3, device="cuda"))
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        out.logprobs.sum().backward()
    x = (w * 2)[None]                       # seen as rows by a view
    out = token_logprobs(x, torch.arange(3, device="cuda")[None])
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        out.logprobs.sum().backward()


def test_other_streams_and_a_captured_step():
    from ccfuser_b200.ops.logprobs import token_logprobs
    g = _gen(6)
    x = _randn(g, 20, 30011).bfloat16().requires_grad_(True)
    t = torch.randint(0, 30011, (20,), generator=g, device="cuda")

    def step():
        out = token_logprobs(x, t, top_k=4)
        d, = torch.autograd.grad(out.logprobs.mean() + 0.1 * out.entropy.sum(), [x])
        return [o.detach() for o in out], d      # an eager graph that stays alive would tie a captured backward pass of the same leaf to its stream
    ref = step()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got.append(step())
    graph.replay()
    torch.cuda.synchronize()
    for out, d in got:
        assert all(torch.equal(a, b) for a, b in zip(out, ref[0])) and torch.equal(d, ref[1])
