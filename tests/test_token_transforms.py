"""Transforms of torch.func, forward mode and second derivatives through whole models, in fp32 on a GPU and on the host, against fp64 on the host."""
import pytest
import torch
from torch.nn.attention import SDPBackend, sdpa_kernel

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# fp32 through two layers of matrix products of at most 64 terms: 2^-24 of the magnitudes for each of a few thousand dependent operations at most, twice
# that many where a derivative is taken again
TOL = 2.0 ** -24 * 8192


def _model(name, dtype, device):
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    torch.manual_seed(0)
    if name == "gpt":
        m = GPTMoE(GPTMoEConfig(vocab_size=50, n_layer=2, n_head=2, d_model=32, d_ffn=64, seq_len=8, moe_every=0, dtype=dtype))
    else:
        m = TransformerXLMoE(TransformerXLMoEConfig(n_token=50, n_layer=2, n_head=2, d_model=32, d_head=16, d_inner=64, tgt_len=8, mem_len=0, moe=False,
                                                    dtype=dtype))
    for p in m.parameters():         # of a size that shows
        with torch.no_grad():
            p.add_(torch.randn(p.shape, dtype=torch.float64).to(p.dtype) * 0.1)
    x, y = torch.randint(0, 50, (4, 8)), torch.randint(0, 50, (4, 8))
    y[1, 3:] = -100
    tangents = {k: torch.randn(p.shape, dtype=torch.float64).to(p.dtype) for k, p in m.named_parameters()}
    return m.to(device), x.to(device), y.to(device), {k: t.to(device) for k, t in tangents.items()}


def _loss(m, x, y, params=None):
    out = m(x, y) if params is None else torch.func.functional_call(m, params, (x, y))
    return out[0] if isinstance(out, tuple) else out


def _calls(m, x, y, tangents):
    params = dict(m.named_parameters())
    tables = [n for n in params if n in ("wte.weight", "wpe.weight", "word_emb.weight")]

    def one(p, a, b):
        return _loss(m, a[None], b[None], {**params, **p})

    def twice():
        grads = torch.autograd.grad(_loss(m, x, y), list(params.values()), create_graph=True)
        return [*grads, *torch.autograd.grad(sum((g * t).sum() for g, t in zip(grads, tangents.values())), list(params.values()))]
    subset = {n: params[n] for n in tables}
    return {"grad": lambda: list(torch.func.grad(one)(subset, x[0], y[0]).values()),
            "vmap": lambda: list(torch.func.vmap(torch.func.grad(one), in_dims=(None, 0, 0))(subset, x, y).values()),
            "jvp": lambda: list(torch.func.jvp(lambda p: _loss(m, x, y, p), (params,), (tangents,))),
            "twice": twice}


@pytest.mark.parametrize("function", ["C++", "Python"])
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", ["grad", "vmap", "jvp", "twice"])
@pytest.mark.parametrize("name", ["gpt", "txl"])
def test_derivatives(monkeypatch, name, what, device, function):
    from ccfuser_b200 import native as N
    if function == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)
    with sdpa_kernel(SDPBackend.MATH):
        m, *args = _model(name, torch.float32, device)
        got = _calls(m, *args)[what]()
        ref = _model(name, torch.float64, "cpu")[0]
        ref.load_state_dict(m.state_dict())
        x, y, tangents = args
        wants = _calls(ref, x.cpu(), y.cpu(), {k: t.double().cpu() for k, t in tangents.items()})[what]()
    if what == "twice":              # first and second derivatives apart
        assert len(got) == len(wants) == 2 * len(list(m.parameters()))
    for part in (slice(0, len(got) // 2), slice(len(got) // 2, None)) if what == "twice" else (slice(None),):
        largest = max(float(w.norm()) for w in wants[part])
        assert largest > 0
        for g, w in zip(got[part], wants[part]):
            assert float((g.detach().double().cpu() - w.detach()).norm()) <= TOL * largest


@pytest.mark.gpu
@pytest.mark.parametrize("function", ["C++", "Python"])
def test_what_counts_for_nothing_counts_for_nothing_again(monkeypatch, function):
    """Ignored targets, columns behind the vocabulary, rows without a finite logit, the padding row, positions of several sequences: the gradient that can be
    differentiated is the kernels', and so is its derivative that of the formula."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.embedding import Embedding
    from ccfuser_b200.ops.logprobs import cross_entropy
    if function == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)
    torch.manual_seed(0)
    table = Embedding(20, 24, padding_idx=3, scale=2.0, device="cuda")
    place, kind = (torch.randn(r, 24, device="cuda", requires_grad=True) for r in (9, 2))
    ids, kinds = torch.randint(0, 20, (3, 7), device="cuda"), torch.randint(0, 2, (3, 7), device="cuda").int()
    ids[0, :4] = 3
    targets = torch.randint(0, 21, (3, 7), device="cuda")
    targets[1, 2:5] = -100
    mask = torch.zeros(3, 7, 24, device="cuda")
    mask[2, 1], mask[2, 3, ::2] = -float("inf"), -float("inf")
    targets[2, 1] = -100
    targets[2, 3] = 1
    leaves = [table.weight, place, kind]

    def loss(again):
        x = table(ids, position_weight=place, type_weight=kind, type_ids=kinds) + mask
        value = cross_entropy(x, targets, vocab_size=21)
        return torch.autograd.grad(value, leaves, create_graph=again)
    plain, first = loss(False), loss(True)
    ups = [torch.randn_like(g) for g in first]
    second = torch.autograd.grad(sum((g * u).sum() for g, u in zip(first, ups)), leaves)
    # the same in fp64 by torch's functions
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    x = torch.nn.functional.embedding(ids, wide[0], 3) * 2.0 + wide[1][:7] + wide[2][kinds.long()]
    live = targets != -100
    x, rows = (x + mask.double())[..., :21][live], targets[live]
    value = torch.nn.functional.cross_entropy(x, rows)
    want = torch.autograd.grad(value, wide, create_graph=True)
    want2 = torch.autograd.grad(sum((g * u.double()).sum() for g, u in zip(want, ups)), wide)
    for a, b, c in zip(plain, first, want):
        torch.testing.assert_close(a, b, rtol=2.0 ** -18, atol=2.0 ** -24 * 64)
        torch.testing.assert_close(b.double(), c, rtol=2.0 ** -18, atol=2.0 ** -24 * 64)
    for b, c in zip(second, want2):
        torch.testing.assert_close(b.double(), c, rtol=2.0 ** -16, atol=2.0 ** -24 * 256)
    assert not bool(first[0][3].any())


def _small(name, device):
    m, x, y, _ = _model(name, torch.float32, device)
    return m, x, y


@pytest.mark.parametrize("name", ["gpt", "txl"])
@pytest.mark.parametrize("device", ["meta", *DEVICES])
def test_without_memory(name, device):
    """Shapes alone: the meta device and fake tensors, forward and backward."""
    import contextlib

    from torch._subclasses.fake_tensor import FakeTensorMode
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    with contextlib.nullcontext() if device == "meta" else FakeTensorMode():      # where a module cannot be moved
        if name == "gpt":
            m = GPTMoE(GPTMoEConfig(vocab_size=50, n_layer=1, n_head=2, d_model=32, d_ffn=64, seq_len=8, moe_every=0, dtype=torch.float32), device=device)
        else:
            m = TransformerXLMoE(TransformerXLMoEConfig(n_token=50, n_layer=1, n_head=2, d_model=32, d_head=16, d_inner=64, tgt_len=8, mem_len=8, moe=False,
                                                        dtype=torch.float32), device=device)
        x = torch.zeros(4, 8, dtype=torch.long, device=device)
        loss = _loss(m, x, x)
        loss.backward()
    assert loss.shape == () and loss.device.type == device
    assert all(p.grad is not None and p.grad.shape == p.shape for p in m.parameters())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", ["compile", "export", "make_fx"])
def test_graphs_of_a_whole_model(how, device):
    """One graph of a step's loss, which gives on other inputs what the model gives."""
    m, x, y = _small("gpt", device)
    u, v = y.clamp_min(0), x.roll(1, 1)
    with torch.no_grad():
        if how == "compile":
            f = torch.compile(m, backend="eager", fullgraph=True)
            f(x, y)
        elif how == "export":
            f = torch.export.export(m, (x, y)).module()
        else:
            from torch.fx.experimental.proxy_tensor import make_fx
            f = make_fx(lambda a, b: m(a, b), tracing_mode="real")(x, y)
        want = m(u, v)
        assert abs(float(f(u, v)) - float(want)) <= TOL * float(want)


@pytest.mark.gpu
def test_kernels_serve_what_is_not_transformed():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.logprobs import cross_entropy
    m, x, _ = _small("gpt", "cuda")
    before = N.LAUNCHES[0]
    y = m.wte(x, position_weight=m.wpe.weight)
    loss = cross_entropy(y, x % 32)
    assert y.grad_fn.name() == "CcfEmbeddingBackward" and N.LAUNCHES[0] == before + 2
    loss.backward()
    assert m.wte.weight.grad is not None
    with FakeTensorMode(), pytest.raises(Exception):
        torch.zeros(3, device="cuda").tolist()
    assert not N.transformed(m.wte.weight) and not N.transformed(y)
