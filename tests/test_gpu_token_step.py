"""Embedding, dropout and log probabilities together, as the models run them: whole steps against 64 bits on the host, captured and replayed, and
through the fused layers."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(m, args):
    for p in m.parameters():
        p.grad = None
    out = m(*args)
    loss = out[0] if isinstance(out, tuple) else out
    loss.backward()
    return loss.detach(), [p.grad for p in m.parameters()]


def _near(a, b, tol, of=0.0):
    a, b = a.double().cpu(), b.double().cpu()
    assert float((a - b).norm()) <= tol * max(float(b.norm()), of), (float((a - b).norm()), float(b.norm()))


def _all_near(m, grads, wants):
    """The tables' gradients relative to themselves. The others relative to the largest: a key bias adds the same to all of a row's scores, so its
    gradient is zero by the formula, a sum over p_j (d_j - sum_i p_i d_i) whose terms, of the size of the other gradients, cancel; what fp32 leaves of it is
    2^-24 of those terms and nothing of the sum."""
    largest = max(float(w.norm()) for w in wants)
    for (name, _), g, w in zip(m.named_parameters(), grads, wants):
        table = any(name.startswith(t) for t in ("wte", "wpe", "word", "position", "token_type"))
        _near(g, w, TOL, 0.0 if table else largest)


# fp32 through two layers of matrix products of at most 64 terms: 2^-24 of the magnitudes for each of a few thousand dependent operations at most
TOL = 2.0 ** -24 * 4096


def test_gpt_step_against_64_bits():
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    torch.manual_seed(0)
    kw = dict(vocab_size=203, n_layer=2, n_head=2, d_model=32, d_ffn=64, seq_len=24, moe_every=0)
    ref = GPTMoE(GPTMoEConfig(dtype=torch.float64, **kw))
    m = GPTMoE(GPTMoEConfig(dtype=torch.float32, **kw), device="cuda")
    m.load_state_dict(ref.state_dict())
    ids = torch.randint(0, 203, (5, 23))
    labels = ids.roll(-1, 1)
    labels[:, -1] = -100
    loss, grads = _step(m, (ids.cuda(), labels.cuda()))
    want, wants = _step(ref, (ids, labels))
    _near(loss, want, TOL)
    _all_near(m, grads, wants)
    with torch.no_grad():
        a, b = m.score(ids.cuda(), top_k=4), ref.score(ids, top_k=4)
    for x, y in zip(a[:3], b[:3]):
        _near(x, y, TOL)
    assert torch.equal(a.top_ids.cpu(), b.top_ids)


@pytest.mark.parametrize("pre_lnorm", [False, True])
def test_transformer_xl_steps_against_64_bits(pre_lnorm):
    """Two steps with memory and dropout: the host's whole-number masks are the kernel's."""
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    torch.manual_seed(0)
    kw = dict(n_token=50, n_layer=2, n_head=2, d_model=32, d_head=16, d_inner=64, tgt_len=12, mem_len=12, moe=False, dropout=0.25, dropout_seed=9,
              pre_lnorm=pre_lnorm)
    ref = TransformerXLMoE(TransformerXLMoEConfig(dtype=torch.float64, **kw))
    m = TransformerXLMoE(TransformerXLMoEConfig(dtype=torch.float32, **kw), device="cuda")
    m.load_state_dict(ref.state_dict())
    mems, ref_mems = None, None
    for _ in range(2):
        x, y = torch.randint(0, 50, (3, 12)), torch.randint(0, 50, (3, 12))
        loss, grads = _step(m, (x.cuda(), y.cuda(), mems))
        want, wants = _step(ref, (x, y, ref_mems))
        _near(loss, want, TOL)
        _all_near(m, grads, wants)
        with torch.no_grad():
            m.drop.state.tensor[1] -= 1           # the same step's masks once more, for the memories
            ref.drop.state.tensor[1] -= 1
            mems, ref_mems = m(x.cuda(), y.cuda(), mems)[1], ref(x, y, ref_mems)[1]


def test_bert_embeddings_against_64_bits():
    from ccfuser_b200.models.bert_moe import BertMoEConfig, BertMoEForQuestionAnswering
    torch.manual_seed(0)
    kw = dict(vocab_size=60, n_layer=1, n_head=2, d_model=32, d_ffn=64, max_position=40, moe_layers=())
    ref = BertMoEForQuestionAnswering(BertMoEConfig(dtype=torch.float64, **kw))
    m = BertMoEForQuestionAnswering(BertMoEConfig(dtype=torch.float32, **kw), device="cuda")
    m.load_state_dict(ref.state_dict())
    ids, mask = torch.randint(0, 60, (4, 33)), torch.ones(4, 33, dtype=torch.long)
    mask[1, 20:] = 0
    tt, st, en = torch.randint(0, 2, (4, 33)), torch.randint(0, 20, (4,)), torch.randint(0, 20, (4,))
    loss, grads = _step(m, [t.cuda() for t in (ids, mask, tt, st, en)])
    # the host's logits are taken to fp32 in front of its loss: 2^-24 of them
    want, wants = _step(ref, [ids, mask, tt, st, en])
    _near(loss, want, TOL)
    _all_near(m, grads, wants)


def test_a_captured_step_trains_like_an_eager_one():
    """Embedding, dropout, log probabilities and their backward passes in one graph: replays give the bits of eager steps, new masks every time."""
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    torch.manual_seed(0)
    c = TransformerXLMoEConfig(n_token=97, n_layer=2, n_head=2, d_model=64, d_head=32, d_inner=128, tgt_len=48, mem_len=0, moe=False, dropout=0.2,
                               dropout_seed=3, dtype=torch.bfloat16)
    m = TransformerXLMoE(c, device="cuda")
    twin = copy.deepcopy(m)
    batches = [(torch.randint(0, 97, (8, 48), device="cuda"), torch.randint(0, 97, (8, 48), device="cuda")) for _ in range(3)]
    x, y = batches[0][0].clone(), batches[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(m, (x, y))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = _step(m, (x, y))
    for _ in range(2):
        twin.drop.state.advance()
    losses = []
    for a, b in batches:
        x.copy_(a)
        y.copy_(b)
        graph.replay()
        want, wants = _step(twin, (a, b))
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and all(torch.equal(g, w) for g, w in zip(grads, wants))
        losses.append(float(loss))
    assert m.drop.state.tensor.tolist() == twin.drop.state.tensor.tolist() == [3, 5]
    x.copy_(batches[0][0])
    y.copy_(batches[0][1])
    graph.replay()
    torch.cuda.synchronize()
    assert float(loss) != losses[0]            # the same batch under other masks


def test_through_the_fused_layers():
    """A Transformer-XL step with MoE layers and dropout on the fused backend, and a GPT step whose loss is that of its own logits."""
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.models.transformer_xl_moe import TransformerXLMoE, TransformerXLMoEConfig
    torch.manual_seed(0)
    m = TransformerXLMoE(TransformerXLMoEConfig(n_layer=2, n_head=4, d_model=256, d_head=64, d_inner=512, tgt_len=64, mem_len=64, num_experts=8,
                                                backend="fused", max_tokens=4 * 64, dropout=0.1), device="cuda")
    x, y = torch.randint(1, 50, (4, 64), device="cuda"), torch.randint(1, 50, (4, 64), device="cuda")
    mems = None
    for _ in range(3):
        m.zero_grad(set_to_none=True)
        loss, mems = m(x, y, mems)
        loss.backward()
        assert bool(torch.isfinite(loss)) and all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())
    m.moe_layers()[0].check_status()
    g = GPTMoE(GPTMoEConfig(vocab_size=1000, n_layer=2, n_head=4, d_model=256, d_ffn=512, seq_len=128, num_experts=8, max_tokens=512,
                            backend="fused"), device="cuda")
    ids = torch.randint(0, 1000, (4, 128), device="cuda")
    with torch.no_grad():
        logits = g(ids).float()
        loss, scores = g(ids, ids.roll(-1, 1)), g.score(ids, top_k=2)
    want = torch.nn.functional.cross_entropy(logits.reshape(-1, 1000).double(), ids.roll(-1, 1).reshape(-1))
    assert abs(float(loss) - float(want)) <= 2.0 ** -24 * 256 * (1 + float(want))
    assert torch.equal(scores.top_ids[..., 0], logits[:, :-1].argmax(-1))
    for layer in (*m.moe_layers(), *g.moe_layers()):
        layer.release()


def test_transforms_are_refused():
    import torch.autograd.forward_ad as fwd
    from ccfuser_b200.ops.dropout import dropout
    from ccfuser_b200.ops.embedding import embedding
    from ccfuser_b200.ops.logprobs import token_logprobs
    x, ids, state = torch.randn(4, 3, 64, device="cuda"), torch.arange(3, device="cuda"), torch.tensor([1, 2], device="cuda")
    calls = (lambda t: embedding(ids, t), lambda t: token_logprobs(t, ids).logprobs, lambda t: dropout(t, 0.5, state))
    for f in calls:
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x)
        with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            f(fwd.make_dual(x[0], torch.ones_like(x[0])))


def test_a_traced_graph_replays_the_kernels():
    """torch.jit.trace records the operations, not only the allocation of their outputs: on other inputs the graph gives what the functions give."""
    from ccfuser_b200.ops.dropout import dropout
    from ccfuser_b200.ops.embedding import embedding
    from ccfuser_b200.ops.logprobs import token_logprobs
    w, state = torch.randn(50, 64, device="cuda"), torch.tensor([1, 2], device="cuda")

    def chain(ids, targets):
        y = dropout(embedding(ids, w, 2.0), 0.3, state)
        out = token_logprobs(y, targets, top_k=3)
        return out.logprobs, out.entropy, out.top_logprobs, out.top_ids
    one = (torch.arange(10, device="cuda"), torch.arange(10, device="cuda"))
    two = (torch.arange(10, device="cuda") + 7, torch.arange(10, device="cuda") + 20)
    with torch.no_grad():
        traced = torch.jit.trace(chain, one, check_trace=False)
        for args in (one, two):
            for a, b in zip(traced(*args), chain(*args)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("function", ["C++", "Python"])
def test_refusals_on_the_gpu(monkeypatch, function):
    """The checks beside the kernels, in both forms of the functions."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.dropout import dropout
    from ccfuser_b200.ops.embedding import embedding, embedding_grad
    from ccfuser_b200.ops.logprobs import token_logprobs
    if function == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)
    w, ids = torch.randn(10, 8, device="cuda"), torch.tensor([[1, 2, 3]], device="cuda")
    for kw in (dict(position_ids=ids), dict(type_weight=w), dict(type_ids=ids), dict(padding_idx=10), dict(padding_idx=-11), dict(position_weight=w[:2]),
               dict(position_weight=w[:, :4]), dict(position_weight=w.half()), dict(position_weight=w.cpu()), dict(position_weight=w[:0], position_ids=ids)):
        with pytest.raises(ValueError):
            embedding(ids, w, **kw)
    for bad, error in ((ids.float(), TypeError), (ids.bool(), TypeError), (ids.cpu(), ValueError)):
        with pytest.raises(error):
            embedding(bad, w)
        with pytest.raises(error):
            embedding_grad(torch.randn(1, 3, 8, device="cuda"), bad, 10)
    with pytest.raises(TypeError):
        embedding(ids, w.double())
    with pytest.raises(ValueError):
        embedding(ids, w[0])
    with pytest.raises(ValueError):
        embedding(ids, w[:0])
    with pytest.raises(RuntimeError):
        embedding(ids, w, position_weight=w, position_ids=torch.zeros(2, 2, dtype=torch.long, device="cuda"))
    for grad, rows in ((torch.randn(2, 8, device="cuda"), 10), (torch.randn(1, 3, 8, device="cuda"), 0)):
        with pytest.raises(ValueError):
            embedding_grad(grad, ids, rows)
    x, t = torch.randn(3, 10, device="cuda"), torch.tensor([1, 2, 3], device="cuda")
    for kw in (dict(top_k=-1), dict(top_k=11), dict(top_k=33), dict(vocab_size=0), dict(vocab_size=11), dict(vocab_size=4, top_k=5),
               dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            token_logprobs(x, t, **kw)
    for bad, error in ((t[:2], ValueError), (t[:, None], ValueError), (t.cpu(), ValueError), (t.float(), TypeError)):
        with pytest.raises(error):
            token_logprobs(x, bad)
    s = torch.tensor([1, 2], device="cuda")
    for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(call=-1), dict(call=2 ** 32), dict(state=s.int()), dict(state=s[:1]),
               dict(state=torch.zeros(4, dtype=torch.int64, device="cuda")[::2]), dict(state=s.cpu()), dict(residual=x[:2]), dict(residual=x.half())):
        with pytest.raises(ValueError):
            dropout(**{"x": x, "p": 0.5, "state": s, **kw})
    # nothing to do
    assert embedding(ids[:0], w).shape == (0, 3, 8) and embedding(ids, w[:, :0]).shape == (1, 3, 0)
    assert token_logprobs(x[:0], t[:0]).logprobs.shape == (0,) and dropout(x[:0], 0.5, s).shape == (0, 10)


@pytest.mark.parametrize("function", ["C++", "Python"])
def test_tables_beyond_32_bits_are_refused(monkeypatch, function):
    """Numbers of rows and columns that the kernels' 32 bits would wrap: refused before anything is read or copied."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.embedding import embedding, embedding_grad
    if function == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)
    ids, one = torch.tensor([0, 0], device="cuda"), torch.ones(1, 1, device="cuda")
    for rows, cols in ((1, 2 ** 24 + 1), (1, 2 ** 32 + 8), (2 ** 31, 1), (2 ** 32 + 1, 1)):
        with pytest.raises(ValueError):
            embedding(ids, one.expand(rows, cols))
        w = torch.ones(2, min(cols, 2 ** 24), device="cuda")
        if cols == 1:
            with pytest.raises(ValueError):
                embedding(ids, w, position_weight=one.expand(rows, 1))
            with pytest.raises(ValueError):
                embedding(ids, w, type_weight=one.expand(rows, 1), type_ids=ids)
            with pytest.raises(ValueError):
                embedding_grad(torch.ones(2, 1, device="cuda"), ids, rows)
        else:
            with pytest.raises(ValueError):
                embedding_grad(one.expand(2, cols), ids, 1)


def test_ids_of_other_shapes():
    """A single id, positions and types given for all sequences at once."""
    from ccfuser_b200.ops.embedding import embedding
    w, p = torch.randn(10, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    one = embedding(torch.tensor(3, device="cuda"), w, 2.0, position_weight=p)
    assert torch.equal(one, w[3] * 2 + p[0])
    ids = torch.arange(6, device="cuda").int().view(2, 3)
    for shape in ((3,), (1, 3), (2, 1), (2, 3), ()):
        at = torch.full(shape, 4, device="cuda", dtype=torch.int32) if shape != (3,) else torch.tensor([5, 0, 2], device="cuda")
        y = embedding(ids, w, position_weight=p, position_ids=at, type_weight=p, type_ids=at.long())
        assert torch.equal(y, w[ids.long()] + p[at.long()].expand(2, 3, 8) + p[at.long()].expand(2, 3, 8))
