"""Hooks on saved tensors that hand them back in other memory: the backward passes go by the strides of what they get."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _spread(t):
    """The same values with gaps between the elements."""
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def _shifted(t):
    """The same values off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.view(t.shape).copy_(t)


HOOKS = {"cpu": lambda: torch.autograd.graph.save_on_cpu(), "spread": lambda: torch.autograd.graph.saved_tensors_hooks(_spread, lambda t: t),
         "shifted": lambda: torch.autograd.graph.saved_tensors_hooks(_shifted, lambda t: t)}


@pytest.fixture(params=["C++", "Python"])
def function(request, monkeypatch):
    from ccfuser_b200 import native as N
    if request.param == "Python":
        monkeypatch.setattr(N, "torch_module", lambda: None)


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("columns", [slice(0, 1000), slice(0, 1203), slice(3, 900), slice(8, 57)])
def test_log_probabilities(function, hook, columns):
    from ccfuser_b200.ops.logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(9, 7, 1203, generator=g, device="cuda").bfloat16()
    x = base[..., columns].detach().requires_grad_(True)
    t = torch.randint(0, x.shape[-1], (7, 9), generator=g, device="cuda").t()
    ups = [torch.randn(s, generator=g, device="cuda") for s in ((9, 7), (9, 7), (9, 7, 4))]
    grads = []
    for context in (None, HOOKS[hook]):
        if context is None:
            out = token_logprobs(x, t, top_k=4)
        else:
            with context():
                out = token_logprobs(x, t, top_k=4)
        grads.append(torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], [x], ups)[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("hook", list(HOOKS))
def test_embedding_and_dropout(function, hook):
    from ccfuser_b200.ops.dropout import dropout
    from ccfuser_b200.ops.embedding import embedding
    g = torch.Generator(device="cuda").manual_seed(0)
    w, p, t = (torch.randn(r, 24, generator=g, device="cuda").requires_grad_(True) for r in (40, 30, 2))
    ids, at, types = (torch.randint(0, r, (50, 29), generator=g, device="cuda") for r in (40, 30, 2))
    state = torch.tensor([5, 7], device="cuda")

    def step():
        y = dropout(embedding(ids, w, 2.0, position_weight=p, position_ids=at.int(), type_weight=t, type_ids=types.int()), 0.25, state)
        return lambda: torch.autograd.grad(y.square().sum(), [w, p, t])
    want = step()()
    with HOOKS[hook]():
        backward = step()
    assert all(torch.equal(a, b) for a, b in zip(backward(), want))
