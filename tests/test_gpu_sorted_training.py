"""Training steps of a mixture of experts on the sorted tokens and AdamW together: router, rows by expert, experts, rows back by weight, loss, gradients, update.
Against 64 bits, captured and replayed, on the library's grouped GEMM, in the models' training step."""
import pytest
import token_refs as R
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


class SortedMoE(torch.nn.Module):
    """Two-matrix experts with ReLU on sorted rows; every expert sees all rows and keeps its own, so that nothing reads the host."""

    def __init__(self, d, f, experts, k, align=8):
        super().__init__()
        self.router = torch.nn.Linear(d, experts)
        self.w1, self.w2 = torch.nn.Parameter(torch.randn(experts, f, d) * d ** -0.5), torch.nn.Parameter(torch.randn(experts, d, f) * f ** -0.5)
        self.k, self.align = k, align

    def forward(self, x):
        from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
        score, idx = torch.topk(self.router(x), self.k, dim=-1)
        rows, order = sort_by_expert(x, idx, self.w1.shape[0], align=self.align)
        expert = idx.reshape(-1)[order.row_slot.clamp(min=0).long()]
        out = sum(F.relu(rows @ a.t()) @ b.t() * (expert == e).unsqueeze(1) for e, (a, b) in enumerate(zip(self.w1, self.w2)))
        return return_rows(out, order, torch.softmax(score, dim=-1))


def _oracle(model, x):
    """The same by expert, in 64 bits on the host."""
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in model.named_parameters()}
    xd = x.detach().double().cpu().requires_grad_(True)
    score, idx = torch.topk(F.linear(xd, p["router.weight"], p["router.bias"]), model.k, dim=-1)
    w = torch.softmax(score, dim=-1)
    y = torch.zeros_like(xd)
    for e in range(model.w1.shape[0]):
        token, slot = (idx == e).nonzero(as_tuple=True)
        y = y.index_add(0, token, F.relu(xd[token] @ p["w1"][e].t()) @ p["w2"][e].t() * w[token, slot].unsqueeze(1))
    return y, xd, p


def test_a_step_against_64_bits():
    from ccfuser_b200.ops.optim import FusedAdamW
    torch.manual_seed(0)
    d, f, experts, k, tokens = 64, 96, 6, 2, 200
    model = SortedMoE(d, f, experts, k).cuda()
    x, dy = torch.randn(tokens, d, device="cuda", requires_grad=True), torch.randn(tokens, d, device="cuda")
    y = model(x)
    y.backward(dy)
    ref, xd, p = _oracle(model, x)
    ref.backward(dy.double().cpu())
    # chains of products of d, f, d (f) and tokens terms around values of the size of a few; the largest of a result stands for the size of the terms behind it
    for name, got, want, terms in [("y", y, ref, d + f + k)] + [("x", x.grad, xd.grad, 2 * (d + f) + k)] + [(n, t.grad, p[n].grad, 2 * (d + f) + tokens) for n, t in model.named_parameters()]:
        R.assert_close(got, want.detach(), terms * R.U * 8 * float(want.detach().abs().max()), name)
    # the update from these gradients: at step 1 lr g / (|g| + eps) whatever their size; where g is small its sign may be lost
    old = {n: t.detach().double().cpu() for n, t in model.named_parameters()}
    opt = FusedAdamW(model.parameters(), lr=1e-3, weight_decay=0.1)
    opt.step()
    for n, t in model.named_parameters():
        g = t.grad.double().cpu()
        want = old[n] * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)
        R.assert_close(t, want, 4 * R.U * old[n].abs() + 1e-3 * 16 * R.U, n)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_the_eager_ones(bits):
    from ccfuser_b200.ops.optim import FusedAdamW
    data = [torch.randn(300, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(6)]
    side = torch.cuda.Stream()

    def make():
        torch.manual_seed(1)
        model = SortedMoE(64, 128, 8, 2).cuda()
        return model, FusedAdamW(model.parameters(), lr=1e-3, state_bits=bits, capturable=True)

    def step(model, opt, x):
        opt.zero_grad(set_to_none=True)
        loss = (model(x) - x).square().mean()
        loss.backward()
        opt.step()
        return loss

    eager, first = make()
    for x in data:
        step(eager, first, x)
    model, opt = make()
    x = data[0].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(model, opt, x)
    torch.cuda.current_stream().wait_stream(side)
    opt.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(model, opt, x)
    for new in data[1:]:
        x.copy_(new)
        graph.replay()
    torch.cuda.synchronize()
    for (n, a), b in zip(model.named_parameters(), eager.parameters()):
        assert torch.equal(a, b), n
        assert all(torch.equal(s, first.state[b][key]) for key, s in opt.state[a].items())


def test_rows_for_the_grouped_gemm():
    """``base`` and ``counts`` of align=128 are the groups of ops.gemm; rows between them are zeros, which its weight gradients read."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops import gemm as G
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    torch.manual_seed(2)
    tokens, d, n, experts, k = 700, 256, 512, 5, 2
    x = torch.randn(tokens, d, device="cuda").bfloat16()
    w = (torch.randn(experts, n, d, device="cuda") * d ** -0.5).bfloat16()
    idx, weights = torch.randint(0, experts, (tokens, k), device="cuda"), torch.rand(tokens, k, device="cuda")
    rows, order = sort_by_expert(x, idx, experts, align=128)
    out = torch.zeros(rows.shape[0], n, dtype=x.dtype, device="cuda")
    G.launch(a0=rows, b0=w.view(-1, d), a_major=N.MAJ_K, b_major=N.MAJ_K, epi=N.EPI_STORE, n=n, k=d, group_base=order.base[:-1], group_rows=order.counts, num_groups=experts,
             b_group_rows=n, out0=out)
    y = return_rows(out, order, weights)
    xd, wd = x.double().cpu(), w.double().cpu()
    each = torch.einsum("td,tknd->tkn", xd, wd[idx.cpu()])
    size = torch.einsum("td,tknd->tkn", xd.abs(), wd[idx.cpu()].abs())
    # sums of d products in fp32, rounded to bf16 (2^-8), then two of them by weight
    off = ((each.abs() * 2.0 ** -8 + d * R.U * size) * weights.double().cpu().unsqueeze(-1)).sum(dim=1)
    R.assert_close(y, (each * weights.double().cpu().unsqueeze(-1)).sum(dim=1), off + 2 * R.U * size.sum(dim=1))


@pytest.mark.parametrize("name", ["fused_adamw", "fused_adamw8"])
def test_the_models_training_step(name):
    """A GPT with fused MoE layers: the same losses as with torch's optimizer up to where bf16 weights round differently, and a checkpoint that goes on to the bit."""
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.train import TrainStep

    def make():
        torch.manual_seed(3)
        model = GPTMoE(GPTMoEConfig(vocab_size=200, n_layer=2, n_head=2, d_model=128, d_ffn=256, seq_len=32, num_experts=4, max_tokens=128), device="cuda")
        return model, TrainStep(model, lr=1e-3, optimizer=name)

    model, step = make()
    ids = torch.randint(0, 200, (4, 32), generator=torch.Generator().manual_seed(4)).pin_memory()
    losses = [step.step(ids) for _ in range(4)]
    assert all(v == v for v in losses)
    saved = ({k: v.clone() for k, v in model.state_dict().items()}, step.opt.state_dict())
    other, again = make()
    other.load_state_dict(saved[0])
    again.opt.load_state_dict(saved[1])
    assert step.step(ids) == again.step(ids)
    for (n, p), q in zip(model.named_parameters(), other.parameters()):
        assert torch.equal(p, q), n
    eights = sum("exponents" in s for s in step.opt.state.values())
    assert eights > 0 if name == "fused_adamw8" else eights == 0
