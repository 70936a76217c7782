"""Dropout (csrc/dropout.cu): the masks of the published generator, values and gradients of every type, state on the device."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,p,residual", [((1,), 0.5, True), ((7,), 0.1, False), ((8,), 0.1, True), ((9,), 0.9, True), ((5, 3, 11), 0.25, False),
                                              ((64, 512), 0.1, True), ((1021, 17), 0.3, True), ((4, 6), 0.0, True), ((4, 6), 1.0, True),
                                              ((4, 6), 1.0, False)])
def test_values_and_gradients(dtype, shape, p, residual):
    from ccfuser_b200.ops.dropout import dropout
    dt, g = TYPES[dtype], _gen(len(shape))
    x, r, dy = (torch.randn(*shape, generator=g, device="cuda").to(dt) for _ in range(3))
    x.requires_grad_(True)
    r.requires_grad_(True)
    seed, step, call = 0x1234567890ABCDEF, 3, 17
    state = torch.tensor([seed, step], device="cuda")
    y = dropout(x, p, state, call, residual=r if residual else None)
    n, drop = x.numel(), round(p * 65536)
    keep = (R.philox_bits(seed, step, call, n) >= drop).double().view(shape) * (65536 / max(1, 65536 - drop))
    xs = x.detach().double().cpu() * keep
    ref = xs + r.detach().double().cpu() if residual else xs
    R.assert_close(y, ref, 2 * R.U * (xs.abs() + ref.abs()), "y")
    grads = torch.autograd.grad(y, [x, r] if residual else [x], dy)
    want = dy.double().cpu() * keep
    R.assert_close(grads[0], want, 2 * R.U * want.abs(), "dx")
    if residual:
        assert torch.equal(grads[1], dy)


def test_a_large_mask():
    """Groups beyond 2^16, against the whole-number form in torch; the share that is kept, and no relation between calls, steps and seeds."""
    from ccfuser_b200.ops.dropout import dropout, keep_mask
    x = torch.ones(3000, 1111, device="cuda")
    masks = []
    for seed, step, call in ((1, 0, 0), (2, 0, 0), (1, 1, 0), (1, 0, 1)):
        state = torch.tensor([seed, step], device="cuda")
        y = dropout(x, 0.25, state, call)
        assert torch.equal(y != 0, keep_mask(x.shape, 0.25, state, call))
        masks.append(y != 0)
        n = x.numel()
        assert abs(float(masks[-1].double().mean()) - 0.75) < 6 * (0.75 * 0.25 / n) ** 0.5       # six standard deviations
    for i in range(4):
        for j in range(i):
            both = float((masks[i] & masks[j]).double().mean())
            assert abs(both - 0.5625) < 6 * (0.5625 * 0.4375 / n) ** 0.5


def test_dropped_elements_are_zero_whatever_they_were():
    from ccfuser_b200.ops.dropout import dropout, keep_mask
    state = torch.tensor([5, 5], device="cuda")
    x = torch.full((999,), float("nan"), device="cuda", dtype=torch.bfloat16)
    keep = keep_mask((999,), 0.5, state)
    y = dropout(x, 0.5, state)
    assert torch.equal(torch.isnan(y), keep) and bool((y[~keep] == 0).all())


def test_strides_alignment_and_the_python_function(monkeypatch):
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.dropout import dropout, keep_mask
    state = torch.tensor([8, 0], device="cuda")
    base, res = torch.randn(40, 33, 4, device="cuda").half(), torch.randn(33, 40, 3, device="cuda").half()
    keep = keep_mask((33, 40, 3), 0.2, state, 1)
    runs = []
    for module in (N.torch_module, lambda: None):
        monkeypatch.setattr(N, "torch_module", module)
        x = base.transpose(0, 1)[..., 1:].detach().requires_grad_(True)
        y = dropout(x, 0.2, state, 1, residual=res)
        dx, = torch.autograd.grad(y, [x], res)
        assert torch.equal((y - res) != 0, keep & ((y - res) != 0)) and torch.equal(dx != 0, keep & (res != 0))
        runs.append((y, dx))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert dropout(base[:0], 0.5, state).shape == (0, 33, 4)


def test_the_state_may_move_on_before_the_backward_pass_and_in_a_graph():
    from ccfuser_b200.ops.dropout import Dropout, DropoutState, keep_mask
    rng = DropoutState(77, device="cuda")
    drop = Dropout(0.5, rng)
    x = torch.ones(4096, device="cuda").requires_grad_(True)
    y = drop(x)
    rng.advance()
    z = drop(x)
    assert not torch.equal(y, z)
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert torch.equal(dx, y)
    del y, z, dx        # an eager graph of a leaf that is still alive would tie a captured backward pass to its stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rng.advance()
        y = drop(x)
        dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    seen = []
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, y) and rng.tensor.tolist() == [77, 2 + i]
        assert torch.equal(y != 0, keep_mask(y.shape, 0.5, rng.tensor, rng.calls))
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_other_streams():
    from ccfuser_b200.ops.dropout import dropout
    state = torch.tensor([1, 1], device="cuda")
    x = torch.randn(100_000, device="cuda")
    ref = dropout(x, 0.1, state)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(dropout(x, 0.1, state))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref) for y in got)
