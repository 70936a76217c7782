"""Log probabilities (csrc/logprobs.cu) of logits far from zero and at temperatures far from one, against 64 bits: the products of logits with
log2(e) / T, to which the exponents are relative, are then large numbers whose rounding must not show."""
import pytest
import torch
import token_refs as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# a warp a row, 128 threads, 256 threads, clusters of two and four blocks
SHAPES = [(5, 300), (600, 5000), (30, 6000), (100, 20000), (3, 40000)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(x, t, top_k=0, temperature=1.0):
    """Values, alternatives and the gradient of everything; gradients come in with the temperature, so that those of the logits are of the size of one."""
    from ccfuser_b200.ops.logprobs import token_logprobs
    x = x.detach().requires_grad_(True)
    out = token_logprobs(x, t, top_k=top_k, temperature=temperature)
    ref = R.Scores(x, t, x.shape[1], top_k, temperature)
    R.assert_close(out.logprobs, ref.picked, ref.of_lp(ref.picked), "log probability")
    R.assert_close(out.entropy, ref.h, ref.of_h(), "entropy")
    if top_k:
        assert torch.equal(out.top_ids.cpu(), ref.top_ids)
        R.assert_close(out.top_logprobs, ref.top, ref.of_lp(ref.top), "alternatives")
    g = _gen(1)
    ups = [torch.randn(s, generator=g, device="cuda") * temperature for s in [t.shape, t.shape] + [(*t.shape, top_k)] * bool(top_k)]
    dx, = torch.autograd.grad([out.logprobs, out.entropy] + [out.top_logprobs] * bool(top_k), [x], ups)
    want, off = ref.grad(*ups)
    # a probability below 2^-126 is zero in fp32; with |lp| + H of less than 2^7 there, what it is multiplied with
    row = sum(u.double().cpu().abs().reshape(t.numel(), -1).sum(dim=1, keepdim=True) for u in ups)
    R.assert_close(dx, want, off + 2.0 ** -119 * row / temperature, "gradient")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("temperature", [1e-35, 1e-9, 1e-8, 2e-8, 1e-7, 1e-6, 1e-5, 1e-4, 1e4, 1e30])
def test_temperatures(dtype, rows, vocab, temperature):
    g = _gen(vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 10 + 30).to(TYPES[dtype])
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[::2] = x[::2].argmax(dim=1)
    _check(x, t, 3, temperature)


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("offset", [1e3, -1e3, 1e4, -1e4, 1e5, 1e6, -1e6, 3e6, 1e9, -5.3e9, 1.2e10, 1e12, 3e38])
def test_a_common_offset(rows, vocab, offset):
    g = _gen(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 3 + offset
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    _check(x, t, 3)
    _check(x, t, temperature=0.7)
    _check(x.bfloat16(), t)


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("offset", [0.0, 1e3, -1e4, 1e5, 7.2e5, -1e6])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_the_largest_comes_last_or_first(rows, vocab, offset, order):
    """Every turn of every thread finds a larger one, or none does: sums taken under many maxima, within a thread, between threads, warps and blocks, with offsets
    on both sides of, and across, where the rounded products stop being what the exponents are relative to."""
    place = torch.arange(vocab, device="cuda").double() / vocab * 6 * (1 if order == "rising" else -1)
    g = _gen(vocab)
    x = (place + torch.rand(rows, vocab, generator=g, device="cuda", dtype=torch.float64) * 0.5 + offset).float()
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    _check(x, t, 2)


@pytest.mark.parametrize("vocab", [300, 6000, 40000])
def test_maxima_on_both_sides(vocab):
    """Products of 2^20 lie between the maxima of one row's threads."""
    limit = 2.0 ** 20 / 1.4426950408889634
    place = torch.arange(vocab, device="cuda").double() / vocab * 40 - 38
    g = _gen(vocab)
    for sign in (1, -1):
        x = (sign * limit + place + torch.rand(4, vocab, generator=g, device="cuda", dtype=torch.float64)).float()
        x = x[:, torch.randperm(vocab, generator=g, device="cuda")]
        _check(x, torch.randint(0, vocab, (4,), generator=g, device="cuda"), 2)
