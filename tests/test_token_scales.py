"""Log probabilities on the host of large logits and small temperatures: quotients beyond the type's range. No GPU."""
import pytest
import torch
import token_refs as R

from ccfuser_b200.ops.logprobs import token_logprobs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("temperature", [1e-37, 1e-30, 1e-8, 1e30])
@pytest.mark.parametrize("scale", [1.0, 300.0])
def test_finite_logits_give_numbers(dtype, temperature, scale):
    torch.manual_seed(0)
    x = (torch.randn(4, 50) * scale).to(dtype)
    x[1, 7] = x[1, 30] = x[1].max()
    x[2, 3:] = -float("inf")
    x.requires_grad_(True)
    t = x.argmax(dim=1)
    out = token_logprobs(x, t, top_k=2, temperature=temperature)
    ref = R.Scores(x, t, 50, 2, temperature)
    R.assert_close(out.logprobs, ref.picked, ref.of_lp(ref.picked), "log probability")
    R.assert_close(out.entropy, ref.h, ref.of_h(), "entropy")
    assert torch.equal(out.top_ids, ref.top_ids)
    dx, = torch.autograd.grad(out.logprobs, [x], torch.full((4,), temperature))
    assert bool(torch.isfinite(dx).all())


def test_rows_with_an_infinite_logit_are_nan():
    x = torch.zeros(3, 8)
    x[0, 2], x[1, 5] = float("inf"), float("nan")
    out = token_logprobs(x, torch.tensor([0, 0, 0]))
    assert torch.isnan(out.logprobs).tolist() == torch.isnan(out.entropy).tolist() == [True, True, False]
