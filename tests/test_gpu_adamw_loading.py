"""Checkpoints of FusedAdamW and of torch's AdamW that come back on a GPU."""
import pytest
import torch

from ccfuser_b200.ops.optim import FusedAdamW

pytestmark = pytest.mark.gpu


def _params():
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(shape, generator=g).to(torch.bfloat16).cuda()) for shape in ((90, 60), (9,))]


def _set_gradients(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()


def test_a_rate_on_the_device_read_back_through_the_host(tmp_path):
    params, others = _params(), _params()
    a = FusedAdamW(params, lr=torch.tensor(0.1, device="cuda"), capturable=True, state_bits=8, seed=3)
    _set_gradients(params, 1)
    a.step()
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    b = FusedAdamW(others, lr=torch.tensor(0.5, device="cuda"), capturable=True)
    b.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu"))
    lr = b.param_groups[0]["lr"]
    assert lr.is_cuda and float(lr) == float(torch.tensor(0.1))
    with torch.no_grad():
        for p, q in zip(params, others):
            q.copy_(p)
    for opt, mine in ((a, params), (b, others)):
        _set_gradients(mine, 2)
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others)) and int(b.state[others[0]]["step"]) == 2


@pytest.mark.parametrize("capturable", [False, True])
def test_torchs_moments_come_into_the_same_codes_as_on_a_cpu(capturable):
    """Also into an optimizer whose next steps are captured."""
    params, theirs = _params(), _params()
    ref = torch.optim.AdamW(theirs, lr=0.1, fused=True)
    _set_gradients(theirs, 1)
    ref.step()
    opt = FusedAdamW(params, state_bits=8, seed=3, capturable=capturable)
    opt.load_state_dict(ref.state_dict())
    host = [torch.nn.Parameter(p.detach().cpu()) for p in theirs]
    on_cpu = FusedAdamW(host, state_bits=8, seed=3)
    on_cpu.load_state_dict(ref.state_dict())
    for name in ("exp_avg", "exp_avg_sq", "exponents"):
        assert torch.equal(opt.state[params[0]][name].cpu(), on_cpu.state[host[0]][name])
    assert opt.state[params[1]]["exp_avg"].dtype == torch.float32
    # it trains on: one step, then two captured ones or two more
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    eager = FusedAdamW(other, state_bits=8, seed=3)
    eager.load_state_dict(ref.state_dict())
    for o, mine in ((opt, params), (eager, other)):
        _set_gradients(mine, 2)
        o.step()
    eager.step()
    eager.step()
    if capturable:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        graph.replay()
        graph.replay()
    else:
        opt.step()
        opt.step()
    torch.cuda.synchronize()
    assert int(opt.state[params[0]]["step"]) == 4 and all(torch.equal(p, q) for p, q in zip(params, other))
