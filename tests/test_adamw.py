"""AdamW on the host: refusals of the functions and of the C entry point, the torch path against 64 bits, the codes of 8-bit moments against the definition in
Python's numbers, their mean over many steps, checkpoints, re-placed experts, training steps."""
import copy
import ctypes as C
import math

import pytest
import token_refs as R
import torch
import training_refs as T

from ccfuser_b200 import native as N
from ccfuser_b200.ops import optim as O
from ccfuser_b200.ops.optim import FusedAdamW, adamw_step, state8, state_values

A = 1 << 20
RATES = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _call(tensor=None, **kw):
    t = (N.AdamwTensor * 1)(N.AdamwTensor(p=A, g=A, m=A, v=A, e=None, n=8, rows=1))
    for k, v in (tensor or {}).items():
        setattr(t[0], k, v)
    a = N.Adamw(tensors=C.addressof(t), count=1, type=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return N.load().ccf_adamw(C.byref(a), None)


@pytest.mark.parametrize("bad", [dict(tensors=None), dict(count=0), dict(type=3), dict(type=-1), dict(lr=-1.0), dict(lr=math.nan), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0),
                                 dict(eps=-1.0), dict(weight_decay=-1.0), dict(step=0), dict(scalars=A + 8)])
def test_entry_point_refuses(bad):
    assert _call(**bad) == -2


@pytest.mark.parametrize("bad", [dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(n=0), dict(n=2 ** 41), dict(rows=0), dict(rows=3), dict(p=A + 1), dict(g=A + 1), dict(m=A + 2),
                                 dict(v=A + 1), dict(e=A, n=2 ** 34, rows=2 ** 33)])
def test_entry_point_refuses_tensors(bad):
    assert _call(bad) == -2


def test_other_entry_points_refuse():
    lib = N.load()
    a = N.Adamw(lr=1e-3, beta1=0.9, beta2=0.999)
    assert lib.ccf_adamw_scalars(C.byref(a), None, None, A, None) == lib.ccf_adamw_scalars(C.byref(a), A, None, None, None) == -2
    assert lib.ccf_adamw_scalars(C.byref(a), A, None, A + 8, None) == -2
    assert lib.ccf_adamw_scalars(C.byref(N.Adamw(lr=-1.0)), A, None, A, None) == -2
    for args in ((None, A, A, 8, 1, 0, 0), (A, None, A, 8, 1, 0, 0), (A, A, None, 8, 1, 0, 0), (A, A, A, 0, 1, 0, 0), (A, A, A, 8, 3, 0, 0), (A, A, A, 8, 0, 0, 0), (A, A, A, 8, 1, 0, 3)):
        assert lib.ccf_state_values(*args, None) == -2


def test_functions_refuse():
    p, g, m, v = [torch.zeros(300)], [torch.ones(300)], [torch.zeros(300)], [torch.zeros(300)]
    c, d, e = ([t] for t in state8(p[0]))
    for kw in (dict(step=0), dict(step=-1), dict(), dict(step=1, counter=torch.zeros(1, dtype=torch.int64)), dict(step=1, lr=-1.0), dict(step=1, lr=math.nan), dict(step=1, betas=(1.0, 0.9)),
               dict(step=1, betas=(0.9, -0.1)), dict(step=1, eps=-1.0), dict(step=1, weight_decay=-1.0), dict(step=1, lr=torch.tensor(1e-3)), dict(counter=torch.zeros(1)),
               dict(counter=torch.zeros(2, dtype=torch.int64)), dict(step=1, numbers=[1, 2])):
        with pytest.raises(ValueError):
            adamw_step(p, g, m, v, **kw)
    for args in ((p, g + g, m, v), (p, g, [], v), (p, [g[0][:299]], m, v), (p, g, [m[0][None]], v), (p * 2, g * 2, m * 2, v * 2), (p, [g[0].to("meta")], m, v)):
        with pytest.raises(ValueError):
            adamw_step(*args, 1)
    for args in ((p, [g[0].half()], m, v), (p, [g[0].to_sparse()], m, v), (p, g, [m[0].half()], v), (p, g, c, d), ([p[0].int()], [g[0].int()], m, v)):
        with pytest.raises(TypeError):
            adamw_step(*args, 1)
    for kw in (dict(exponents=[]), dict(exponents=[e[0][:, :1]]), dict(exponents=[e[0][0]])):
        with pytest.raises(ValueError):
            adamw_step(p, g, c, d, 1, **kw)
    for args in ((p, g, m, d), ([p[0].double()], [g[0].double()], c, d)):
        with pytest.raises(TypeError):
            adamw_step(*args, 1, exponents=e)
    with pytest.raises(ValueError):
        state8(p[0], 7)
    for args in ((c[0], e[0][:, :1]), (c[0][:200], e[0]), (c[0], e[0].to("meta"))):
        with pytest.raises(ValueError):
            state_values(*args)
    for args, kw in (((m[0], e[0]), {}), ((c[0], e[0].int()), {}), ((c[0], e[0]), dict(dtype=torch.float64))):
        with pytest.raises(TypeError):
            state_values(*args, **kw)
    q = [torch.nn.Parameter(p[0])]
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            FusedAdamW(q, **kw)
    assert all(torch.equal(t, z) for t, z in ((p[0], torch.zeros(300)), (m[0], torch.zeros(300)), (v[0], torch.zeros(300))))      # nothing was changed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_moments_in_full(dtype):
    g = torch.Generator().manual_seed(1)
    kind = torch.float64 if dtype == torch.float64 else torch.float32
    for step in (1, 2, 50000):
        p, gr = torch.randn(7, 30, generator=g).to(dtype), (torch.randn(7, 30, generator=g) * 0.1).to(dtype)
        m, v = torch.randn(7, 30, generator=g).to(kind) * 0.05, torch.rand(7, 30, generator=g).to(kind) * 0.01
        want, off = T.adamw(p, gr, m, v, step, *RATES.values())
        adamw_step([p], [gr], [m], [v], step, **RATES)
        for name, a, b, o in zip("pmv", (p, m, v), want, off):
            R.assert_close(a, b, o, f"{name}, step {step}")


def test_codes_are_those_of_the_definition():
    """Blocks over the whole range of fp32, short blocks, rows; to the bit."""
    g = torch.Generator().manual_seed(2)
    for shape, rows in (((700,), 1), ((3, 300), 3), ((5, 7, 11), 5)):
        n = math.prod(shape)
        x = torch.randn(shape, generator=g)
        for scale in (torch.ones(()), 10.0 ** (6 * torch.rand(shape, generator=g) - 3), 10.0 ** (70 * torch.rand(shape, generator=g) - 38), torch.tensor(1e38), torch.tensor(1e-40)):
            bits = torch.randint(0, 1 << 20, shape, generator=g)
            for second in (False, True):
                value = (x * scale).abs() if second else x * scale
                codes, e = O._encode(value, rows, bits.int(), second)
                both = torch.stack([e, e], dim=-1)
                got = O._decode(codes, both, second)
                want = T.stored(value, rows, bits.reshape(-1).tolist(), second)
                assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.double().nan_to_num(), want.nan_to_num()), (shape, second)
                # a code is one of the two next to the value: off by less than an eighth of it, or than the smallest step of the block
                finite = torch.isfinite(got)
                smallest = 2.0 ** (e.int() - 127 - (33 if second else 17)).double().repeat_interleave(256, dim=-1)[:, :n // rows].reshape(shape)
                off = (got.double() - value.double()).abs()
                assert bool((off <= torch.maximum(value.double().abs() / 8, smallest))[finite].all())


def test_the_mean_of_what_is_stored_is_the_value():
    """400 roundings of 4096 values each: their mean is off by six standard deviations of it at most (a rounding between two codes a step apart has one of half a step)."""
    g = torch.Generator().manual_seed(3)
    value = torch.randn(4096, generator=g).abs() + 0.01
    total, key = torch.zeros(4096, dtype=torch.float64), 0
    for step in range(400):
        key = O._split_mix(O._split_mix(7) ^ step) >> 32
        h = O._mix((torch.arange(4096) + key) & 0xFFFFFFFF)
        codes, e = O._encode(value, 1, (h >> 12).int(), True)
        total += O._decode(codes, torch.stack([e, e], dim=-1), True).double()
    step_size = 2.0 ** (torch.frexp(value)[1].double() - 1 - 3)
    off = (total / 400 - value.double()) / step_size
    assert float(off.abs().max()) < 6 * 0.5 / 20 and abs(float(off.mean())) < 6 * 0.5 / (20 * 64)


def test_second_moments_follow_small_changes():
    """b2 = 0.999: a step moves them by a thousandth of their distance, where codes lie an eighth apart. From v to 4 v after n steps: 4 - 3 b2^n; of 8192 weights
    with chains of roundings whose spread is at most a step each, the mean is off by less than six standard errors."""
    p, m, v, e = torch.zeros(8192), *state8(torch.zeros(8192))
    ones, b2 = torch.full((8192,), 1.0), 0.999
    adamw_step([p], [ones], [m], [v], 1, lr=0.0, betas=(0.9, 0.0), exponents=[e])      # v = 1 to begin with
    for n in range(1, 1201):
        adamw_step([p], [2 * ones], [m], [v], n + 1, lr=0.0, betas=(0.9, b2), exponents=[e], seed=5)
    want = 4 - 3 * b2 ** 1200
    got = state_values(v, e, True, torch.float32).double()
    # a rounding adds a variance of at most step^2 / 4 and is forgotten by b2; between two codes it is p (1 - p) step^2 with p about a thousandth of 3 / step: 0.003 step
    spread = math.sqrt(0.003 * 0.5 / (1 - b2 ** 2))
    assert abs(float(got.mean()) - want) < 6 * spread / math.sqrt(8192), (float(got.mean()), want)


def _train(opt, params, seed, steps):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype)
        opt.step()


def test_as_torch_adamw_and_its_checkpoints():
    make = lambda: [torch.nn.Parameter(torch.ones(20, 30)), torch.nn.Parameter(torch.ones(7))]  # noqa: E731
    ours, ref = make(), make()
    a, b = FusedAdamW(ours, **RATES), torch.optim.AdamW(ref, **RATES)
    _train(a, ours, 1, 5)
    _train(b, ref, 1, 5)
    for p, q in zip(ours, ref):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
    # what torch's optimizer has saved is taken up, its groups' other keys among it
    other = make()
    c = FusedAdamW(other)
    c.load_state_dict(b.state_dict())
    assert c.param_groups[0]["lr"] == RATES["lr"] and c.param_groups[0]["state_bits"] == 32 and all(c.state[p]["step"] == 5 for p in other)
    with torch.no_grad():
        for p, q in zip(other, ref):
            p.copy_(q)
    _train(c, other, 2, 3)
    _train(b, ref, 2, 3)
    for p, q in zip(other, ref):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpoints_keep_the_bits(dtype, bits, tmp_path):
    make = lambda: [torch.nn.Parameter(torch.ones(90, 60, dtype=dtype)), torch.nn.Parameter(torch.ones(9, dtype=dtype))]  # noqa: E731
    ours = make()
    a = FusedAdamW(ours, **RATES, state_bits=bits, seed=9)
    _train(a, ours, 1, 4)
    assert ("exponents" in a.state[ours[0]]) == (bits == 8) and "exponents" not in a.state[ours[1]]
    assert a.state[ours[1]]["exp_avg"].dtype == torch.float32
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    others = make()
    with torch.no_grad():
        for p, q in zip(others, ours):
            p.copy_(q)
    b = FusedAdamW(others)
    b.load_state_dict(torch.load(tmp_path / "opt.pt"))
    c = copy.deepcopy(a)
    third = c.param_groups[0]["params"]
    for opt, params in ((a, ours), (b, others), (c, third)):
        _train(opt, params, 2, 3)
    for p, q, r in zip(ours, others, third):
        assert torch.equal(p, q) and torch.equal(p, r)
        for name, t in a.state[p].items():
            u = b.state[q][name]
            assert torch.equal(t, u) and t.dtype == u.dtype if torch.is_tensor(t) else t == u


def test_parameters_without_gradients_do_not_shift_the_others():
    """Replicas of a parameter on ranks where others had no gradient round alike."""
    runs = []
    for skip in (False, True):
        torch.manual_seed(4)
        params = [torch.nn.Parameter(torch.randn(80, 80)) for _ in range(3)]
        opt = FusedAdamW(params, state_bits=8)
        for i in range(3):
            for p in params:
                p.grad = torch.randn_like(p)
            if skip:
                params[0].grad = None
            opt.step()
        runs.append((params[2], opt.state[params[2]]))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1]["exp_avg"], runs[1][1]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_move_with_their_experts(bits):
    """A step, experts moved, a step: as without the move, whatever the width of an expert."""
    from ccfuser_b200 import MoEConfig, MoELayer
    from ccfuser_b200.parallel.placement import rebalance_experts
    cfg = MoEConfig(d_model=20, d_ffn=70, num_experts=4, dtype=torch.float32, backend="cpu")      # 1400 weights a matrix: no multiple of a block
    torch.manual_seed(5)
    layer = MoELayer(cfg)
    opt = FusedAdamW(layer.parameters(), lr=1e-2, state_bits=bits)
    x = torch.randn(50, 20)
    for _ in range(2):
        opt.zero_grad()
        layer(x).square().sum().backward()
        opt.step()
    w = layer.experts.htoh4.weight
    if bits == 8:
        assert opt.state[w]["exponents"].shape == (4, 6, 2)
    before = {k: v.clone() for k, v in opt.state[w].items() if torch.is_tensor(v)}
    values = [state_values(before["exp_avg"], before["exponents"], dtype=torch.float32) if bits == 8 else before["exp_avg"], w.detach().clone()]
    placement = [2, 0, 3, 1]
    rebalance_experts(layer, placement, opt)
    after = opt.state[w]
    assert torch.equal(w, values[1][placement])
    assert torch.equal(state_values(after["exp_avg"], after["exponents"], dtype=torch.float32) if bits == 8 else after["exp_avg"], values[0][placement])
    if bits == 8:      # a parameter whose exponents were laid out without its rows is not moved
        opt.state[w]["exponents"] = state8(w)[2]
        with pytest.raises(ValueError, match="exponents by row"):
            rebalance_experts(layer, placement, opt)


def test_training_steps_take_it():
    from ccfuser_b200.models.gpt_moe import GPTMoE, GPTMoEConfig
    from ccfuser_b200.train import TrainStep
    losses = {}
    for name in ("adamw", "fused_adamw", "fused_adamw8"):
        torch.manual_seed(6)
        model = GPTMoE(GPTMoEConfig(vocab_size=50, n_layer=2, n_head=2, d_model=32, d_ffn=64, seq_len=8, num_experts=4, backend="cpu", dtype=torch.float32))
        step = TrainStep(model, lr=1e-3, optimizer=name)
        ids = torch.arange(16).reshape(2, 8) % 50
        losses[name] = [step.step(ids) for _ in range(3)]
    assert losses["adamw"][0] == losses["fused_adamw"][0] == losses["fused_adamw8"][0]
    # both follow the same formula in fp32
    assert all(abs(a - b) <= 1e-4 * abs(a) for a, b in zip(losses["adamw"], losses["fused_adamw"]))
    assert all(math.isfinite(v) for v in losses["fused_adamw8"])
    with pytest.raises(ValueError):
        TrainStep(model, optimizer="adamw9")


def test_example_takes_it(capsys):
    import json
    import sys

    from ccfuser_b200.examples import train
    old = sys.argv
    sys.argv = ["train", "--model", "txl", "--variant", "nccl", "--steps", "2", "--warmup", "0", "--layers", "1", "--batch", "2", "--seq", "8", "--experts-per-gpu", "2",
                "--optimizer", "fused_adamw8"]
    try:
        train.main()
    finally:
        sys.argv = old
    rec = [json.loads(l) for l in capsys.readouterr().out.splitlines() if l.startswith("{")][0]
    assert math.isfinite(rec["final_loss"])


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    for bits in (32, 8):
        with FakeTensorMode():
            params = [torch.nn.Parameter(torch.empty(100, 100)), torch.nn.Parameter(torch.empty(3))]
            opt = FusedAdamW(params, state_bits=bits)
            for p in params:
                p.grad = torch.empty_like(p)
            opt.step()
            assert opt.state[params[0]]["exp_avg"].shape == (100, 100)


def test_a_small_decay_is_not_rounded_away():
    """1000 steps of lr wd = 3e-7 without gradients: 1 - lr wd is 1 - 2.98e-7 or 1 - 3.58e-7 in fp32; what is taken off is a sum of its own and rounded to a step of the weights, which
    spread over a binade are off by half a step up or down."""
    p = torch.linspace(1.0, 2.0, 4096)
    old, zeros = p.double(), [torch.zeros(4096) for _ in range(3)]
    for step in range(1, 1001):
        adamw_step([p], [zeros[0]], [zeros[1]], [zeros[2]], step, lr=3e-3, weight_decay=1e-4)
    lost = float(((old - p.double()) / old).mean())
    assert abs(lost - 3e-4) < 0.05 * 3e-4, lost


def _ranks(rank, world):
    from ccfuser_b200 import MoEConfig, MoELayer
    from ccfuser_b200.parallel.ddp import allreduce_replicated_grads
    from ccfuser_b200.parallel.placement import rebalance_experts
    torch.manual_seed(10)
    layer = MoELayer(MoEConfig(d_model=70, d_ffn=90, num_experts=6, dtype=torch.float32, backend="cpu", ep_size=world, max_tokens=64))
    opt = FusedAdamW(layer.parameters(), lr=1e-2, state_bits=8)

    def step(seed):
        opt.zero_grad()
        layer(torch.randn(64, 70, generator=torch.Generator().manual_seed(seed + rank))).square().sum().backward()
        allreduce_replicated_grads(layer)
        opt.step()

    def moments():
        return {n: [state_values(s["exp_avg"], s["exponents"], False, torch.float32), state_values(s["exp_avg_sq"], s["exponents"], True, torch.float32), p.detach().clone()]
                for n, p in layer.named_parameters() for s in [opt.state[p]] if "exponents" in s}

    step(1)
    step(3)
    before = moments()
    placement = [4, 1, 5, 0, 3, 2]
    rebalance_experts(layer, placement, opt)
    after = moments()
    step(5)
    return before, after, placement, layer.gate.gate.weight.detach().clone()


def test_moments_move_between_ranks_and_replicas_stay_alike():
    from mp_util import run_ranks
    res = run_ranks(_ranks, 2)
    before, after, placement = [r[0] for r in res], [r[1] for r in res], res[0][2]
    assert set(before[0]) == {"experts.htoh4.weight", "experts.h4toh.weight"}
    for rank in range(2):
        for name in before[0]:
            for k in range(3):
                for slot in range(3):
                    source = placement[rank * 3 + slot]
                    assert torch.equal(after[rank][name][k][slot], before[source // 3][name][k][source % 3]), (name, k)
    assert torch.equal(res[0][3], res[1][3])


def test_meta_tensors():
    for bits in (32, 8):
        params = [torch.nn.Parameter(torch.empty(100, 100, device="meta")), torch.nn.Parameter(torch.empty(3, device="meta"))]
        opt = FusedAdamW(params, state_bits=bits)
        for p in params:
            p.grad = torch.empty_like(p)
        opt.step()
        assert opt.state[params[0]]["exp_avg"].device.type == "meta"
