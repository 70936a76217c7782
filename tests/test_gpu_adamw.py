"""AdamW over many tensors (csrc/adamw.cu): against 64 bits at every type, size and alignment; codes of 8-bit moments to the bit against the definition in Python's numbers and against
torch's operations; many tensors, streams, captured steps, values that are not finite."""
import math

import pytest
import token_refs as R
import torch
import training_refs as T

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
RATES = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
# around vectors, blocks of 256 and the 2048 of a thread block
SIZES = [(1,), (7,), (8,), (9,), (255,), (256,), (257,), (3, 100), (2047,), (2048,), (2049,), (4, 33, 65), (123, 457)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tensor(g, shape, dtype, scale=1.0, off=0):
    """A tensor that begins `off` elements behind a 16-byte boundary."""
    n = math.prod(shape)
    flat = torch.empty(n + off, dtype=dtype, device="cuda")
    flat[off:] = (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)
    return flat[off:].view(shape)


def _set(seed, shapes, dtype, off=0):
    g = _gen(seed)
    p, gr = ([_tensor(g, s, dtype, k, off) for s in shapes] for k in (1.0, 0.1))
    m = [_tensor(g, s, torch.float32, 0.05, off) for s in shapes]
    v = [_tensor(g, s, torch.float32, 0.1, off).square_() for s in shapes]
    return p, gr, m, v


@pytest.mark.parametrize("off", [0, 1, 4])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_moments_in_fp32(dtype, off):
    from ccfuser_b200.ops.optim import adamw_step
    for step in (1, 2, 100000):
        p, g, m, v = _set(step, SIZES, TYPES[dtype], off)
        want = [T.adamw(*t, step, *RATES.values()) for t in zip(p, g, m, v)]
        versions = [t._version for t in p + m + v]
        adamw_step(p, g, m, v, step, **RATES)
        assert all(t._version > old for t, old in zip(p + m + v, versions))
        for got, (ref, off_by) in zip(zip(p, m, v), want):
            for name, a, b, o in zip("pmv", got, ref, off_by):
                R.assert_close(a, b, o, f"{name} of {tuple(a.shape)}, step {step}")


def _state8(seed, p, rows):
    """8-bit moments that a step has left."""
    from ccfuser_b200.ops.optim import adamw_step, state8
    g = _gen(seed)
    states = [state8(t, r) for t, r in zip(p, rows)]
    m, v, e = map(list, zip(*states))
    scale = [torch.exp(2 * torch.randn(t.shape, generator=g, device="cuda")) for t in p]
    grads = [(torch.randn(t.shape, generator=g, device="cuda") * s * 0.1).to(t.dtype) for t, s in zip(p, scale)]
    adamw_step([t.clone() for t in p], grads, m, v, 1, exponents=e, seed=5, **RATES)
    return m, v, e


@pytest.mark.parametrize("dtype", list(TYPES))
def test_moments_in_8_bits(dtype):
    """p against 64 bits; what is stored, to the bit, from m and v as fp32 operations one after another give them."""
    from ccfuser_b200.ops.optim import adamw_step, state_values
    shapes = SIZES + [(6, 50, 7), (3, 300), (2, 4096)]
    rows = [1] * len(SIZES) + [6, 3, 2]
    p, g, _, _ = _set(3, shapes, TYPES[dtype])
    m, v, e = _state8(4, p, rows)
    step, seed = 17, -3
    old = [(state_values(a, x, dtype=torch.float32), state_values(b, x, True, torch.float32)) for a, b, x in zip(m, v, e)]
    want = [T.adamw(a, b, *c, step, *RATES.values()) for a, b, c in zip(p, g, old)]
    adamw_step(p, g, m, v, step, exponents=e, seed=seed, **RATES)
    b1, b2 = RATES["betas"]
    for i, (a, gr, (om, ov)) in enumerate(zip(p, g, old)):
        ref, off_by = want[i]
        R.assert_close(a, ref[0], off_by[0], f"p of {tuple(a.shape)}")
        gr = gr.float()
        bits = T.rounding_bits(seed, step, i, a.numel())
        for codes, value, low, second in ((m[i], om * b1 + gr * (1 - b1), [h & 0xFFFFF for h in bits], False),
                                          (v[i], ov * b2 + gr * gr * (1 - b2), [h >> 12 for h in bits], True)):
            got = state_values(codes, e[i], second, torch.float32)
            assert torch.equal(got.double().cpu(), T.stored(value, rows[i], low, second)), (tuple(a.shape), second)
            assert torch.equal(state_values(codes, e[i], second).float(), got)      # bf16 holds them as well
            if second:
                assert bool((got[value > 0] > 0).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_8_bits_as_torch_operations_have_them(dtype):
    """The same codes on the CPU, over a block's whole range, and from offsets that no vector begins at."""
    from ccfuser_b200.ops.optim import adamw_step
    g = _gen(6)
    for off in (0, 3):
        shapes = [(5000,), (3, 1001), (40, 40)]
        p = [_tensor(g, s, TYPES[dtype], 1.0, off) for s in shapes]
        scale = [10.0 ** (10 * torch.rand(s, generator=g, device="cuda") - 9) for s in shapes]
        gr = [(torch.randn(s, generator=g, device="cuda") * k).to(TYPES[dtype]) for s, k in zip(shapes, scale)]
        rows = [1, 3, 1]
        state = _state8(7, p, rows)
        host = [[t.cpu() for t in ts] for ts in (p, gr, *state)]
        for step in (2, 3, 4):
            for (a, b, m, v, e) in ((p, gr, *state), host):
                adamw_step(a, b, m, v, step, exponents=e, seed=11, **RATES)
        for ts, hs in zip((*state,), host[2:]):
            for a, b in zip(ts, hs):
                assert torch.equal(a.cpu(), b)
        for a, b in zip(p, host[0]):      # both are near the same value; three steps of RATES["lr"] long at most
            R.assert_close(a, b.double(), 3 * (R.half_step(a.dtype) * 2 * b.double().abs() + 64 * R.U * (b.double().abs() + 0.1)))


def test_values_that_are_not_finite():
    from ccfuser_b200.ops.optim import adamw_step, state8, state_values
    for bad in (math.nan, math.inf, -math.inf):
        p, g = [torch.ones(1000, device="cuda")], [torch.full((1000,), 0.5, device="cuda")]
        m, v, e = ([t] for t in state8(p[0]))
        g[0][300] = bad
        adamw_step(p, g, m, v, 1, exponents=e, **RATES)
        assert bool(torch.isnan(p[0][300])) and bool(torch.isfinite(p[0][torch.arange(1000) != 300]).all())
        block = torch.zeros(1000, dtype=torch.bool, device="cuda")
        block[256:512] = True
        assert torch.equal(torch.isnan(state_values(m[0], e[0])), block) and e[0][0, :, 0].tolist()[1] == 255
        g[0][300] = 0.5
        adamw_step(p, g, m, v, 2, exponents=e, **RATES)
        assert torch.equal(torch.isnan(p[0]), block)
    # the largest and the smallest magnitudes: no infinity, no zero second moment of a gradient whose square fp32 holds
    p, g = [torch.zeros(512, device="cuda")], [torch.zeros(512, device="cuda")]
    g[0][0], g[0][1], g[0][256], g[0][257] = 1.8e19, 1e-3, 1e-19, -1e-22
    m, v, e = ([t] for t in state8(p[0]))
    adamw_step(p, g, m, v, 1, exponents=e, **RATES)
    second = state_values(v[0], e[0], True, torch.float32)
    assert bool(torch.isfinite(second).all()) and second[0] > 0 and second[1] > 0 and bool(torch.isfinite(p[0]).all())
    assert bool((second[2:256] == 0).all()) and second[256] > 0


def test_zero_gradients_leave_zero_moments():
    from ccfuser_b200.ops.optim import adamw_step, state8, state_values
    p, g = [torch.randn(3000, device="cuda").bfloat16()], [torch.zeros(3000, device="cuda").bfloat16()]
    old = p[0].clone()
    m, v, e = ([t] for t in state8(p[0]))
    for step in range(1, 4):
        adamw_step(p, g, m, v, step, exponents=e, lr=1e-3, weight_decay=0.0)
    assert torch.equal(p[0], old) and not bool(m[0].any()) and not bool(v[0].any()) and bool((e[0] == 40).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than a launch takes, of several types and places, against each by itself."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.optim import adamw_step
    g = _gen(8)
    types = list(TYPES.values())
    shapes = [(1 + 37 * i % 900,) for i in range(1300)]
    p = [_tensor(g, s, types[i % 3], 1.0, i % 5) for i, s in enumerate(shapes)]
    gr = [_tensor(g, t.shape, t.dtype, 0.1) for t in p]
    gr[5] = gr[5].repeat_interleave(2)[::2]      # not contiguous
    state = _state8(9, p, [1] * len(p)) if bits == 8 else ([torch.zeros(t.shape, device="cuda") for t in p], [torch.zeros(t.shape, device="cuda") for t in p], None)
    copy = [None if ts is None else [t.clone() for t in ts] for ts in (p, *state)]
    before = N.LAUNCHES[0]
    adamw_step(p, gr, state[0], state[1], 3, exponents=state[2], seed=2, **RATES)
    assert N.LAUNCHES[0] - before == 6      # 434 or 433 of each type
    from ccfuser_b200.ops import optim as O
    ref = list(zip(copy[0], gr, copy[1], copy[2], copy[3] or [None] * len(p)))
    key = O._split_mix(O._split_mix(2) ^ 3) >> 32
    for i, t in enumerate(ref):
        if i % 13 == 0 or i > 1250:
            O._adamw_torch(*t, (key + i * 0x9E3779B9) & 0xFFFFFFFF, RATES["lr"], *RATES["betas"], RATES["eps"], RATES["weight_decay"], 3)
            if bits == 8:
                assert torch.equal(state[0][i], t[2]) and torch.equal(state[1][i], t[3]) and torch.equal(state[2][i], t[4])
            R.assert_close(p[i], t[0].double(), 2 * R.half_step(p[i].dtype) * t[0].double().abs() + 64 * R.U * (t[0].double().abs() + 0.1))


@pytest.mark.parametrize("bits", [32, 8])
def test_streams_and_captured_steps(bits):
    from ccfuser_b200.ops.optim import FusedAdamW

    def model():
        torch.manual_seed(1)
        return [torch.nn.Parameter(torch.randn(100, 100, device="cuda").bfloat16()), torch.nn.Parameter(torch.randn(30, device="cuda").bfloat16())]

    grads = [[torch.randn(p.shape, device="cuda", generator=_gen(10 + i)).bfloat16() for p in model()] for i in range(5)]
    lrs = [1e-2, 1e-2, 5e-3, 2e-3, 1e-3]

    def run(opt, params, i):
        for p, g in zip(params, grads[i]):
            p.grad = g
        for group in opt.param_groups:
            if torch.is_tensor(group["lr"]):
                group["lr"].fill_(lrs[i])
            else:
                group["lr"] = lrs[i]
        opt.step()

    want = model()
    opt = FusedAdamW(want, state_bits=bits, seed=4)
    for i in range(5):
        run(opt, want, i)
    other = model()
    opt = FusedAdamW(other, state_bits=bits, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(5):
            run(opt, other, i)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    # rates from the device are rounded to fp32 before the others are computed from them: the same but for a step of the weights' type here and there
    params = model()
    opt = FusedAdamW(params, lr=torch.tensor(1e-2, device="cuda"), state_bits=bits, seed=4, capturable=True)
    run(opt, params, 0)
    static = [torch.empty_like(g) for g in grads[0]]
    for p, g in zip(params, static):
        p.grad = g
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(1, 5):
        for s, g in zip(static, grads[i]):
            s.copy_(g)
        opt.param_groups[0]["lr"].fill_(lrs[i])
        graph.replay()
    assert all(int(opt.state[p]["step"]) == 5 for p in params)
    for a, b in zip(params, want):
        R.assert_close(a, b.double().detach(), 5 * 2 * R.half_step(a.dtype) * b.detach().double().abs())
    plain = FusedAdamW(model(), state_bits=bits)
    for p, g in zip(plain.param_groups[0]["params"], grads[0]):
        p.grad = g
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            plain.step()


def test_the_python_launches(monkeypatch):
    """Without the C++ module: the same bits."""
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.optim import FusedAdamW
    runs = []
    for module in (N.torch_module, lambda: None):
        monkeypatch.setattr(N, "torch_module", module)
        for bits in (32, 8):
            g = _gen(12)
            params = [torch.nn.Parameter(_tensor(g, s, t)) for s in ((70, 70), (5,), (0,)) for t in TYPES.values()]
            opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
            for _ in range(3):
                for p in params:
                    p.grad = torch.randn(p.shape, generator=g, device="cuda").to(p.dtype)
                opt.step()
            runs.append([t for p in params for t in (p, *(s for s in opt.state[p].values() if torch.is_tensor(s)))])
    for a, b in ((0, 2), (1, 3)):
        assert all(torch.equal(x, y) for x, y in zip(runs[a], runs[b]))


def test_tensors_that_the_kernels_do_not_take():
    """fp64, not contiguous and on the CPU, next to one that they take."""
    from ccfuser_b200.ops.optim import FusedAdamW
    g = _gen(13)
    make = lambda: [torch.nn.Parameter(torch.ones(40, 50, device="cuda").t()), torch.nn.Parameter(torch.ones(30, dtype=torch.float64, device="cuda")),
                    torch.nn.Parameter(torch.ones(20)), torch.nn.Parameter(torch.ones(60, 90, device="cuda"))]  # noqa: E731
    ours, ref = make(), make()
    a, b = FusedAdamW(ours, lr=1e-2), torch.optim.AdamW(ref, lr=1e-2)
    for _ in range(4):
        for p, q in zip(ours, ref):
            p.grad = torch.randn(p.shape, generator=g, device="cuda").to(device=p.device, dtype=p.dtype)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(ours, ref):
        assert torch.allclose(p.double(), q.double(), rtol=1e-5, atol=1e-6)      # both follow the formula in fp32, in another order


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_two_to_the_31_weights(bits):
    """The weights around 2^31 and the last ones, against the same weights as a tensor of their own (whose codes differ, as their numbers do)."""
    from ccfuser_b200.ops.optim import adamw_step, state8, state_values
    n = 2 ** 31 + 5000
    p, g = torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_(0, 1, generator=_gen(14)), torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_(0, 1, generator=_gen(15))
    if bits == 8:
        m, v, e = state8(p)
    else:
        m, v, e = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), None
    parts = [(2 ** 31 - 5 * 256, 2 ** 31 + 5 * 256), (n - 4 * 256 - 5000 % 256, n)]
    small = [(p[a:b].clone(), g[a:b].clone()) for a, b in parts]
    adamw_step([p], [g], [m], [v], 1, exponents=None if e is None else [e], seed=3, **RATES)
    for (a, b), (q, h) in zip(parts, small):
        if bits == 8:
            cm, cv, ce = state8(q)
            adamw_step([q], [h], [cm], [cv], 1, exponents=[ce], seed=3, **RATES)
            block = slice(a // 256, a // 256 + ce.shape[1])
            assert a % 256 == 0 and torch.equal(e[0, block], ce[0])
            got = state_values(m[a:b], e[:, block]).float()
            exact = h.float() * (1 - RATES["betas"][0])
            assert bool(((got - exact).abs() <= exact.abs() / 8 + 2.0 ** -16).all())
        else:
            cm, cv = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape, device="cuda")
            adamw_step([q], [h], [cm], [cv], 1, **RATES)
            assert torch.equal(m[a:b], cm) and torch.equal(v[a:b], cv)
        assert torch.equal(p[a:b], q)


def test_steps_in_inference_mode_and_on_another_stream():
    from ccfuser_b200.ops.optim import adamw_step, state8
    runs = []
    for how in (torch.no_grad, torch.inference_mode):
        with how():
            p, g = torch.ones(5000, device="cuda").half(), torch.full((5000,), 0.5, device="cuda").half()
            m, v, e = state8(p)
            for step in range(1, 4):
                adamw_step([p], [g], [m], [v], step, exponents=[e], seed=1, **RATES)
            runs.append([t.clone() for t in (p, m, v, e)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_turns_of_large_tensors():
    """Blocks of weights that a warp takes one after another, ends of tensors and rows among them: the codes of torch's operations."""
    from ccfuser_b200.ops.optim import adamw_step
    shapes, rows = [(3, 1500001), (9,), (2, 2000003), (4096,), (4000007,), (5, 700, 1024)], [3, 1, 2, 1, 1, 5]
    p, g, _, _ = _set(16, shapes, torch.bfloat16)
    state = _state8(17, p, rows)
    host = [[t.cpu() for t in ts] for ts in (p, g, *state)]
    for (a, b, m, v, e) in ((p, g, *state), host):
        adamw_step(a, b, m, v, 2, exponents=e, seed=11, **RATES)
    for ts, hs in zip(state, host[2:]):
        for a, b in zip(ts, hs):
            assert torch.equal(a.cpu(), b)
    for a, b in zip(p, host[0]):
        R.assert_close(a, b.double(), R.half_step(a.dtype) * 2 * b.double().abs() + 64 * R.U * (b.double().abs() + 0.1))
