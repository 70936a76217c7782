"""Embedding, log probabilities and dropout on the host: refusals of the functions and of the C entry points, and the torch path against the
definitions and against differences. No GPU, made-up addresses."""
import ctypes as C

import pytest
import torch
import token_refs as R

from ccfuser_b200 import native as N
from ccfuser_b200.ops import dropout as D
from ccfuser_b200.ops import embedding as E
from ccfuser_b200.ops import logprobs as L

A = 1 << 20      # an address that nothing reads


# ---- embedding ---------------------------------------------------------------------------------------------------------
def _embed(**kw):
    e = N.Embed(tokens=8, seq=4, tables=1, d=64, type=0)
    t = e.table[0]
    t.weight, t.ids, t.grad, t.scratch, t.rows, t.ld, t.skip, t.scale, t.wide = A, A, A, A, 10, 64, -1, 1.0, 1
    for k, v in kw.items():
        setattr(t if hasattr(t, k) else e, k, v)
    return e


@pytest.mark.parametrize("bad", [dict(tables=0), dict(tables=4), dict(type=3), dict(type=-1), dict(d=0), dict(tokens=0), dict(tokens=2 ** 26 + 4), dict(tokens=2 ** 31),
                                 dict(seq=0), dict(seq=3), dict(rows=0), dict(rows=2 ** 31), dict(ids=None, rows=3)])
def test_embedding_entry_points_refuse(bad):
    lib = N.load()
    e = _embed(**bad)
    assert lib.ccf_embedding_fwd(C.byref(e), A, A, None) == -2
    assert lib.ccf_embedding_bwd(C.byref(e), A, A, None) == -2


def test_embedding_entry_points_refuse_missing_memory():
    lib = N.load()
    assert lib.ccf_embedding_fwd(C.byref(_embed(weight=None)), A, A, None) == -2
    assert lib.ccf_embedding_fwd(C.byref(_embed(ld=63)), A, A, None) == -2
    assert lib.ccf_embedding_fwd(C.byref(_embed()), None, A, None) == -2
    assert lib.ccf_embedding_bwd(C.byref(_embed(grad=None)), A, A, None) == -2
    assert lib.ccf_embedding_bwd(C.byref(_embed(tokens=1028, scratch=None)), A, A, None) == -2
    assert lib.ccf_embedding_bwd(C.byref(_embed(tokens=1028, scratch=A + 8)), A, A, None) == -2
    assert lib.ccf_embedding_bwd(C.byref(_embed()), None, A, None) == -2
    assert lib.ccf_embedding_scratch(0, 1, 10, 64, 1) == lib.ccf_embedding_scratch(8, 1, 0, 64, 1) == lib.ccf_embedding_scratch(8, 3, 5, 64, 1) == -1
    assert lib.ccf_embedding_scratch(1024, 1, 10, 64, 1) == 0
    assert lib.ccf_embedding_scratch(5000, 50, 100, 64, 1) > lib.ccf_embedding_scratch(5000, 50, 100, 64, 0) > 0


def test_embedding_entry_points_refuse_wide_tables():
    lib = N.load()
    e = _embed(d=2 ** 24 + 1, ld=2 ** 24 + 1)
    assert lib.ccf_embedding_fwd(C.byref(e), A, A, None) == lib.ccf_embedding_bwd(C.byref(e), A, A, None) == -2
    assert lib.ccf_embedding_scratch(5000, 50, 100, 2 ** 24 + 1, 1) == -1 < lib.ccf_embedding_scratch(5000, 50, 100, 2 ** 24, 1)


def test_embedding_refuses():
    w, ids = torch.randn(10, 8), torch.tensor([[1, 2, 3]])
    for kw in (dict(position_ids=ids), dict(type_weight=w), dict(type_ids=ids), dict(padding_idx=10), dict(padding_idx=-11),
               dict(position_weight=w[:2]), dict(position_weight=w[:, :4]), dict(position_weight=w.double())):
        with pytest.raises(ValueError):
            E.embedding(ids, w, **kw)
    for bad in (ids.float(), ids.bool()):
        with pytest.raises(TypeError):
            E.embedding(bad, w)
    with pytest.raises(ValueError):
        E.embedding(ids, w[0])
    with pytest.raises(ValueError):
        E.embedding(ids, w.to("meta"))
    with pytest.raises(IndexError):
        E.embedding(torch.tensor([10]), w)
    with pytest.raises(ValueError):
        E.embedding_grad(torch.randn(2, 8), ids, 10)
    with pytest.raises(ValueError):
        E.embedding_grad(torch.randn(1, 3, 8), ids, 0)
    for kw in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(ValueError):
            E.Embedding(4, 8, **kw)


def test_embedding_on_the_host():
    torch.manual_seed(0)
    w, p, t = (torch.randn(r, 6, dtype=torch.float64, requires_grad=True) for r in (9, 7, 2))
    ids, tt = torch.tensor([[1, 4, 0, 4], [0, 0, 8, 1]]), torch.tensor([0, 0, 1, 1])
    y = E.embedding(ids, w, 2.5, position_weight=p, type_weight=t, type_ids=tt, padding_idx=0)
    dy = torch.randn_like(y)
    y.backward(dy)
    places = torch.arange(4).expand(2, 4)
    ref, _ = R.embedding_sum([(ids, w, 2.5), (places, p, 1.0), (tt.expand(2, 4), t, 1.0)])
    torch.testing.assert_close(y, ref)
    torch.testing.assert_close(w.grad, R.table_grad(ids, dy, 9, 2.5, 0)[0])
    torch.testing.assert_close(p.grad, R.table_grad(places, dy, 7, 1.0)[0])
    torch.testing.assert_close(t.grad, R.table_grad(tt.expand(2, 4), dy, 2, 1.0)[0])
    torch.testing.assert_close(E.embedding_grad(dy, ids, 9, 2.5, 0), w.grad)
    m = E.Embedding(9, 6, scale=2.5, dtype=torch.float64)
    m.load_state_dict({"weight": w.detach()})
    torch.testing.assert_close(m(ids), w[ids].detach() * 2.5)
    assert E.embedding(ids[:0], w).shape == (0, 4, 6) and E.embedding(torch.tensor(3), w).shape == (6,)


# ---- log probabilities -------------------------------------------------------------------------------------------------
def _scores(**kw):
    a = N.Logprobs(x=A, targets=A, logprobs=A, entropy=A, stats=A, dx=A, rows=4, ld=64, vocab=64, width=64, inv_t=1.0, ignore=-100)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(x=None), dict(x=A + 2), dict(targets=None), dict(rows=0), dict(rows=2 ** 28), dict(vocab=0), dict(vocab=65),
                                 dict(width=2 ** 30 + 1, ld=2 ** 31), dict(ld=63), dict(top_k=-1), dict(top_k=33), dict(vocab=3, top_k=4),
                                 dict(type=3), dict(inv_t=0.0), dict(inv_t=float("nan"))])
def test_logprobs_entry_points_refuse(bad):
    lib = N.load()
    assert lib.ccf_logprobs_fwd(C.byref(_scores(**bad)), None) == -2
    assert lib.ccf_logprobs_bwd(C.byref(_scores(**bad)), None) == -2


def test_logprobs_entry_points_refuse_missing_memory():
    lib = N.load()
    for bad in (dict(logprobs=None), dict(entropy=None), dict(top_k=1, top_ids=A), dict(top_k=1, top_logprobs=A)):
        assert lib.ccf_logprobs_fwd(C.byref(_scores(**bad)), None) == -2
    for bad in (dict(dx=None), dict(dx=A + 8), dict(stats=None), dict(d_top=A), dict(d_top=A, top_k=2)):
        assert lib.ccf_logprobs_bwd(C.byref(_scores(**bad)), None) == -2


def test_logprobs_entry_point_refuses_rows_of_another_alignment():
    lib = N.load()
    for bad in (dict(dx_ld=0), dict(dx_ld=63), dict(dx_ld=65), dict(dx_ld=68), dict(dx_ld=66, type=2), dict(dx_ld=-64), dict(ld=65, dx_ld=64)):
        assert lib.ccf_logprobs_bwd(C.byref(_scores(**bad)), None) == -2


def test_logprobs_refuses():
    x, t = torch.randn(3, 10), torch.tensor([1, 2, 3])
    for kw in (dict(top_k=-1), dict(top_k=11), dict(top_k=33), dict(vocab_size=0), dict(vocab_size=11), dict(vocab_size=4, top_k=5),
               dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            L.token_logprobs(x, t, **kw)
    for bad in (t[:2], t[:, None], t.to("meta")):
        with pytest.raises(ValueError):
            L.token_logprobs(x, bad)
    with pytest.raises(TypeError):
        L.token_logprobs(x, t.float())
    with pytest.raises(IndexError):
        L.token_logprobs(x, t, vocab_size=3)


def test_logprobs_on_the_host():
    torch.manual_seed(1)
    x = torch.randn(5, 12, dtype=torch.float64)
    x[0, 3:] = -float("inf")
    x[1] = -float("inf")
    x[2, 4] = x[2, 7] = 9.0
    x.requires_grad_(True)
    t = torch.tensor([1, 2, 7, -100, 9])
    out = L.token_logprobs(x, t, top_k=5, temperature=0.7, vocab_size=11)
    g, gh, gk = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64), torch.randn(5, 5, dtype=torch.float64)
    dx, = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], [x], [g, gh, gk])
    ref = R.Scores(x, t, 11, 5, 0.7)
    torch.testing.assert_close(out.logprobs, ref.picked)
    torch.testing.assert_close(out.entropy, ref.h)
    torch.testing.assert_close(out.top_logprobs, ref.top)
    assert torch.equal(out.top_ids, ref.top_ids) and out.top_ids[0].tolist()[3:] == [-1, -1] and out.top_ids[2].tolist()[:2] == [4, 7]
    torch.testing.assert_close(dx, ref.grad(g, gh, gk)[0])
    assert out.logprobs[3] == 0 and out.logprobs[1] == -float("inf") and out.entropy[1] == 0 and not bool(dx[1].any())
    plain = torch.nn.functional.cross_entropy(x[[0, 2, 4]], t[[0, 2, 4]])
    torch.testing.assert_close(-L.token_logprobs(x[[0, 2, 4]], t[[0, 2, 4]]).logprobs.mean(), plain)


def test_the_64_bit_gradient_is_that_of_differences():
    torch.manual_seed(2)
    x, t = torch.randn(2, 7, dtype=torch.float64), torch.tensor([3, 6])
    g, gh, gk = (torch.randn(*s, dtype=torch.float64) for s in ((2,), (2,), (2, 3)))

    def value(y):
        r = R.Scores(y, t, 7, 3, 1.3)
        return (r.picked * g).sum() + (r.h * gh).sum() + (r.top * gk).sum()
    d, step = R.Scores(x, t, 7, 3, 1.3).grad(g, gh, gk)[0], 1e-6
    for i in range(2):
        for j in range(7):
            up, down = x.clone(), x.clone()
            up[i, j] += step
            down[i, j] -= step
            assert abs(float(value(up) - value(down)) / (2 * step) - float(d[i, j])) < 1e-8


# ---- dropout -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [dict(x=None), dict(y=None), dict(state=None), dict(n=0), dict(drop=65537), dict(type=3), dict(type=-1), dict(x=A + 2),
                                 dict(y=A + 8), dict(residual=A + 4)])
def test_dropout_entry_point_refuses(bad):
    a = dict(x=A, residual=None, y=A, state=A, copy=None, call=0, drop=100, n=8, type=0)
    a.update(bad)
    assert N.load().ccf_dropout(a["x"], a["residual"], a["y"], a["state"], a["copy"], a["call"], a["drop"], a["n"], a["type"], None) == -2


def test_dropout_refuses():
    x, s = torch.randn(4, 4), torch.tensor([1, 2])
    for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(call=-1), dict(call=2 ** 32), dict(state=s.int()), dict(state=s[:1]),
               dict(state=torch.zeros(4, dtype=torch.int64)[::2]), dict(state=s.to("meta")), dict(residual=x[:2]), dict(residual=x.double())):
        with pytest.raises(ValueError):
            D.dropout(**{"x": x, "p": 0.5, "state": s, **kw})
    with pytest.raises(TypeError):
        D.dropout(x.long(), 0.5, s)
    with pytest.raises(ValueError):
        D.Dropout(2.0, D.DropoutState(0))


@pytest.mark.parametrize("seed,step,call", [(0, 0, 0), (1 << 62 | 12345, 7, 3), (-5, (1 << 32) + 1, 0xFFFFFFFF)])
def test_masks_on_the_host(seed, step, call):
    state = torch.tensor([seed, step])
    bits = R.philox_bits(seed % (1 << 64), step, call, 203)
    for p in (0.0, 0.1, 0.5, 1.0):
        assert torch.equal(D.keep_mask((7, 29), p, state, call).reshape(-1), bits >= round(p * 65536))


def test_philox_of_the_paper():
    """The known answers of the generator's authors for Philox4x32-10 (Random123's test vectors, as published)."""
    def words(c, k):
        low = 0xFFFFFFFF
        k0, k1 = k
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k0, b & low, (a >> 32) ^ c[3] ^ k1, a & low]
            k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
        return c
    assert words([0, 0, 0, 0], (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    low = 0xFFFFFFFF
    assert words([low] * 4, (low, low)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    bits = R.philox_bits(0, 0, 0, 8).tolist()
    assert bits == [0xe8d5, 0x6627, 0xc58d, 0xe169, 0xac4c, 0xbc57, 0xdbd8, 0x9b00]


def test_dropout_on_the_host():
    x = torch.randn(33, 7, dtype=torch.float64, requires_grad=True)
    r = torch.randn(33, 7, dtype=torch.float64, requires_grad=True)
    state = torch.tensor([9, 4])
    y = D.dropout(x, 0.25, state, 2, residual=r)
    keep = (R.philox_bits(9, 4, 2, 231) >= 16384).view(33, 7)
    torch.testing.assert_close(y, r + keep * x * (65536 / (65536 - 16384)))
    dy = torch.randn_like(y)
    dx, dr = torch.autograd.grad(y, [x, r], dy)
    torch.testing.assert_close(dx, keep * dy * (65536 / (65536 - 16384)))
    assert torch.equal(dr, dy)
    bad = torch.full((64,), float("nan"))
    assert bool((D.dropout(bad, 1.0, state) == 0).all())
    rng = D.DropoutState(3)
    m = D.Dropout(0.5, rng)
    one, two = m(torch.ones(64)), m(torch.ones(64))
    assert not torch.equal(one, two) and torch.equal(m.eval()(one), one)
    rng.advance()
    assert rng.tensor.tolist() == [3, 1] and rng.calls == 2


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_repeated_forward_pass_draws_the_same_masks(device):
    """Activation checkpointing: the gradients of the same pass without it, also where the state has moved on; refused where the masks would differ."""
    from torch.utils.checkpoint import checkpoint
    w = torch.arange(1.0, 65.0, device=device)

    def run(wrap, later):
        rng = D.DropoutState(5, device)
        drop = D.Dropout(0.5, rng)
        x = w.clone().requires_grad_(True)

        def block(h):
            return drop(drop(h * w).sin(), residual=h)

        rng.begin_step(x.device)
        y = wrap(rng, block, wrap(rng, block, x))
        if later:
            rng.begin_step(x.device)
            drop(w)
        y.sum().backward(retain_graph=True)
        one = x.grad.clone()
        y.sum().backward()
        assert torch.equal(x.grad, one + one)
        return y.detach(), one, rng.tensor.tolist(), rng.calls

    for later in (False, True):
        plain = run(lambda rng, f, h: f(h), later)
        again = run(lambda rng, f, h: checkpoint(f, h, use_reentrant=False, context_fn=rng.recomputed), later)
        assert torch.equal(plain[0], again[0]) and torch.equal(plain[1], again[1]) and plain[2:] == again[2:]
        for reentrant in (False, True):
            with pytest.raises(RuntimeError, match="other masks"):
                run(lambda rng, f, h: checkpoint(f, h, use_reentrant=reentrant), later)
