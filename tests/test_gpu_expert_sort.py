"""Tokens sorted by expert and back (csrc/expert_sort.cu): the order against loops, rows and gradients against 64 bits at the edges of vectors, pieces, warps,
blocks and tiles; masks, capacities, strides, alignment, streams, captured calls."""
import pytest
import token_refs as R
import torch
import training_refs as T

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _idx(g, tokens, k, experts, wide=False, none=0.1, skew=0):
    """Choices that leave some slots without an expert, by numbers on either side of the range; with skew most go to one expert."""
    idx = torch.randint(0, experts, (tokens, k), generator=g, device="cuda")
    if skew:
        idx[torch.rand(tokens, k, generator=g, device="cuda") < 0.8] = experts - 1
    off = torch.rand(tokens, k, generator=g, device="cuda")
    idx[off < none / 2] = -1
    idx[(off >= none / 2) & (off < none)] = experts + 3
    return idx if wide else idx.int()


# one block up to 32 threads' worth of slots and more, several blocks, eight slots a thread, several tiles a block
@pytest.mark.parametrize("tokens,k,experts,capacity,align", [
    (1, 1, 1, None, 1), (1, 2, 64, None, 128), (5, 3, 7, None, 1), (31, 1, 3, None, 16), (33, 1, 3, 2, 1), (16, 2, 64, None, 1), (512, 2, 256, None, 16),
    (513, 2, 1024, 1, 3), (1025, 1, 5, 100, 128), (4096, 8, 33, None, 128), (16384, 2, 64, 300, 1), (9001, 4, 256, None, 128), (70001, 3, 8, None, 7),
    (40000, 8, 300, 1000, 16), (300001, 1, 2, None, 1)])
def test_order(tokens, k, experts, capacity, align):
    from ccfuser_b200.ops.expert_sort import expert_order
    g = _gen(tokens)
    for wide, skew in ((False, 0), (True, 1)):
        idx = _idx(g, tokens, k, experts, wide, skew=skew)
        got = expert_order(idx, experts, capacity, align)
        T.check_order(got, idx, experts, capacity, align)


def test_order_without_and_with_one_expert():
    from ccfuser_b200.ops.expert_sort import expert_order
    for value, experts in ((-1, 9), (9, 9), (8, 9), (0, 1), (2 ** 40, 9), (-2 ** 40, 9)):
        idx = torch.full((700, 3), value, device="cuda")
        T.check_order(expert_order(idx, experts, 1000, 4), idx, experts, 1000, 4)


@pytest.mark.parametrize("dtype", list(TYPES))
# units of 2, 4, 8 and 16 bytes; one lane to several pieces of a row; slots in one, two and more rounds
@pytest.mark.parametrize("tokens,k,experts,d,capacity,align", [
    (1, 1, 1, 1, None, 1), (1, 2, 8, 2048, None, 16), (3, 2, 4, 7, None, 2), (17, 3, 5, 8, None, 1), (64, 1, 4, 30, 8, 8), (33, 4, 6, 100, None, 128),
    (65, 8, 16, 64, None, 1), (130, 9, 12, 24, 50, 4), (257, 2, 64, 1032, None, 128), (40, 6, 8, 4100, None, 1), (1000, 2, 7, 765, 200, 1), (2500, 5, 32, 136, None, 16)])
def test_rows_and_gradients(dtype, tokens, k, experts, d, capacity, align):
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    dt, g = TYPES[dtype], _gen(d + k)
    idx = _idx(g, tokens, k, experts)
    x = torch.randn(tokens, d, generator=g, device="cuda").to(dt).requires_grad_(True)
    rows, order = sort_by_expert(x, idx, experts, capacity, align)
    T.check_order(order, idx, experts, capacity, align)
    assert torch.equal(rows.cpu(), T.sorted_rows(x, order.row_slot, k))
    g_rows = torch.randn(rows.shape, generator=g, device="cuda").to(dt)
    dx, = torch.autograd.grad(rows, [x], g_rows)
    ref, size = T.returned(g_rows, order.slot_row)
    R.assert_close(dx, ref, k * R.U * size, "dx")

    for weight_type in (torch.float32, dt):
        values = torch.randn(rows.shape, generator=g, device="cuda").to(dt).requires_grad_(True)
        w = torch.rand(tokens, k, generator=g, device="cuda").to(weight_type).requires_grad_(True)
        y = return_rows(values, order, w)
        ref, size = T.returned(values, order.slot_row, w)
        R.assert_close(y, ref, k * R.U * size, "y")
        dy = torch.randn(tokens, d, generator=g, device="cuda").to(dt)
        d_rows, d_w = torch.autograd.grad(y, [values, w], dy)
        ref, ref_w, size_w = T.return_grads(dy, values, order.slot_row, order.row_slot, w)
        R.assert_close(d_rows, ref, R.U * ref.abs(), "d_rows")
        # a lane's chain of products, five exchanges and up to eight warps
        R.assert_close(d_w, ref_w, (d / 32 + 32) * R.U * size_w, "d_w")
        assert bool((d_w[order.slot_row < 0] == 0).all())
        for need in ((values,), (w,)):
            y = return_rows(values if need[0] is values else values.detach(), order, w if need[0] is w else w.detach())
            one, = torch.autograd.grad(y, need, dy)
            assert torch.equal(one, d_rows if need[0] is values else d_w)
    y = return_rows(values, order)
    ref, size = T.returned(values, order.slot_row)
    R.assert_close(y, ref, k * R.U * size, "sum")


def test_nothing_of_rows_without_a_slot_or_of_weights_without_a_row():
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    idx = torch.tensor([[0, -1], [-1, -1], [1, 0], [5, 1]], device="cuda")
    x = torch.full((4, 96), float("inf"), device="cuda", dtype=torch.bfloat16)
    x[1] = float("nan")
    rows, order = sort_by_expert(x, idx, 2, align=8)
    empty = order.row_slot < 0
    assert bool((rows[empty] == 0).all()) and bool(torch.isinf(rows[~empty]).all())      # the token of NaN has no row
    rows = torch.where(empty[:, None], torch.full_like(rows, float("nan")), torch.ones_like(rows)).requires_grad_(True)
    w = torch.tensor([[1.0, float("nan")], [float("inf"), float("nan")], [2.0, 3.0], [float("nan"), 4.0]], device="cuda", requires_grad=True)
    y = return_rows(rows, order, w)
    assert y[:, 0].tolist() == [1.0, 0.0, 5.0, 4.0]
    d_rows, d_w = torch.autograd.grad(y, [rows, w], torch.ones_like(y))
    assert bool((d_rows[empty] == 0).all()) and d_w.tolist() == [[96, 0], [0, 0], [96, 96], [0, 96]]


def test_strides_alignment_shapes_and_the_python_functions(monkeypatch):
    from ccfuser_b200 import native as N
    from ccfuser_b200.ops.expert_sort import expert_order, return_rows, sort_by_expert, sort_rows
    g = _gen(3)
    wide = torch.randn(6, 7, 72, generator=g, device="cuda").half()
    idx = _idx(g, 42, 3, 5).view(6, 7, 3).transpose(1, 2).contiguous().transpose(1, 2)
    weights = torch.rand(6, 3, 7, generator=g, device="cuda").transpose(1, 2)
    runs = []
    for module in (N.torch_module, lambda: None):
        monkeypatch.setattr(N, "torch_module", module)
        for x in (wide[..., 3:67], wide[..., ::2], wide[:, :, :64], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :64]):
            x = x.detach().requires_grad_(True)
            rows, order = sort_by_expert(x, idx, 5, align=4)
            T.check_order(order, idx, 5, None, 4)
            assert torch.equal(rows.cpu(), T.sorted_rows(x, order.row_slot, 3)) and torch.equal(rows, sort_rows(x, expert_order(idx, 5, align=4)))
            storage = torch.randn(rows.shape[0] * (rows.shape[1] + 1) + 1, generator=_gen(4), device="cuda").half()
            for values in (storage[1:1 + rows.numel()].view(rows.shape), storage[:-1].view(rows.shape[0], -1)[:, 1:], storage[:rows.numel()].view(rows.shape[1], -1).t()):
                values, w = values.detach().requires_grad_(True), weights.detach().requires_grad_(True)
                y = return_rows(values, order, w)
                assert y.shape == x.shape
                ref, size = T.returned(values, order.slot_row, w)
                R.assert_close(y, ref, 3 * R.U * size, "y")
                dy = torch.randn(7, 6, x.shape[-1], generator=_gen(5), device="cuda").half().transpose(0, 1)
                d_rows, d_w = torch.autograd.grad(y, [values, w], dy)
                dx, = torch.autograd.grad(rows, [x], values.detach(), retain_graph=True)
                runs.append((y, d_rows, d_w, dx))
    half = len(runs) // 2
    for a, b in zip(runs[:half], runs[half:]):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_empty_calls():
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    for tokens, k, d in ((0, 2, 8), (3, 0, 8), (3, 2, 0)):
        x = torch.randn(tokens, d, device="cuda", requires_grad=True)
        idx = torch.zeros(tokens, k, dtype=torch.int32, device="cuda")
        rows, order = sort_by_expert(x, idx, 4, align=8)
        assert rows.shape[0] == order.row_slot.shape[0] and order.counts.sum() == tokens * k
        y = return_rows(rows, order, torch.rand(tokens, k, device="cuda"))
        assert y.shape == (tokens, d)
        y.sum().backward()
        assert x.grad.shape == x.shape and bool((x.grad == 0).all() if k == 0 else True)


def test_an_order_that_names_rows_it_has_not():
    """Row numbers behind the rows are no rows; nothing is read or written there."""
    from ccfuser_b200.ops.expert_sort import ExpertOrder, return_rows
    slot_row = torch.tensor([[0, 4], [2 ** 31 - 1, 1], [-7, 3]], dtype=torch.int32, device="cuda")
    order = ExpertOrder(slot_row, torch.tensor([0, 3, -1, 5], dtype=torch.int32, device="cuda"), None, None)
    rows = torch.arange(1, 5, device="cuda", dtype=torch.float32)[:, None].expand(4, 32).contiguous().requires_grad_(True)
    y = return_rows(rows, order)
    assert y[:, 0].tolist() == [1, 2, 4]
    d_rows, = torch.autograd.grad(y, [rows], torch.ones_like(y))
    assert d_rows[:, 0].tolist() == [1, 1, 0, 1]


def test_second_derivatives_and_versions():
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(7)
    idx = _idx(g, 6, 2, 3)
    x = torch.randn(6, 5, generator=g, device="cuda", requires_grad=True)
    w = torch.rand(6, 2, generator=g, device="cuda", requires_grad=True)

    def there_and_back(x, w):
        rows, order = sort_by_expert(x, idx, 3, align=4)
        return return_rows(rows * rows, order, w)

    # differences of fp32 results: a step of 2^-6 leaves 2^-24 / 2^-6 of the values (at most 16) and nothing of third order in w, and the cubes' in x
    y = there_and_back(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w], create_graph=True)
    total = (dx * dx).sum() + (dw * dw).sum()
    gx, gw = torch.autograd.grad(total, [x, w])
    xd, wd = x.detach().double().cpu().requires_grad_(True), w.detach().double().cpu().requires_grad_(True)
    on = ((idx >= 0) & (idx < 3)).double().cpu()
    yd = (xd * xd) * (wd * on).sum(dim=1, keepdim=True)
    dxd, dwd = torch.autograd.grad(yd.sum(), [xd, wd], create_graph=True)
    gxd, gwd = torch.autograd.grad((dxd * dxd).sum() + (dwd * dwd).sum(), [xd, wd])
    for got, ref in ((dx, dxd), (dw, dwd), (gx, gxd), (gw, gwd)):
        R.assert_close(got, ref.detach(), 64 * R.U * (1 + ref.detach().abs().max()))
    rows, order = sort_by_expert(x.detach(), idx, 3)
    rows = rows.requires_grad_(True)
    y = return_rows(rows, order, w)
    with torch.no_grad():
        rows.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_streams_and_captured_calls():
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(9)
    data = []
    for i in range(2):
        idx, x, w = _idx(g, 3000, 2, 16), torch.randn(3000, 256, generator=g, device="cuda").bfloat16(), torch.rand(3000, 2, generator=g, device="cuda")
        data.append((idx, x.requires_grad_(True), w.requires_grad_(True), torch.randn(3000, 256, generator=g, device="cuda").bfloat16()))

    def call(idx, x, w, dy):
        rows, order = sort_by_expert(x, idx, 16, align=16)
        y = return_rows(rows, order, w)
        return (rows, *order, y, *torch.autograd.grad(y, [x, w], dy))

    want = [call(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):      # two streams at once
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(run, want[i]))
    del got
    static = [t.detach().clone().requires_grad_(t.requires_grad) for t in data[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]):
        call(*static)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = call(*static)
    for i in (1, 0, 1):
        with torch.no_grad():
            for s, t in zip(static, data[i]):
                s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_transforms_take_torch_operations():
    from ccfuser_b200.ops.expert_sort import ExpertOrder, return_rows, sort_by_expert, sort_rows
    g = _gen(11)
    idx = _idx(g, 20, 2, 4)
    x, w = torch.randn(20, 16, generator=g, device="cuda"), torch.rand(20, 2, generator=g, device="cuda")

    def f(x, w):
        rows, order = sort_by_expert(x, idx, 4, align=4)
        return return_rows(rows, order, w)

    y = f(x, w)
    with torch.autograd.forward_ad.dual_level():
        out = f(torch.autograd.forward_ad.make_dual(x, x), w)
        tangent = torch.autograd.forward_ad.unpack_dual(out).tangent
    R.assert_close(tangent, y.double(), 8 * R.U * y.double().abs())      # linear in x
    order = sort_by_expert(x, idx, 4)[1]
    batch = torch.func.vmap(lambda v: return_rows(sort_rows(v, order), order, w))(torch.stack([x, 2 * x]))
    R.assert_close(batch[1], 2 * y.double(), 16 * R.U * y.double().abs())
    gx = torch.func.grad(lambda v: f(v, w).sum())(x)
    xs = x.clone().requires_grad_(True)
    f(xs, w).sum().backward()
    R.assert_close(gx, xs.grad.double(), 8 * R.U * xs.grad.double().abs())
    assert isinstance(order, ExpertOrder)


@pytest.mark.parametrize("tokens,k,experts,capacity,align", [(700000, 2, 8, None, 16), (300000, 8, 100, 20000, 1), (1100000, 1, 300, None, 128)])
def test_orders_of_many_tiles(tokens, k, experts, capacity, align):
    """More slots than a wave of blocks holds at a time, against torch's operations on the host (which are tested against loops)."""
    from ccfuser_b200.ops.expert_sort import expert_order
    idx = _idx(_gen(k), tokens, k, experts, skew=1)
    for got, want in zip(expert_order(idx, experts, capacity, align), expert_order(idx.cpu(), experts, capacity, align)):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("tokens,d", [(70001, 32768), (33000, 65537)])
def test_more_than_two_to_the_31_elements(tokens, d):
    """Rows of 16 bytes and odd ones; a third of the tokens is looked at."""
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(d)
    idx = _idx(g, tokens, 1, 5)
    x = torch.empty(tokens, d, device="cuda", dtype=torch.bfloat16).normal_(0, 1, generator=g).requires_grad_(True)
    rows, order = sort_by_expert(x, idx, 5)
    look = torch.arange(0, order.row_slot.numel(), 3, device="cuda")
    look = look[order.row_slot[look] >= 0]
    assert bool((rows.detach()[look] == x.detach()[order.row_slot[look].long()]).all())
    w = torch.rand(tokens, 1, device="cuda", generator=g)
    values = rows.detach().requires_grad_(True)
    y = return_rows(values, order, w)
    token = torch.arange(1, tokens, 3, device="cuda")
    on = order.slot_row[token, 0] >= 0
    want = torch.where(on[:, None], x.detach()[token].float() * w[token], 0.0).bfloat16()
    assert torch.equal(y.detach()[token], want)
    d_rows, = torch.autograd.grad(y, [values], y.detach())
    want = torch.where((order.row_slot[look] >= 0)[:, None], (y.detach().float()[order.row_slot[look].long()] * w[order.row_slot[look].long()]), 0.0).bfloat16()
    assert torch.equal(d_rows[look], want)
    dx, = torch.autograd.grad(rows, [x], d_rows)
    assert torch.equal(dx[token], torch.where(on[:, None], d_rows[order.slot_row[token, 0].clamp(min=0).long()], torch.zeros((), dtype=dx.dtype, device="cuda")))


def test_inference_mode_saved_tensor_hooks_and_recomputation():
    from torch.utils.checkpoint import checkpoint

    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(21)
    idx = _idx(g, 90, 2, 6)
    x, w = torch.randn(90, 40, generator=g, device="cuda").half().requires_grad_(True), torch.rand(90, 2, generator=g, device="cuda").requires_grad_(True)

    def f(x, w):
        rows, order = sort_by_expert(x, idx, 6, align=4)
        return return_rows(torch.tanh(rows), order, w)

    want = torch.autograd.grad(f(x, w), [x, w], torch.ones(90, 40, device="cuda").half())
    with torch.inference_mode():
        y = f(x, w)
    assert torch.equal(y.clone(), f(x, w).detach())
    strided = lambda t: t if t.dim() == 0 else torch.stack([t, t], dim=-1)[..., 1]  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: strided(t.cuda())):
        y = f(x, w)
    got = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    again = checkpoint(f, x, w, use_reentrant=False)
    third = torch.autograd.grad(again, [x, w], torch.ones_like(again))
    for a, b, c in zip(want, got, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_calls_from_two_threads():
    import threading

    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(22)
    sets = [(_idx(g, 2000, 2, 16), torch.randn(2000, 129, generator=g, device="cuda")) for _ in range(2)]
    want, got = [], [[], []]

    def call(i):
        rows, order = sort_by_expert(sets[i][1], sets[i][0], 16)
        return return_rows(rows, order)

    want = [call(i) for i in range(2)]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(call(i))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(r) == 20 and torch.equal(y, want[i]) for i, r in enumerate(got) for y in r)


def test_traced_calls():
    """A trace holds the order as operations of torch and the rows as functions of their own: other inputs give other rows."""
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(23)

    def f(x, idx, w):
        rows, order = sort_by_expert(x, idx, 6, align=4)
        return return_rows(rows * 2, order, w)

    sets = [(torch.randn(50, 24, generator=g, device="cuda"), _idx(g, 50, 2, 6), torch.rand(50, 2, generator=g, device="cuda")) for _ in range(2)]
    traced = torch.jit.trace(f, sets[0], check_trace=False)
    for s in sets:
        assert torch.equal(traced(*s), f(*s))


@pytest.mark.parametrize("shape,d", [((2,), 16), ((3,), 7), ((2, 3, 4, 2), 40), ((1, 1, 5), 33)])
def test_tokens_of_any_shape(shape, d):
    from ccfuser_b200.ops.expert_sort import return_rows, sort_by_expert
    g = _gen(24)
    idx = torch.randint(0, 4, shape, generator=g, device="cuda")
    x, w = torch.randn(*shape[:-1], d, generator=g, device="cuda").requires_grad_(True), torch.rand(shape, generator=g, device="cuda").requires_grad_(True)
    rows, order = sort_by_expert(x, idx, 4, align=2)
    T.check_order(order, idx, 4, None, 2)
    y = return_rows(rows, order, w)
    assert y.shape == x.shape
    ref, size = T.returned(rows, order.slot_row, w)
    R.assert_close(y, ref, shape[-1] * R.U * size)
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape
    R.assert_close(dx, w.detach().double().sum(dim=-1, keepdim=True).expand(x.shape), shape[-1] * 2 * R.U * w.detach().double().sum(dim=-1, keepdim=True).expand(x.shape))
