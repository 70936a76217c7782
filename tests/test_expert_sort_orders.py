"""Orders that are not whole: a slot's row behind the last is none, a row's slot behind the last neither. On the host and on a GPU, whose paths by torch's operations
(fp64, second derivatives) would end the process over such a number."""
import pytest
import torch

from ccfuser_b200.ops.expert_sort import ExpertOrder, expert_order, return_rows, sort_rows


def _cut(device):
    """An order of 12 tokens without the last of its rows, as one who knows how many are filled may hand it on, and the same with -1 in their place."""
    idx = torch.randint(0, 3, (12, 2), generator=torch.Generator().manual_seed(3))
    whole = expert_order(idx, 3, align=4)
    rows = int(whole.base[2]) + 1
    assert 0 < rows < int(whole.base[3]) and int((whole.slot_row >= rows).sum()) > 1
    marked = whole._replace(slot_row=torch.where(whole.slot_row >= rows, -1, whole.slot_row), row_slot=whole.row_slot[:rows])
    return [ExpertOrder(*(t.to(device) for t in o)) for o in (whole._replace(row_slot=whole.row_slot[:rows]), marked)]


def _results(order, dtype, device, twice):
    g = torch.Generator().manual_seed(4)
    x, rows, w, dy, drows = (torch.randn(s, generator=g).to(device=device, dtype=dtype) for s in ((12, 8), (order.row_slot.numel(), 8), (12, 2), (12, 8), (order.row_slot.numel(), 8)))
    w = w.masked_fill(order.slot_row.eq(-1) | order.slot_row.ge(rows.shape[0]), torch.nan)      # of a slot without a row: not looked at
    x, rows, w = (t.requires_grad_(True) for t in (x, rows, w))
    out = []
    for f, args, dout in ((lambda: sort_rows(x, order), [x], drows), (lambda: return_rows(rows, order, w), [rows, w], dy), (lambda: return_rows(rows, order), [rows], dy)):
        y = f()
        dout = dout.detach().requires_grad_(twice)
        grads = torch.autograd.grad(y, args, dout, create_graph=twice)
        out += [y.detach()] + [t.detach() for t in grads]
        if twice:
            out += [t.detach() for t in torch.autograd.grad([t.nansum() for t in grads], [dout])]
    return out


@pytest.mark.parametrize("twice", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_behind_the_last_are_none(device, dtype, twice):
    cut, marked = _cut(device)
    for a, b in zip(_results(cut, dtype, device, twice), _results(marked, dtype, device, twice)):
        assert torch.equal(a.nan_to_num(nan=-77.0), b.nan_to_num(nan=-77.0)) and not a[..., 0].isnan().all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_slots_behind_the_last_are_none(device):
    """By torch's operations such a row is zeros."""
    order = ExpertOrder(*(torch.tensor(v, dtype=torch.int32, device=device) for v in ([[0], [2]], [0, 2, 1, 7], [4], [0, 4])))
    x = torch.arange(1.0, 7.0, dtype=torch.float64, device=device).view(2, 3)
    assert sort_rows(x, order).tolist() == [[1, 2, 3], [0, 0, 0], [4, 5, 6], [0, 0, 0]]


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("device", [pytest.param("cuda", marks=pytest.mark.gpu)])
def test_second_derivatives_do_not_see_the_weight_of_a_slot_without_a_row(device, bad):
    """The first slot's, which rows without a slot would read."""
    idx = torch.tensor([[-1, 0], [1, 0], [0, 1]], device=device)
    order = expert_order(idx, 2, align=4)
    assert int((order.row_slot < 0).sum()) > 0
    g = torch.Generator().manual_seed(5)
    rows, w, dy, c = (torch.randn(s, generator=g).to(device) for s in ((order.row_slot.numel(), 8), (3, 2), (3, 8), (order.row_slot.numel(), 8)))
    got = []
    for value in (1.0, bad):
        w[0, 0] = value
        args = [t.clone().requires_grad_(True) for t in (rows, w, dy)]
        d_rows, d_w = torch.autograd.grad(return_rows(args[0], order, args[1]), args[:2], args[2], create_graph=True)
        got.append([t.detach() for t in (d_rows, d_w) + torch.autograd.grad((d_rows * c).sum() + d_w.square().sum(), args)])
    for a, b in zip(*got):
        assert a.isfinite().all() and torch.equal(a, b)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_spreading_does_not_see_it_either(bad):
    """The same operations on the host, as the Python nodes take them."""
    from ccfuser_b200.ops.expert_sort import _spread
    idx = torch.tensor([[-1, 0], [1, 0], [0, 1]])
    order = expert_order(idx, 2, align=4)
    dy, w = torch.ones(3, 8, requires_grad=True), torch.tensor([[bad, 1.0], [2.0, 3.0], [4.0, 5.0]], requires_grad=True)
    out = _spread(dy, order.slot_row, order.row_slot, w)
    d, dw = torch.autograd.grad(out, [dy, w], torch.ones_like(out))
    assert out.isfinite().all() and d[:, 0].tolist() == [1.0, 5.0, 9.0] and dw.tolist() == [[0.0, 8.0], [8.0, 8.0], [8.0, 8.0]]
