"""Tokens sorted by expert and back on the host: refusals of the functions and of the C entry points, the torch path against loops in 64 bits and against differences,
the row count, traced and fake tensors. No GPU, made-up addresses."""
import ctypes as C

import pytest
import token_refs as R
import torch
import training_refs as T

from ccfuser_b200 import native as N
from ccfuser_b200.ops import expert_sort as S

A = 1 << 20      # an address that nothing reads


def _order(**kw):
    o = N.Order(idx=A, slot_row=A, row_slot=A, counts=A, base=A, scratch=A, slots=8, rows=8, capacity=8, experts=4, align=1, wide=1)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


def _rows(**kw):
    r = N.Rows(tokens_in=A, rows_in=A, tokens_out=A, rows_out=A, slot_row=A, row_slot=A, weights=A, d_weights=A, tokens=4, rows=8, ld=16, top_k=2, d=16, type=0,
               weight_type=2)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("bad", [dict(slots=0), dict(slots=2 ** 30 + 1), dict(experts=0), dict(experts=1025), dict(capacity=0), dict(align=0), dict(align=65537), dict(rows=7),
                                 dict(rows=9), dict(idx=None), dict(slot_row=None), dict(row_slot=None), dict(counts=None), dict(base=None),
                                 dict(slots=5000, rows=5000, capacity=5000, scratch=None)])
def test_order_entry_point_refuses(bad):
    assert N.load().ccf_order(C.byref(_order(**bad)), None) == -2
    if "scratch" not in bad:
        assert N.load().ccf_sort_by_expert(C.byref(_order(**bad)), C.byref(_rows()), None) == -2


@pytest.mark.parametrize("bad", [dict(tokens=0), dict(tokens=2 ** 30 + 1), dict(tokens=2 ** 29, top_k=3), dict(top_k=0), dict(d=0), dict(d=2 ** 24 + 1), dict(rows=-1),
                                 dict(rows=2 ** 31), dict(type=3), dict(type=-1), dict(weight_type=3), dict(slot_row=None)])
def test_row_entry_points_refuse(bad):
    lib, r = N.load(), _rows(**bad)
    assert lib.ccf_sort_rows(C.byref(r), 0, None) == lib.ccf_return_rows(C.byref(r), None) == lib.ccf_return_rows_bwd(C.byref(r), None) == -2
    assert lib.ccf_sort_by_expert(C.byref(_order()), C.byref(r), None) == -2


def test_row_entry_points_refuse_missing_memory_and_elements_cut_in_two():
    lib = N.load()
    for bad in (dict(tokens_in=None), dict(rows_out=None), dict(row_slot=None), dict(ld=15), dict(tokens_in=A + 1), dict(rows_out=A + 2, type=2)):
        assert lib.ccf_sort_rows(C.byref(_rows(**bad)), 0, None) == -2
    for bad in (dict(tokens_out=None), dict(rows_in=None), dict(rows_in=A + 1)):
        assert lib.ccf_return_rows(C.byref(_rows(**bad)), None) == -2
    for bad in (dict(tokens_in=None), dict(rows_in=None), dict(row_slot=None), dict(ld=15)):
        assert lib.ccf_return_rows_bwd(C.byref(_rows(**bad)), None) == -2
    # an order for other rows
    for bad in (dict(tokens=3), dict(rows=9), dict(slot_row=2 * A), dict(row_slot=2 * A)):
        assert lib.ccf_sort_by_expert(C.byref(_order()), C.byref(_rows(**bad)), None) == -2
    assert lib.ccf_return_rows_bwd(C.byref(_rows(rows_out=None, d_weights=None)), None) == 0      # nothing to do


def test_row_counts():
    lib = N.load()
    for slots, experts, capacity, align in ((0, 4, 1, 8), (8, 4, 8, 1), (8, 4, 1, 1), (8, 4, 8, 128), (3, 64, 3, 16), (100, 7, 10, 4), (2 ** 30, 1024, 2 ** 30, 1)):
        want = S.order_rows(slots, experts, capacity, align)
        assert lib.ccf_order_rows(slots, experts, capacity, align) == want
        assert want % align == 0
    assert lib.ccf_order_rows(2 ** 30, 1024, 2 ** 30, 65536) == S.order_rows(2 ** 30, 1024, None, 65536) == 2 ** 30 + 1023 * 65536
    assert lib.ccf_order_rows(-1, 4, 1, 1) == lib.ccf_order_rows(8, 0, 1, 1) == lib.ccf_order_rows(8, 4, 0, 1) == lib.ccf_order_rows(8, 4, 1, 0) == -1
    assert lib.ccf_order_scratch(512, 65) == 0 < lib.ccf_order_scratch(513, 65) == 2 * 65 * 4 and lib.ccf_order_scratch(1024, 1024) == 0
    assert lib.ccf_order_scratch(0, 4) == lib.ccf_order_scratch(8, 0) == lib.ccf_order_scratch(8, 1025) == -1


def test_functions_refuse():
    x, idx = torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for bad in (idx.float(), idx.short(), idx.bool()):
        with pytest.raises(TypeError):
            S.sort_by_expert(x, bad, 4)
    for kw in (dict(num_experts=0), dict(num_experts=1025), dict(num_experts=4, capacity=0), dict(num_experts=4, align=0), dict(num_experts=4, align=65537)):
        with pytest.raises(ValueError):
            S.sort_by_expert(x, idx, **kw)
        with pytest.raises(ValueError):
            S.expert_order(idx, **kw)
    with pytest.raises(ValueError):
        S.expert_order(torch.tensor(0), 4)
    for bad in (x[:3], x[0], x[None], x.to("meta")):
        with pytest.raises(ValueError):
            S.sort_by_expert(bad, idx, 4)
    with pytest.raises(TypeError):
        S.sort_by_expert(x.int(), idx, 4)
    rows, order = S.sort_by_expert(x, idx, 4)
    w = torch.rand(4, 2)
    for bad in (rows[1:], rows[0], rows[None], rows.to("meta")):
        with pytest.raises(ValueError):
            S.return_rows(bad, order, w)
    for bad in (w[:3], w[:, :1], w.to("meta")):
        with pytest.raises(ValueError):
            S.return_rows(rows, order, bad)
    with pytest.raises(TypeError):
        S.return_rows(rows, order, w.int())
    with pytest.raises(TypeError):
        S.return_rows(rows.int(), order, w)
    with pytest.raises(TypeError):
        S.sort_rows(x, order._replace(slot_row=order.slot_row.long()))
    with pytest.raises(ValueError):
        S.sort_rows(x, order._replace(row_slot=order.row_slot[None]))
    with pytest.raises(ValueError):
        S.sort_rows(x[:3], order)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("shape,experts,capacity,align", [((1, 1), 1, None, 1), ((7, 3), 5, None, 4), ((2, 9, 2), 4, 3, 1), ((40, 4), 64, None, 128), ((3,), 8, 1, 16), ((0, 2), 3, None, 8)])
def test_order_and_values(shape, experts, capacity, align, wide):
    g = torch.Generator().manual_seed(len(shape) + experts)
    idx = torch.randint(-1, experts + 1, shape, generator=g, dtype=torch.int64 if wide else torch.int32)
    order = S.expert_order(idx, experts, capacity, align)
    T.check_order(order, idx, experts, capacity, align)
    for dt in (torch.bfloat16, torch.float16, torch.float32, torch.float64):
        x, w = torch.randn(*shape[:-1], 6, generator=g).to(dt), torch.rand(*shape, generator=g)
        rows = S.sort_rows(x, order)
        assert torch.equal(rows, T.sorted_rows(x, order.row_slot, shape[-1]))
        for weights in (w, w.to(dt), None):
            y = S.return_rows(rows, order, weights)
            ref, size = T.returned(rows, order.slot_row, weights)
            assert y.dtype == dt and y.shape == x.shape
            R.assert_close(y, ref, shape[-1] * R.U * size)


def test_gradients_by_differences():
    """In 64 bits, with slots that have no row and rows that have no slot, first and second order."""
    idx = torch.tensor([[0, 2], [2, -1], [1, 2], [2, 0]])
    order = S.expert_order(idx, 3, capacity=2, align=4)
    assert int((order.slot_row < 0).sum()) == 3 and int((order.row_slot < 0).sum()) > 0
    x = torch.randn(4, 3, dtype=torch.float64, requires_grad=True)
    rows = torch.randn(order.row_slot.numel(), 3, dtype=torch.float64, requires_grad=True)
    w = torch.rand(4, 2, dtype=torch.float64, requires_grad=True)
    for f, args in ((lambda x: S.sort_rows(x, order), (x,)), (lambda r, w: S.return_rows(r, order, w), (rows, w)), (lambda r: S.return_rows(r, order), (rows,))):
        assert torch.autograd.gradcheck(f, args) and torch.autograd.gradgradcheck(f, args)


def test_masked_places_do_not_count():
    idx = torch.tensor([[0, -1], [-1, -1], [1, 0]])
    order = S.expert_order(idx, 2, align=4)
    rows = torch.where((order.row_slot < 0)[:, None], torch.nan, torch.ones(order.row_slot.numel(), 5))
    y = S.return_rows(rows, order, torch.tensor([[1.0, torch.nan], [torch.inf, torch.nan], [2.0, 3.0]]))
    assert y[:, 0].tolist() == [1, 0, 5]


def test_meta_tensors():
    x, idx = torch.empty(5, 8, device="meta", dtype=torch.bfloat16), torch.empty(5, 2, dtype=torch.int32, device="meta")
    rows, order = S.sort_by_expert(x, idx, 4, capacity=3, align=8)
    assert rows.shape == (S.order_rows(10, 4, 3, 8), 8) and S.return_rows(rows, order, torch.empty(5, 2, device="meta")).shape == (5, 8)


def test_fake_tensors_and_compile():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, idx = torch.empty(5, 8), torch.empty(5, 2, dtype=torch.int32)
        rows, order = S.sort_by_expert(x, idx, 4, align=8)
        assert rows.shape == (S.order_rows(10, 4, None, 8), 8) and S.return_rows(rows, order).shape == (5, 8)
    x, idx = torch.randn(5, 8), torch.randint(0, 4, (5, 2))
    f = lambda x, idx: S.return_rows(S.sort_by_expert(x, idx, 4, align=8)[0] * 2, S.expert_order(idx, 4, align=8))  # noqa: E731
    out = torch.compile(f, backend="eager", fullgraph=True)(x, idx)
    assert torch.equal(out, f(x, idx))
