"""Tokens sorted by expert and back with the router's weights (csrc/expert_sort.cu), for experts that are not the layer's own.

    rows, order = sort_by_expert(x, idx, num_experts, align=128)     # idx [tokens, top_k]: the router's choices
    out = my_experts(rows, order.counts, order.base)                 # rows of expert e: base[e] ... base[e] + counts[e]
    y = return_rows(out, order, weights)                             # sum over a token's choices, by weight

Nothing reads the host: ``rows`` has room for every slot whatever the routing, and rows without a slot are zeros. The order is that of ``ops.routing``: inside an
expert by token, slots from ``capacity`` on dropped, an expert outside the range (-1) none. ``align=128`` is what the grouped GEMM of ``ops.gemm`` asks of
its groups (``base`` without its last element and ``counts``). Sums are taken in fp32 and rounded once; gradients of tokens, rows and weights, also of second order,
by torch's operations then. The graph's nodes are C++ (csrc/torch_training.cpp); the Python functions below stand in where that module is missing and while a
graph is traced; on the CPU, for other types and under transforms the same values come from torch's operations. The reference sorts its rows inside
its exchange (mix_moe/csrc/cuda/local_exchange.cu).
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from .. import native as N

MAX_EXPERTS, MAX_ALIGN, MAX_SLOTS, MAX_D = 1024, 65536, 2 ** 30, 2 ** 24


class ExpertOrder(NamedTuple):
    """Where the slots of a call went, all int32."""
    slot_row: torch.Tensor   # [..., top_k] row of each slot, -1: none
    row_slot: torch.Tensor   # [rows] slot (token * top_k + choice) of each row, -1: none
    counts: torch.Tensor     # [num_experts] rows of each expert
    base: torch.Tensor       # [num_experts + 1] first row of each expert, a multiple of align; the last: behind the last expert's


def order_rows(slots: int, num_experts: int, capacity: Optional[int] = None, align: int = 1) -> int:
    """Rows that hold ``slots`` slots whatever their experts are."""
    kept = slots if capacity is None else min(slots, num_experts * capacity)
    return (kept + min(num_experts, kept) * (align - 1)) // align * align


def _check_idx(idx, num_experts, capacity, align):
    if idx.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"idx is int64 or int32, not {idx.dtype}")
    if idx.dim() < 1:
        raise ValueError(f"idx: [..., top_k], got {tuple(idx.shape)}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts: 1 to {MAX_EXPERTS}, got {num_experts}")
    if capacity is not None and capacity < 1:
        raise ValueError(f"capacity: at least 1, got {capacity}")
    if not 1 <= align <= MAX_ALIGN:
        raise ValueError(f"align: 1 to {MAX_ALIGN}, got {align}")
    if idx.numel() > MAX_SLOTS:
        raise ValueError(f"{idx.numel()} slots: at most 2^30 in one call")
    if order_rows(idx.numel(), num_experts, capacity, align) > 2 ** 31 - 1:
        raise ValueError("at most 2^31 - 1 rows in one call")


def _check_tokens(x, idx):
    if x.dim() != idx.dim() or x.dim() < 1 or x.shape[:-1] != idx.shape[:-1]:
        raise ValueError(f"x: [..., d] with the tokens of the experts' ids, [..., top_k], got {tuple(x.shape)} and {tuple(idx.shape)}")
    if x.device != idx.device:
        raise ValueError(f"x is on {x.device}, the tensor beside it on {idx.device}")
    if not x.is_floating_point():
        raise TypeError(f"x: a floating type, got {x.dtype}")
    if x.shape[-1] > MAX_D:
        raise ValueError(f"at most 2^24 columns, got {x.shape[-1]}")


def _check_order(order):
    if order.slot_row.dtype != torch.int32 or order.row_slot.dtype != torch.int32:
        raise TypeError(f"an order's numbers are int32, not {order.slot_row.dtype} and {order.row_slot.dtype}")
    if order.slot_row.dim() < 1 or order.row_slot.dim() != 1 or order.slot_row.device != order.row_slot.device:
        raise ValueError(f"an order: slot_row [..., top_k] and row_slot [rows] on one device, got {tuple(order.slot_row.shape)} on {order.slot_row.device} and "
                         f"{tuple(order.row_slot.shape)} on {order.row_slot.device}")
    if order.slot_row.numel() > MAX_SLOTS or order.row_slot.numel() > 2 ** 31 - 1:
        raise ValueError("at most 2^30 slots and 2^31 - 1 rows in one call")


def _check_return(rows, order, weights):
    if rows.dim() != 2 or rows.shape[0] != order.row_slot.shape[0] or rows.device != order.slot_row.device:
        raise ValueError(f"rows: [{order.row_slot.shape[0]}, d] on {order.slot_row.device}, got {tuple(rows.shape)} on {rows.device}")
    if not rows.is_floating_point():
        raise TypeError(f"rows: a floating type, got {rows.dtype}")
    if rows.shape[1] > MAX_D:
        raise ValueError(f"at most 2^24 columns, got {rows.shape[1]}")
    if weights is not None:
        if weights.shape != order.slot_row.shape or weights.device != rows.device:
            raise ValueError(f"weights: {tuple(order.slot_row.shape)} on {rows.device}, got {tuple(weights.shape)} on {weights.device}")
        if not weights.is_floating_point():
            raise TypeError(f"weights: a floating type, got {weights.dtype}")


def _on_kernels(x, weights=None) -> bool:
    """Whether the kernels take these tensors, and have anything to do."""
    return (x.is_cuda and x.dtype in N.DTYPE_CODE and x.numel() > 0 and not N.transformed(x)
            and (weights is None or (weights.dtype in N.DTYPE_CODE and not N.transformed(weights))))


def _module():
    module = N.torch_module()
    return module if module is not None and not torch.jit.is_tracing() else None


# ---- on the kernels, from Python -----------------------------------------------------------------------------------------
def _order_py(idx, num_experts, capacity, align):
    lib, idx = N.load(), idx.contiguous()
    slots = idx.numel()
    i32 = dict(dtype=torch.int32, device=idx.device)
    o = N.Order(idx=idx.data_ptr(), slots=slots, capacity=slots if capacity is None else capacity, experts=num_experts, align=align,
                wide=int(idx.dtype == torch.int64))
    o.rows = lib.ccf_order_rows(o.slots, o.experts, o.capacity, o.align)
    scratch = torch.empty(lib.ccf_order_scratch(slots, num_experts) // 4, **i32)
    order = ExpertOrder(torch.empty(idx.shape, **i32), torch.empty(o.rows, **i32), torch.empty(num_experts, **i32), torch.empty(num_experts + 1, **i32))
    o.slot_row, o.row_slot, o.counts, o.base = (t.data_ptr() for t in order)
    o.scratch = scratch.data_ptr()
    with torch.cuda.device(idx.device):
        launches = lib.ccf_order(C.byref(o), N.stream_ptr())
    N.check(min(launches, 0), "ccf_order")
    N.count(launches)
    return order


def _args(slot_row, rows, d, dtype):
    return N.Rows(slot_row=slot_row.data_ptr(), top_k=slot_row.shape[-1], tokens=slot_row.numel() // slot_row.shape[-1], rows=rows, d=d, ld=d,
                  type=N.DTYPE_CODE[dtype])


def _token_rows(x):
    x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 and (x.shape[0] == 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _run(name, a, device, *more):
    with torch.cuda.device(device):
        N.check(getattr(N.load(), name)(C.byref(a), *more, N.stream_ptr()), name)
    N.count(1)


def _run_sort(x, slot_row, row_slot):
    x = _token_rows(x)
    rows = torch.empty(row_slot.shape[0], x.shape[1], dtype=x.dtype, device=x.device)
    a = _args(slot_row, rows.shape[0], x.shape[1], x.dtype)
    a.tokens_in, a.row_slot, a.rows_out = x.data_ptr(), row_slot.data_ptr(), rows.data_ptr()
    a.ld = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    _run("ccf_sort_rows", a, x.device, 0)
    return rows


def _run_return(rows, slot_row, weights):
    rows = rows.contiguous()
    y = torch.empty(*slot_row.shape[:-1], rows.shape[1], dtype=rows.dtype, device=rows.device)
    a = _args(slot_row, rows.shape[0], rows.shape[1], rows.dtype)
    a.rows_in, a.tokens_out = rows.data_ptr(), y.data_ptr()
    if weights is not None:
        a.weights, a.weight_type = weights.data_ptr(), N.DTYPE_CODE[weights.dtype]
    _run("ccf_return_rows", a, rows.device)
    return y


class _SortFn(torch.autograd.Function):
    """The C++ node in Python."""

    @staticmethod
    def forward(ctx, x, slot_row, row_slot):
        ctx.save_for_backward(slot_row, row_slot)
        ctx.shape = x.shape
        return _run_sort(x, slot_row, row_slot)

    @staticmethod
    def backward(ctx, g):
        slot_row = ctx.saved_tensors[0].contiguous()
        if torch.is_grad_enabled():      # the gradient is to be differentiated in its turn
            return _slots(g, slot_row).sum(dim=-2).to(g.dtype).reshape(ctx.shape), None, None
        return _run_return(g, slot_row, None).view(ctx.shape), None, None


class _ReturnFn(torch.autograd.Function):
    """The C++ node in Python."""

    @staticmethod
    def forward(ctx, rows, slot_row, row_slot, weights):
        ctx.save_for_backward(slot_row, row_slot, weights, rows if ctx.needs_input_grad[3] else None)
        ctx.rows = rows.shape[0]
        return _run_return(rows, slot_row, None if weights is None else weights.contiguous())

    @staticmethod
    def backward(ctx, dy):
        slot_row, row_slot, weights, rows = ctx.saved_tensors
        need_rows, need_weights = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        if torch.is_grad_enabled():
            g = _spread(dy, slot_row, row_slot, weights) if need_rows else None
            return g, None, None, ((_slots(rows, slot_row) * dy.float().unsqueeze(-2)).sum(dim=-1).to(weights.dtype) if need_weights else None)
        slot_row, row_slot, d = slot_row.contiguous(), row_slot.contiguous(), dy.shape[-1]
        a, x = _args(slot_row, ctx.rows, d, dy.dtype), _token_rows(dy)
        a.tokens_in, a.row_slot = x.data_ptr(), row_slot.data_ptr()
        a.ld = x.stride(0) if x.shape[0] > 1 else d
        g = dw = None
        if weights is not None:
            w = weights.contiguous()
            a.weights, a.weight_type = w.data_ptr(), N.DTYPE_CODE[w.dtype]
        if need_rows:
            g = torch.empty(ctx.rows, d, dtype=dy.dtype, device=dy.device)
            a.rows_out = g.data_ptr()
        if need_weights:
            values, dw = rows.contiguous(), torch.empty(weights.shape, dtype=weights.dtype, device=dy.device)
            a.rows_in, a.d_weights = values.data_ptr(), dw.data_ptr()
        _run("ccf_return_rows_bwd", a, dy.device)
        return g, None, None, dw


# ---- by torch's operations ----------------------------------------------------------------------------------------------
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _order_torch(idx, num_experts, capacity, align):
    flat, dev = idx.reshape(-1).long(), idx.device
    rows = order_rows(flat.numel(), num_experts, capacity, align)
    key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
    sorted_key, order = torch.sort(key, stable=True)
    ends = torch.searchsorted(sorted_key, torch.arange(num_experts + 1, device=dev), right=True)
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    counts = (ends - starts)[:num_experts]
    if capacity is not None:
        counts = counts.clamp(max=capacity)
    base = torch.cat([ends.new_zeros(1), torch.cumsum((counts + align - 1) // align * align, 0)])
    pos = torch.arange(flat.numel(), device=dev) - starts[sorted_key]
    kept = (sorted_key < num_experts) & (pos < torch.cat([counts, counts.new_zeros(1)])[sorted_key])
    row = torch.where(kept, base[sorted_key] + pos, rows)      # the others go to a row behind the last
    row_slot = torch.full((rows + 1,), -1, dtype=torch.int32, device=dev).scatter(0, row, order.int())
    slot_row = torch.empty_like(flat, dtype=torch.int32).scatter(0, order, torch.where(kept, row, -1).int())
    return ExpertOrder(slot_row.view(idx.shape), row_slot[:rows], counts.int(), base.int())


def _outside(numbers, count):
    """Where a number is none of ``count``: what the kernels leave out, and torch's operations must not see."""
    return (numbers < 0) | (numbers >= count)


def _slots(rows, slot_row):
    """Each slot's row in fp32 (fp64), zeros where it has none: [..., top_k, d]."""
    if rows.shape[0] == 0:
        return _wide(rows).sum(dim=0).expand(*slot_row.shape, rows.shape[1])      # zeros, with the graph of the rows
    none = _outside(slot_row, rows.shape[0])
    return _wide(rows)[slot_row.masked_fill(none, 0).long()].masked_fill(none.unsqueeze(-1), 0.0)


def _spread(values, slot_row, row_slot, weights):
    """weights[slot] * values[token] in the rows, zeros in those without a slot."""
    values = values.reshape(math.prod(values.shape[:-1]), values.shape[-1])
    if row_slot.shape[0] == 0:
        return values[:0]
    none = _outside(row_slot, values.shape[0] * slot_row.shape[-1])
    slot = row_slot.masked_fill(none, 0).long()
    rows = _wide(values)[torch.div(slot, slot_row.shape[-1], rounding_mode="floor")]
    if weights is not None:
        rows = rows * _wide(weights.reshape(-1))[slot].masked_fill(none, 0.0).unsqueeze(1)
    return rows.masked_fill(none.unsqueeze(1), 0.0).to(values.dtype)


# ---- what users call ------------------------------------------------------------------------------------------------------
def expert_order(idx: torch.Tensor, num_experts: int, capacity: Optional[int] = None, align: int = 1) -> ExpertOrder:
    """The rows of a call's slots. ``idx [..., top_k]`` (int64 or int32): the expert of each slot; a number outside [0, num_experts) is no expert's, and that slot
    has no row. ``capacity``: rows that an expert takes at most, the first ones. ``align``: every expert's rows begin at a multiple of it."""
    if idx.is_cuda and idx.numel() > 0 and not N.transformed(idx) and not torch.jit.is_tracing():      # a trace would miss the launches
        module = N.torch_module()
        if module is not None:      # checks its arguments as below
            return ExpertOrder(*module.expert_order(idx, num_experts, capacity, align))
        _check_idx(idx, num_experts, capacity, align)
        return _order_py(idx, num_experts, capacity, align)
    _check_idx(idx, num_experts, capacity, align)
    return _order_torch(idx, num_experts, capacity, align)


def sort_rows(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """``x [..., d]`` in the rows of an order: ``[rows, d]``, zeros in rows without a slot. Differentiable."""
    if _on_kernels(x) and order.slot_row.numel() > 0:
        module = _module()
        if module is not None:
            return module.sort_rows(x, order.slot_row, order.row_slot)
        _check_order(order)
        _check_tokens(x, order.slot_row)
        return _SortFn.apply(x, order.slot_row.contiguous(), order.row_slot.contiguous())
    _check_order(order)
    _check_tokens(x, order.slot_row)
    return _spread(x, order.slot_row, order.row_slot, None)


def sort_by_expert(x: torch.Tensor, idx: torch.Tensor, num_experts: int, capacity: Optional[int] = None, align: int = 1) -> Tuple[torch.Tensor, ExpertOrder]:
    """``order = expert_order(idx, ...)`` and ``sort_rows(x, order)`` in one call."""
    if _on_kernels(x) and idx.numel() > 0:
        module = _module()
        if module is not None:
            rows, *order = module.sort_by_expert(x, idx, num_experts, capacity, align)
            return rows, ExpertOrder(*order)
    _check_idx(idx, num_experts, capacity, align)
    _check_tokens(x, idx)
    order = expert_order(idx, num_experts, capacity, align)
    return sort_rows(x, order), order


def return_rows(rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] = sum over j of weights[t, j] * rows[slot_row[t, j]]`` of ``rows [rows, d]``: the sum of each token's slots that have a row, with ``weights [..., top_k]``
    (any floating type) or without. Differentiable in rows and weights: a row without a slot gets zeros, the weight of a slot without a row 0."""
    if _on_kernels(rows, weights) and order.slot_row.numel() > 0:
        module = _module()
        if module is not None:
            return module.return_rows(rows, order.slot_row, order.row_slot, weights)
        _check_order(order)
        _check_return(rows, order, weights)
        return _ReturnFn.apply(rows, order.slot_row.contiguous(), order.row_slot.contiguous(), weights)
    _check_order(order)
    _check_return(rows, order, weights)
    slots = _slots(rows, order.slot_row)
    if weights is not None:
        slots = slots * _wide(weights).masked_fill(_outside(order.slot_row, rows.shape[0]), 0.0).unsqueeze(-1)
    return slots.sum(dim=-2).to(rows.dtype)
