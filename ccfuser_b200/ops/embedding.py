"""Sums of embedding lookups on the library's kernels (csrc/embedding.cu): what the models put in front of their first block.

``embedding`` adds up to three lookups in one pass, ``scale * weight[ids] + position_weight[position] + type_weight[type_ids]``, in fp32
with one rounding: word and position table of GPT, word table times sqrt(d_model) of Transformer-XL, word, position and type table of BERT
(mix_moe/mix_moe/examples/models/moe_gpt.py, transformer-xl/mem_transformer_mix_moe.py, models/moe_bert.py of the reference use torch's). The
gradients are dense. A word's gradient is the sum over its tokens in their order, in fp32, after a sort of the tokens by id: no atomics,
the same bits every time. The autograd function is C++ (csrc/torch_tokens.cpp); the Python one below stands in where that module is missing and
while a graph is traced.

An id outside its table does not fault the GPU: its row is NaN, it adds nothing to a gradient, and it is recorded in the device's status word, which
``ops.gemm.Workspace.get(device).check()`` raises as ``TokenIndexError``. On the CPU the same sums run on torch's operations, which raise
``IndexError``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import native as N
from . import gemm as G

MAX_TOKENS = 2 ** 26
MAX_ROWS = 2 ** 31 - 1
MAX_COLUMNS = 2 ** 24
_INDEX = (torch.int64, torch.int32)


def _fill(e, ids, rows, scale, skip):
    t = e.table[e.tables]
    t.rows, t.scale, t.skip = rows, scale, skip
    if ids is not None:
        t.ids, t.wide = ids.data_ptr(), int(ids.dtype == torch.int64)
    e.tables += 1
    return t


def _run_grad(e, dy, grads, status):
    lib = N.load()
    scratch = []
    for k, g in enumerate(grads):
        t = e.table[k]
        scratch.append(torch.empty(lib.ccf_embedding_scratch(e.tokens, e.seq, t.rows, e.d, int(bool(t.ids))), dtype=torch.uint8, device=dy.device))
        t.scratch, t.grad = scratch[-1].data_ptr(), g.data_ptr()
    n = lib.ccf_embedding_bwd(C.byref(e), dy.data_ptr(), status, N.stream_ptr())
    N.check(min(n, 0), "ccf_embedding_bwd")
    N.count(n)


class _EmbeddingFn(torch.autograd.Function):
    """The C++ function in Python."""

    @staticmethod
    def forward(ctx, ids, weight, position, position_ids, types, type_ids, scale, skip, twice):
        index = [None if t is None else t.contiguous() for t in (ids, position_ids, type_ids)]
        e = N.Embed(tokens=ids.numel(), seq=ids.shape[-1] if ids.dim() else 1, d=weight.shape[1], type=N.DTYPE_CODE[weight.dtype])
        held = []
        for k, w in enumerate((weight, position, types)):
            if w is None:
                continue
            held.append(w if w.stride(1) == 1 and w.stride(0) >= w.shape[1] else w.contiguous())
            t = _fill(e, index[k], w.shape[0], scale if k == 0 else 1.0, skip if k == 0 else -1)
            t.weight, t.ld = held[-1].data_ptr(), held[-1].stride(0) if w.shape[0] > 1 else e.d
        y = torch.empty(*ids.shape, e.d, dtype=weight.dtype, device=weight.device)
        with torch.cuda.device(weight.device):
            N.check(N.load().ccf_embedding_fwd(C.byref(e), y.data_ptr(), G.Workspace.status_of(y), N.stream_ptr()), "ccf_embedding_fwd")
        N.count(1)
        ctx.save_for_backward(*index)
        ctx.rows = [0 if w is None else w.shape[0] for w in (weight, position, types)]
        ctx.scale, ctx.skip, ctx.twice = scale, skip, twice
        return y

    @staticmethod
    def backward(ctx, dy):
        index, out, grads = [None if i is None else i.contiguous() for i in ctx.saved_tensors], [None] * 9, []   # hooks may have other strides
        if torch.is_grad_enabled():      # the gradient is to be differentiated in its turn: by operations of torch
            if not ctx.twice:
                raise RuntimeError(N.REFUSED_TWICE)
            dy32 = dy.reshape(-1, dy.shape[-1]).float()
            for k, at in enumerate((1, 2, 4)):
                if not (ctx.rows[k] and ctx.needs_input_grad[at]):
                    continue
                seq = index[0].shape[-1] if index[0].dim() else 1
                i = torch.arange(index[0].numel(), device=dy.device) % seq if index[k] is None else index[k].reshape(-1).long()
                off = (i < 0) | (i >= ctx.rows[k]) | ((i == ctx.skip) if k == 0 else False)
                g = torch.ops.aten.embedding_dense_backward(dy32.masked_fill(off[:, None], 0), i.masked_fill(off, 0), ctx.rows[k], -1, False)
                out[at] = (g * (ctx.scale if k == 0 else 1.0)).to(dy.dtype)
            return tuple(out)
        dy = G.packed(dy)
        e = N.Embed(tokens=index[0].numel(), seq=index[0].shape[-1] if index[0].dim() else 1, d=dy.shape[-1], type=N.DTYPE_CODE[dy.dtype])
        for k, at in enumerate((1, 2, 4)):
            if ctx.rows[k] and ctx.needs_input_grad[at]:
                _fill(e, index[k], ctx.rows[k], ctx.scale if k == 0 else 1.0, ctx.skip if k == 0 else -1)
                out[at] = torch.empty(ctx.rows[k], e.d, dtype=dy.dtype, device=dy.device)
                grads.append(out[at])
        if grads:
            with torch.cuda.device(dy.device):
                _run_grad(e, dy, grads, G.Workspace.status_of(dy))
        return tuple(out)


def _check_ids(name, ids, device):
    if ids.dtype not in _INDEX:
        raise TypeError(f"{name}: indices are int64 or int32, not {ids.dtype}")
    if ids.device != device:
        raise ValueError(f"{name} is on {ids.device}, the table on {device}")


def _check_table(name, table, weight):
    if table.dim() != 2 or table.shape[1] != weight.shape[1] or table.dtype != weight.dtype or table.device != weight.device:
        raise ValueError(f"{name}: [rows, {weight.shape[1]}] of {weight.dtype} on {weight.device}, got {tuple(table.shape)} of "
                         f"{table.dtype} on {table.device}")


def _skip(padding_idx, rows):
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} lies outside the table's {rows} rows")
    return padding_idx % rows


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, *, position_weight: Optional[torch.Tensor] = None,
              position_ids: Optional[torch.Tensor] = None, type_weight: Optional[torch.Tensor] = None,
              type_ids: Optional[torch.Tensor] = None, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids] + position_weight[position_ids] + type_weight[type_ids]``, ``[*ids.shape, d]``.

    ``position_ids`` (broadcast to the shape of ``ids``) default to the index along the last dimension of ``ids``. The tables are ``[rows, d]`` of one
    type. ``padding_idx``: that row of ``weight`` gets no gradient (it is looked up like any other). The result cannot be differentiated twice."""
    return _embedding(ids, weight, scale, position_weight, position_ids, type_weight, type_ids, padding_idx)


def _embedding(ids, weight, scale, position_weight, position_ids, type_weight, type_ids, padding_idx, plain=False, twice=False):
    """plain: by torch's operations on a GPU too. twice: the gradient can be differentiated again, then by torch's operations."""
    if weight.is_cuda and weight.numel() and ids.numel() and not plain:
        module = N.torch_module()
        if module is not None and not torch.jit.is_tracing():      # checks its arguments as below
            return module.embedding(ids, weight, position_weight, position_ids, type_weight, type_ids, scale, padding_idx,
                                    G.Workspace.of(weight).status, twice)
    if weight.dim() != 2:
        raise ValueError(f"weight: [rows, d], got {tuple(weight.shape)}")
    _check_ids("ids", ids, weight.device)
    skip = _skip(padding_idx, weight.shape[0])
    if position_weight is not None:
        _check_table("position_weight", position_weight, weight)
        if position_ids is not None:
            _check_ids("position_ids", position_ids, weight.device)
            if position_ids.shape != ids.shape:
                position_ids = position_ids.expand(ids.shape)
        elif (ids.shape[-1] if ids.dim() else 1) > position_weight.shape[0]:
            raise ValueError(f"{ids.shape[-1]} positions, and {position_weight.shape[0]} rows in position_weight")
    elif position_ids is not None:
        raise ValueError("position_ids without position_weight")
    if (type_weight is None) != (type_ids is None):
        raise ValueError("type_weight and type_ids go together")
    if type_weight is not None:
        _check_table("type_weight", type_weight, weight)
        _check_ids("type_ids", type_ids, weight.device)
        if type_ids.shape != ids.shape:
            type_ids = type_ids.expand(ids.shape)
    if ids.numel() and any(t is not None and t.shape[0] == 0 for t in (weight, position_weight, type_weight)):
        raise ValueError("a table without rows")
    plain = plain or not weight.is_cuda
    if not plain and weight.dtype not in N.DTYPE_CODE:
        raise TypeError(f"tables on a GPU are bf16, fp16 or fp32, not {weight.dtype}")
    if plain or ids.numel() == 0 or weight.shape[1] == 0:
        return _embedding_torch(ids, weight, scale, position_weight, position_ids, type_weight, type_ids, padding_idx)
    if ids.numel() > MAX_TOKENS:
        raise ValueError(f"{ids.numel()} tokens: at most 2^26 in one call")
    if weight.shape[1] > MAX_COLUMNS or any(t is not None and t.shape[0] > MAX_ROWS for t in (weight, position_weight, type_weight)):
        raise ValueError("a table of at most 2^31 - 1 rows and 2^24 columns")
    return _EmbeddingFn.apply(ids, weight, position_weight, position_ids, type_weight, type_ids, float(scale), skip, twice)


def _embedding_torch(ids, weight, scale, position_weight, position_ids, type_weight, type_ids, padding_idx):
    y = F.embedding(ids, weight, padding_idx)
    if scale != 1.0:
        y = y * scale
    if position_weight is not None:
        if position_ids is None:
            position_ids = torch.arange(ids.shape[-1] if ids.dim() else 1, device=ids.device)
            position_ids = position_ids if ids.dim() else position_ids[0]
        y = y + F.embedding(position_ids, position_weight)
    if type_weight is not None:
        y = y + F.embedding(type_ids, type_weight)
    return y


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """The dense gradient ``[num_rows, d]`` of a table from the gradient ``[*ids.shape, d]`` of its lookups: what ``embedding`` does in its
    backward pass, without a graph."""
    if grad.is_cuda and grad.numel():
        module = N.torch_module()
        if module is not None and not torch.jit.is_tracing():
            return module.embedding_grad(grad, ids, num_rows, scale, padding_idx, G.Workspace.of(grad).status)
    _check_ids("ids", ids, grad.device)
    if num_rows < 1 or grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"grad: {list(ids.shape)} + [d] and at least one row, got {list(grad.shape)} and {num_rows} rows")
    skip = _skip(padding_idx, num_rows)
    if grad.is_cuda and grad.dtype not in N.DTYPE_CODE:
        raise TypeError(f"gradients on a GPU are bf16, fp16 or fp32, not {grad.dtype}")
    if not grad.is_cuda or grad.numel() == 0:
        grad = grad.detach()
        out = torch.zeros(num_rows, grad.shape[-1], dtype=grad.dtype if grad.dtype == torch.float64 else torch.float32, device=grad.device)
        out.index_add_(0, ids.reshape(-1).long(), grad.reshape(-1, grad.shape[-1]).to(out.dtype))
        if skip >= 0:
            out[skip] = 0.0
        return out.mul_(scale).to(grad.dtype)
    if ids.numel() > MAX_TOKENS or num_rows > MAX_ROWS or grad.shape[-1] > MAX_COLUMNS:
        raise ValueError("at most 2^26 tokens, 2^31 - 1 rows and 2^24 columns in one call")
    with torch.no_grad():
        dy, index = G.packed(grad), ids.contiguous()
        e = N.Embed(tokens=index.numel(), seq=1, d=dy.shape[-1], type=N.DTYPE_CODE[dy.dtype])
        _fill(e, index, num_rows, float(scale), skip)
        out = torch.empty(num_rows, e.d, dtype=dy.dtype, device=dy.device)
        with torch.cuda.device(dy.device):
            _run_grad(e, dy, [out], G.Workspace.status_of(dy))
        return out


class Embedding(nn.Embedding):
    """``nn.Embedding`` (same parameters, same state-dict keys) on ``embedding``, with a factor ``scale`` and the other tables as arguments of its call.
    What the kernels do not take (fp64 tables, more than 2^26 tokens, 2^31 - 1 rows or 2^24 columns, ``native.transformed`` ones, second
    derivatives) runs on torch's operations.
    ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are refused."""

    def __init__(self, *args, scale: float = 1.0, **kw):
        super().__init__(*args, **kw)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = scale

    def forward(self, ids, position_weight=None, position_ids=None, type_weight=None, type_ids=None, scale: float = 1.0):
        """``scale`` multiplies the module's own."""
        w = self.weight
        plain = (N.transformed(w) or w.dtype not in N.DTYPE_CODE or ids.numel() > MAX_TOKENS or w.shape[1] > MAX_COLUMNS or w.shape[0] > MAX_ROWS
                 or (position_weight is not None and position_weight.shape[0] > MAX_ROWS) or (type_weight is not None and type_weight.shape[0] > MAX_ROWS))
        return _embedding(ids, w, self.scale * scale, position_weight, position_ids, type_weight, type_ids, self.padding_idx, plain, True)


def _untouched(m):
    return type(m) is Embedding and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


def look_up(word: nn.Module, ids: torch.Tensor, scale: float = 1.0, position: Optional[nn.Module] = None, types: Optional[nn.Module] = None,
            type_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The sum of what a model's embedding modules give for tokens, their places and their types: one pass over their tables where all of them are ``Embedding``; module
    after module where one has been replaced (another vocabulary, an adapter) or carries hooks."""
    others = [m for m in (position, types) if m is not None]
    if _untouched(word) and all(_untouched(m) and m.scale == 1.0 and m.padding_idx is None for m in others):
        return word(ids, None if position is None else position.weight, None, None if types is None else types.weight, type_ids, scale)
    x = word(ids)
    if scale != 1.0:
        x = x * scale
    if position is not None:
        x = x + position(torch.arange(ids.shape[-1], device=ids.device))
    return x if types is None else x + types(type_ids)
