"""Log probabilities of given tokens with the entropy and the best alternatives of every row of logits (csrc/logprobs.cu).

``token_logprobs`` is the models' loss (its mean is the cross-entropy) and their scores: one pass over bf16, fp16 or fp32 logits, statistics in
fp32, nothing of the logits' size stored besides their gradient. The autograd function is C++ (csrc/torch_tokens.cpp); the Python one
below stands in where that module is missing and while a graph is traced. The reference's models call torch's cross-entropy on fp32 copies
(mix_moe/mix_moe/examples/models/moe_gpt.py, transformer-xl/mem_transformer_mix_moe.py).

A target outside the vocabulary does not fault the GPU: its log probability is NaN, and it is recorded in the device's status word, which
``ops.gemm.Workspace.get(device).check()`` raises as ``TokenIndexError``. On the CPU the same values come from torch's operations.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from .. import native as N
from . import gemm as G

MAX_TOP = 32
MAX_WIDTH = 2 ** 30
MAX_ROWS = 2 ** 28 - 1


class TokenLogprobs(NamedTuple):
    """``logprobs``, ``entropy`` of the targets' shape in fp32; ``top_logprobs`` (fp32) and ``top_ids`` (int64) with ``top_k`` more columns, or
    None for ``top_k=0``."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _args(x, t, top_k, temperature, vocab, ignore, status):
    return N.Logprobs(x=x.data_ptr(), targets=t.data_ptr(), wide=int(t.dtype == torch.int64), status=status, rows=x.shape[0],
                      ld=x.stride(0) if x.shape[0] > 1 else x.shape[1], ignore=ignore, vocab=vocab, width=x.shape[1], top_k=top_k,
                      type=N.DTYPE_CODE[x.dtype], inv_t=1.0 / temperature)


def _rows_of(logits, rows, width):
    """The logits as the kernels read them: rows with any distance, the first on a 16-byte boundary, their elements next to each other."""
    x = logits.reshape(rows, width)
    if x.stride(1) != 1 or (rows > 1 and x.stride(0) < width):
        x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


class _LogprobsFn(torch.autograd.Function):
    """The C++ function in Python."""

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, vocab, ignore, twice):
        rows, width = targets.numel(), logits.shape[-1]
        x, t = _rows_of(logits, rows, width), targets.contiguous()
        f32 = dict(dtype=torch.float32, device=logits.device)
        lp, entropy, stats = torch.empty(targets.shape, **f32), torch.empty(targets.shape, **f32), torch.empty(rows, 3, **f32)
        a = _args(x, t, top_k, temperature, vocab, ignore, G.Workspace.status_of(x))
        a.logprobs, a.entropy, a.stats = lp.data_ptr(), entropy.data_ptr(), stats.data_ptr()
        top = ids = None
        if top_k:
            top, ids = torch.empty(*targets.shape, top_k, **f32), torch.empty(*targets.shape, top_k, dtype=torch.int64, device=logits.device)
            a.top_logprobs, a.top_ids = top.data_ptr(), ids.data_ptr()
        with torch.cuda.device(logits.device):
            N.check(N.load().ccf_logprobs_fwd(C.byref(a), N.stream_ptr()), "ccf_logprobs_fwd")
        N.count(1)
        ctx.save_for_backward(logits if twice else x, t, stats, ids)      # x has no history
        ctx.args, ctx.shape, ctx.twice = (top_k, temperature, vocab, ignore), logits.shape, twice
        ctx.set_materialize_grads(False)
        if not top_k:
            return lp, entropy
        ctx.mark_non_differentiable(ids)
        return lp, entropy, top, ids

    @staticmethod
    def backward(ctx, *grads):
        x, t, stats, ids = ctx.saved_tensors       # hooks may have put them into memory of their own, with other strides
        if torch.is_grad_enabled():      # the gradient is to be differentiated in its turn: by operations of torch
            if not ctx.twice or ids is not None or grads[1] is not None:
                raise RuntimeError(N.REFUSED_TWICE)
            return (None if grads[0] is None else _grad_torch(x, t, grads[0], *ctx.args[1:]),) + (None,) * 6
        x = _rows_of(x, t.numel(), x.shape[-1])
        t, stats, ids = t.contiguous(), stats.contiguous(), None if ids is None else ids.contiguous()
        g = [None if v is None else v.contiguous() for v in grads[:3]] + [None]
        if all(v is None for v in g):
            return (None,) * 7
        a = _args(x, t, *ctx.args, 0)
        a.dx_ld = a.width + (a.ld - a.width) % (16 // x.element_size())       # rows begin where those of the logits do in their 16 bytes
        whole = torch.empty(x.shape[0], a.dx_ld, dtype=x.dtype, device=x.device)
        a.stats, a.top_ids, a.dx = stats.data_ptr(), N.ptr(ids), whole.data_ptr()
        a.d_logprobs, a.d_entropy, a.d_top = N.ptr(g[0]), N.ptr(g[1]), N.ptr(g[2])
        with torch.cuda.device(x.device):
            N.check(N.load().ccf_logprobs_bwd(C.byref(a), N.stream_ptr()), "ccf_logprobs_bwd")
        N.count(1)
        return (whole[:, :x.shape[1]].view(ctx.shape),) + (None,) * 6


def _grad_torch(logits, targets, g, temperature, vocab, ignore):
    """The gradient of the log probabilities with respect to the logits."""
    z = logits[..., :vocab].float() / temperature
    none = (z.detach() == -math.inf).all(dim=-1, keepdim=True)
    p = torch.softmax(z.masked_fill(none, 0.0), dim=-1)
    t = targets.long()
    off = (t == ignore) | (t < 0) | (t >= vocab) | none[..., 0]
    g = g.masked_fill(off, 0.0)[..., None]
    d = (p * -g).scatter_add(-1, t.masked_fill(off, 0)[..., None], g) / temperature
    return torch.nn.functional.pad(d, (0, logits.shape[-1] - vocab)).to(logits.dtype)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, temperature: float = 1.0, vocab_size: Optional[int] = None,
                   ignore_index: int = -100) -> TokenLogprobs:
    """``log_softmax(logits / temperature)`` at ``targets``, its entropy and its ``top_k`` largest entries, for logits ``[..., width]`` and
    targets ``[...]`` (int64 or int32).

    Only the first ``vocab_size`` columns count (default: all); the gradient of the others is zero. ``ignore_index``: targets of this value give 0 and
    no gradient from their log probability. Alternatives come by value, equal ones by index; ``top_k`` is at most 32 and the vocabulary. A column at -inf has
    no probability: where fewer than ``top_k`` others are left, the id is -1 and the log probability -inf. A row without a finite logit gives -inf, entropy 0
    and a zero gradient; a row with NaN or +inf gives NaN. Log probabilities, entropy and the alternatives' log probabilities are differentiable, once."""
    return _token_logprobs(logits, targets, top_k, temperature, vocab_size, ignore_index, False)


def _token_logprobs(logits, targets, top_k, temperature, vocab_size, ignore_index, twice):
    """twice: the gradient of the log probabilities can be differentiated again, then by torch's operations."""
    if logits.is_cuda and logits.dtype in N.DTYPE_CODE and targets.numel():
        module = N.torch_module()
        if module is not None and not torch.jit.is_tracing():      # checks its arguments as below
            out = module.token_logprobs(logits, targets, top_k, temperature, vocab_size, ignore_index, G.Workspace.of(logits).status, twice)
            return TokenLogprobs(*out) if top_k else TokenLogprobs(out[0], out[1], None, None)
    vocab = _check(logits, targets, top_k, temperature, vocab_size)
    if not (logits.is_cuda and logits.dtype in N.DTYPE_CODE and targets.numel() > 0):
        return _logprobs_torch(logits, targets, top_k, temperature, vocab, ignore_index)
    if logits.shape[-1] > MAX_WIDTH or targets.numel() > MAX_ROWS:
        raise ValueError("at most 2^30 columns and 2^28 - 1 rows in one call")
    out = _LogprobsFn.apply(logits, targets, top_k, float(temperature), vocab, ignore_index, twice)
    return TokenLogprobs(out[0], out[1], *(out[2:] if top_k else (None, None)))


def _check(logits, targets, top_k, temperature, vocab_size):
    """The number of columns that count."""
    if logits.dim() < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets: one per row of the logits, {tuple(logits.shape[:-1])}, got {tuple(targets.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets are int64 or int32, not {targets.dtype}")
    if targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, the logits on {logits.device}")
    width = logits.shape[-1]
    vocab = width if vocab_size is None else vocab_size
    if not 1 <= vocab <= width:
        raise ValueError(f"vocab_size: 1 to the {width} columns of the logits, got {vocab}")
    if not 0 <= top_k <= min(MAX_TOP, vocab):
        raise ValueError(f"top_k: 0 to {min(MAX_TOP, vocab)}, got {top_k}")
    if not 1e-37 <= temperature <= 1e37:       # it and its inverse are normal in fp32
        raise ValueError(f"temperature: a positive number that fp32 holds, got {temperature}")
    return vocab


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, vocab_size: Optional[int] = None, ignore_index: int = -100) -> torch.Tensor:
    """Mean of ``-token_logprobs`` over the targets that are not ignored: ``F.cross_entropy`` of the first ``vocab_size`` columns in fp32. What the
    kernels do not take (fp64 logits, more than 2^28 - 1 rows or 2^30 columns, ``native.transformed`` ones, second derivatives) runs on torch's operations."""
    if N.transformed(logits) or logits.dtype not in N.DTYPE_CODE or not logits.is_cuda or targets.numel() > MAX_ROWS or logits.shape[-1] > MAX_WIDTH:
        vocab = _check(logits, targets, 0, 1.0, vocab_size)
        lp = _picked(_log_softmax(logits, 1.0, vocab)[1], targets, vocab, ignore_index)
    else:
        lp = _token_logprobs(logits, targets, 0, 1.0, vocab_size, ignore_index, True).logprobs
    return -lp.sum() / (targets != ignore_index).sum()


def _log_softmax(logits, temperature, vocab):
    x = logits[..., :vocab]
    x = x if x.dtype == torch.float64 else x.float()
    largest = x.detach().amax(dim=-1, keepdim=True)
    z = x if temperature == 1.0 else (x - largest) / temperature      # without the largest: the quotient may pass the type's range
    none = largest == -math.inf
    if _host_may_look(x) and not bool(none.any()):
        return x, torch.log_softmax(z, dim=-1)
    # a row without a finite logit gets zeros in its place, which give it no gradient
    lp = torch.log_softmax(torch.where(none, torch.zeros_like(x), z), dim=-1)
    return x, torch.where(none, torch.full_like(lp, -math.inf), lp)


def _host_may_look(t):
    """Not where there is no memory to look at, and not in captures."""
    return not N.transformed(t) and t.device.type != "meta" and not (t.is_cuda and torch.cuda.is_current_stream_capturing())


def _picked(lp, targets, vocab, ignore):
    """The targets' log probabilities. One outside the vocabulary raises, or gives NaN where the host may not look."""
    kept = targets != ignore
    outside = kept & ((targets < 0) | (targets >= vocab))
    if _host_may_look(lp) and bool(outside.any()):
        raise IndexError(f"a target lies outside the vocabulary of {vocab}")
    at = torch.where(kept & ~outside, targets, torch.zeros_like(targets)).long()
    picked = lp.gather(-1, at[..., None])[..., 0]
    picked = torch.where(outside, torch.full_like(picked, math.nan), picked)
    return torch.where(kept, picked, torch.zeros_like(picked))


def _logprobs_torch(logits, targets, top_k, temperature, vocab, ignore):
    x, lp = _log_softmax(logits, temperature, vocab)
    gone = lp == -math.inf
    entropy = -torch.where(gone, torch.zeros_like(lp), lp.exp() * torch.where(gone, torch.zeros_like(lp), lp)).sum(dim=-1)
    picked = _picked(lp, targets, vocab, ignore)
    if not top_k:
        return TokenLogprobs(picked, entropy, None, None)
    ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    missing = x.detach().gather(-1, ids) == -math.inf
    top = lp.gather(-1, ids)
    return TokenLogprobs(picked, entropy, torch.where(missing, torch.full_like(top, -math.inf), top),
                         torch.where(missing, torch.full_like(ids, -1), ids))
