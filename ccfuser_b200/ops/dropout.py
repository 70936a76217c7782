"""Dropout from a counter-based generator, alone or with the addition of the residual stream (csrc/dropout.cu).

Whether an element is kept follows from 16 bits of Philox4x32-10 under (seed, step) on the device, the number of the call and the element's
place, so no mask is stored: the backward pass draws the same bits again. The seed and the step lie in a tensor, which is read when the kernel runs:
``DropoutState.advance()`` captured in a CUDA graph gives every replay masks of its own. The probability is rounded to a multiple of 2^-16, and
kept elements are divided by what remains of it. The autograd function is C++ (csrc/torch_tokens.cpp); the Python one below stands in where that
module is missing and while a graph is traced; on the CPU the same masks come from whole-number operations of torch.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import native as N
from . import gemm as G

_LOW = 0xFFFFFFFF


def _run(x, residual, state, copy, call, drop):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        N.check(N.load().ccf_dropout(x.data_ptr(), N.ptr(residual), y.data_ptr(), state.data_ptr(), N.ptr(copy), call, drop, x.numel(),
                                     N.DTYPE_CODE[x.dtype], N.stream_ptr()), "ccf_dropout")
    N.count(1)
    return y


class _DropoutFn(torch.autograd.Function):
    """The C++ function in Python."""

    @staticmethod
    def forward(ctx, x, residual, state, call, drop):
        used = torch.empty_like(state)     # the seed and step of this pass: the state may move on before the backward pass
        y = _run(G.packed(x), None if residual is None else G.packed(residual), state, used, call, drop)
        ctx.save_for_backward(used)
        ctx.call, ctx.drop = call, drop
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        used, = ctx.saved_tensors
        dx = _run(G.packed(dy), None, used.contiguous(), None, ctx.call, ctx.drop) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def keep_mask(shape, p: float, state: torch.Tensor, call: int = 0) -> torch.Tensor:
    """The elements that ``dropout`` keeps, as truth values, in torch's whole-number operations."""
    n = 1
    for s in shape:
        n *= s
    seed, step = state[0], state[1]
    group = torch.arange((n + 7) // 8, dtype=torch.int64, device=state.device)
    c = [group & _LOW, group >> 32, torch.full_like(group, call & _LOW), (step & _LOW).expand_as(group)]
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57       # the low 64 bits of the product, as the hardware keeps them
        c = [((b >> 32) & _LOW) ^ c[1] ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c[3] ^ k1, a & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack(c, dim=1)
    bits = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    return (bits >= round(p * 65536)).view(shape)


def dropout(x: torch.Tensor, p: float, state: torch.Tensor, call: int = 0, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + (kept ? x / (1 - p) : 0)``.

    ``state``: int64 tensor [seed, step] on the device of ``x``. Calls of one step need different numbers ``call`` (0 to 2^32 - 1) for different
    masks; the low 32 bits of the step count. ``residual`` has the shape and type of ``x``. A dropped element is 0 whatever it was."""
    if x.is_cuda and x.dtype in N.DTYPE_CODE and x.numel():
        module = N.torch_module()
        if module is not None and not torch.jit.is_tracing():      # checks its arguments as below
            return module.dropout(x, residual, state, call, p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p: 0 to 1, got {p}")
    if not 0 <= call <= _LOW:
        raise ValueError(f"call: 0 to 2^32 - 1, got {call}")
    if state.dtype != torch.int64 or state.shape != (2,) or state.device != x.device or not state.is_contiguous():
        raise ValueError(f"state: two int64 next to each other on {x.device}, got {tuple(state.shape)} of {state.dtype} on {state.device}")
    if not x.is_floating_point():
        raise TypeError(f"x: a floating type, got {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual: {tuple(x.shape)} of {x.dtype} on {x.device}, got {tuple(residual.shape)} of {residual.dtype} on "
                         f"{residual.device}")
    drop = round(p * 65536)
    if not (x.is_cuda and x.dtype in N.DTYPE_CODE and x.numel() > 0):
        wide = x if x.dtype == torch.float64 else x.float()
        y = torch.where(keep_mask(x.shape, p, state, call), wide * (65536 / max(1, 65536 - drop)), torch.zeros_like(wide))
        return (y if residual is None else y + residual.to(y.dtype)).to(x.dtype)
    return _DropoutFn.apply(x, residual, state, call, drop)


class _First:
    """Notes where a pass begins."""

    def __init__(self, state, start):
        self.state, self.start = state, start

    def __enter__(self):
        self.start[:] = [(self.state.tensor.clone(), self.state.calls)]

    def __exit__(self, *_):
        pass


class _Again:
    """Goes back there, once for every repetition."""

    def __init__(self, state, start):
        self.state, self.start, self.now = state, start, []

    def __enter__(self):
        s = self.state
        self.now.append((s.tensor.clone(), s.calls))
        s.tensor.copy_(self.start[0][0])
        s.calls = self.start[0][1]
        s._again += 1

    def __exit__(self, *_):
        s = self.state
        tensor, s.calls = self.now.pop()
        s.tensor.copy_(tensor)
        s._again -= 1


class DropoutState:
    """Seed, step and call counter that the dropouts of one model share. ``advance()`` begins the next step's masks: an addition on the device, so
    that a captured one advances with every replay. ``rank`` is added to the seed: ranks of a job give the same seed and draw masks of their own.
    ``state_dict()`` is what a checkpoint has to keep for later steps to go on with their masks, the same on every rank
    (``utils.checkpoint.save_ep_checkpoint`` keeps it for the ``Dropout`` modules of a model).

    A forward pass that the backward pass repeats (``torch.utils.checkpoint``) needs the numbers that its calls had, which
    ``checkpoint(..., use_reentrant=False, context_fn=state.recomputed)`` gives them; without that, a call inside a backward pass is an error."""

    def __init__(self, seed: int, device=None, rank: int = 0):
        self.rank = rank
        self.tensor = torch.tensor([self._wrapped(seed + rank), 0], dtype=torch.int64, device=device)
        self.calls = 0
        self._again = 0

    @staticmethod
    def _wrapped(seed):
        """As 64 bits with a sign hold it."""
        return (seed + 2 ** 63) % 2 ** 64 - 2 ** 63

    def state_dict(self) -> dict:
        seed, step = self.tensor.tolist()
        return {"seed": self._wrapped(seed - self.rank), "step": step, "calls": self.calls}

    def load_state_dict(self, state: dict):
        """In place: captured graphs go on with it."""
        self.tensor.copy_(torch.tensor([self._wrapped(state["seed"] + self.rank), state["step"]]))
        self.calls = state["calls"]

    def _not_repeated(self):
        if not self._again and torch._C._current_graph_task_id() != -1:
            raise RuntimeError("a DropoutState used inside a backward pass would draw other masks than the forward pass did: give checkpoint() "
                               "use_reentrant=False and context_fn=state.recomputed, or call dropout() with numbers of your own")

    def recomputed(self):
        """The contexts of a checkpointed forward pass and of its repetition, in which step and call numbers are those of the first one."""
        start = []
        return _First(self, start), _Again(self, start)

    def next_call(self) -> int:
        self._not_repeated()
        self.calls = (self.calls + 1) & _LOW
        return self.calls

    def on(self, device) -> torch.Tensor:
        if self.tensor.device != device:
            self.tensor = self.tensor.to(device)
        return self.tensor

    def advance(self):
        self._not_repeated()
        self.tensor[1:].add_(1)

    def begin_step(self, device):
        """The next step, its calls numbered from one again: the masks of a step follow from the seed and its number alone."""
        self.on(device)
        self.calls = 0
        self.advance()


class Dropout(nn.Module):
    """``dropout`` of a model: ``forward(x, residual=None)`` adds the residual, and in evaluation, or for ``p=0``, adds it alone."""

    def __init__(self, p: float, state: DropoutState):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p: 0 to 1, got {p}")
        self.p, self.state = p, state

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return dropout(x, self.p, self.state.on(x.device), self.state.next_call(), residual)

    def extra_repr(self):
        return f"p={self.p}"
