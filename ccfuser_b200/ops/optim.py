"""Optimizers that run on the library's kernels."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch

from .. import native as N

_BLOCK_ELEMS = 256 * 8 * 4      # elements one block of 256 threads covers in four passes of 16-byte vectors
_MAX_BLOCKS = 148 * 16


class FusedSGD(torch.optim.Optimizer):
    """Plain SGD (optional weight decay) for bf16 / fp16 CUDA parameters on csrc/moe_kernels.cu: full-width passes at the
    memory rate, up to 48 tensors per launch (``sgd_multi_kernel``), so that the hundreds of small tensors of a
    transformer (biases, LayerNorm weights, routers) cost a handful of launches instead of one each. Other parameters
    take the torch path. The reference's benchmark loops use torch.optim.SGD on half-precision parameters
    (mix_moe/mix_moe/examples/mix_moe_ddp.py:155)."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.0):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))
        self._table = None

    @staticmethod
    def _eligible(p, g) -> bool:
        return (p.is_cuda and p.dtype in (torch.bfloat16, torch.float16) and g.dtype == p.dtype and p.is_contiguous()
                and g.is_contiguous() and p.data_ptr() % 16 == 0 and g.data_ptr() % 16 == 0 and p.numel() > 0)

    def _launch(self, lib, batch, lr, wd, fp16, stream):
        t = self._table
        if t is None:
            t = self._table = N.SgdMulti()
        first = 0
        for k, (p, g) in enumerate(batch):
            n = p.numel()
            t.p[k], t.g[k], t.n[k], t.first_block[k] = p.data_ptr(), g.data_ptr(), n, first
            first += max(1, min(_MAX_BLOCKS, (n + _BLOCK_ELEMS - 1) // _BLOCK_ELEMS))
        t.first_block[len(batch)] = first
        t.count, t.lr, t.wd, t.fp16 = len(batch), lr, wd, fp16
        N.check(lib.ccf_sgd_multi(C.byref(t), stream), "ccf_sgd_multi")
        N.count(1)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = None
        for group in self.param_groups:
            lr, wd = float(group["lr"]), float(group["weight_decay"])
            batches = {}                      # (device, dtype) -> tensors waiting for one launch
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if self._eligible(p, g):
                    key = (p.device, p.dtype)
                    batch = batches.setdefault(key, [])
                    batch.append((p, g))
                    if len(batch) == N.SGD_MULTI:
                        lib = lib or N.load()
                        with torch.cuda.device(p.device):
                            self._launch(lib, batch, lr, wd, int(p.dtype == torch.float16), N.stream_ptr())
                        batch.clear()
                else:
                    if wd:
                        g = g.add(p, alpha=wd)
                    p.add_(g, alpha=-lr)
            for (device, dtype), batch in batches.items():
                if batch:
                    lib = lib or N.load()
                    with torch.cuda.device(device):
                        self._launch(lib, batch, lr, wd, int(dtype == torch.float16), N.stream_ptr())
        return loss


# ---- AdamW -----------------------------------------------------------------------------------------------------------------
STATE_BLOCK = 256          # weights that share the exponents of their 8-bit moments (csrc/adamw.h)
STATE8_LEAST = 4096        # weights from which on a tensor's moments are worth 8 bits
_M32, _M64 = 0xFFFFFFFF, 0xFFFFFFFFFFFFFFFF


def state8(p: torch.Tensor, rows: int = 1):
    """Empty 8-bit moments of a tensor: codes of the first and the second (uint8, of ``p``'s shape), and the exponents of their blocks, ``[rows, blocks of a row,
    2]``. ``rows``: parts of equal size that no block crosses, such as the experts of a weight ``[experts, out, in]``."""
    if rows < 1 or p.numel() % rows:
        raise ValueError(f"rows: a divisor of the {p.numel()} weights, got {rows}")
    blocks = -(-(p.numel() // rows) // STATE_BLOCK)
    return (torch.zeros(p.shape, dtype=torch.uint8, device=p.device), torch.zeros(p.shape, dtype=torch.uint8, device=p.device),
            torch.full((rows, blocks, 2), 40, dtype=torch.uint8, device=p.device))


def state_values(codes: torch.Tensor, exponents: torch.Tensor, second: bool = False, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What 8-bit moments stand for: ``codes`` (uint8) with the exponents ``[rows, blocks of a row, 2]`` (or ``[blocks, 2]``) of their blocks; ``second``: they are
    second moments. bf16 and fp32 hold every value as it is (fp16 only those of its range)."""
    if codes.dtype != torch.uint8 or exponents.dtype != torch.uint8:
        raise TypeError(f"codes and exponents are uint8, not {codes.dtype} and {exponents.dtype}")
    if dtype not in N.DTYPE_CODE:
        raise TypeError(f"values in bf16, fp16 or fp32, not {dtype}")
    _check_exponents(codes, exponents if exponents.dim() != 2 else exponents.unsqueeze(0), "codes")
    rows = exponents.shape[0] if exponents.dim() == 3 else 1
    if codes.device != exponents.device:
        raise ValueError(f"codes are on {codes.device}, their exponents on {exponents.device}")
    if not codes.is_cuda or codes.numel() == 0 or N.transformed(codes) or torch.jit.is_tracing():
        return _decode(codes, exponents.reshape(rows, -1, 2), second).to(dtype)
    module = N.torch_module()
    if module is not None:
        return module.state_values(codes, exponents, second, N.DTYPE_CODE[dtype])
    codes, exponents = codes.contiguous(), exponents.contiguous()
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        N.check(N.load().ccf_state_values(codes.data_ptr(), exponents.data_ptr(), out.data_ptr(), codes.numel(), rows, int(second), N.DTYPE_CODE[dtype],
                                          N.stream_ptr()), "ccf_state_values")
    N.count(1)
    return out


def _check_exponents(p, e, name):
    rows = e.shape[0] if e.dim() == 3 else 0
    if rows < 1 or p.numel() % rows or tuple(e.shape[1:]) != (-(-(p.numel() // rows) // STATE_BLOCK), 2):
        raise ValueError(f"exponents of {name}: [rows, blocks of a row, 2] for {p.numel()} weights, got {tuple(e.shape)}")


def _check_state(p, g, m, v, e, i):
    if g.layout != torch.strided or g.dtype != p.dtype:
        raise TypeError(f"grads: tensor {i} is {g.layout} of {g.dtype}, its parameter {p.dtype}")
    if not p.is_floating_point():
        raise TypeError(f"params: tensor {i} is {p.dtype}")
    kind = torch.uint8 if e is not None else torch.float64 if p.dtype == torch.float64 else torch.float32
    if m.dtype != kind or v.dtype != kind or (e is not None and e.dtype != kind):
        raise TypeError(f"moments of tensor {i} are {kind}, not {m.dtype} and {v.dtype}")
    if e is not None and p.dtype == torch.float64:
        raise TypeError(f"params: tensor {i} is of fp64, whose moments have no 8-bit form")
    if g.shape != p.shape or m.shape != p.shape or v.shape != p.shape:
        raise ValueError(f"tensor {i}: {tuple(p.shape)}, its gradient and moments {tuple(g.shape)}, {tuple(m.shape)} and {tuple(v.shape)}")
    if any(t is not None and t.device != p.device for t in (g, m, v, e)):
        raise ValueError(f"tensor {i} and what belongs to it lie on several devices")
    if e is not None:
        _check_exponents(p, e, f"tensor {i}")


@torch.no_grad()
def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor],
               step: Optional[int] = None, *, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               exponents: Optional[Sequence[torch.Tensor]] = None, seed: int = 0, numbers: Optional[Sequence[int]] = None,
               counter: Optional[torch.Tensor] = None) -> None:
    """One AdamW step of every tensor in place, by one launch for up to 400 tensors of a type (csrc/adamw.cu).

    Gradients have their parameters' types (bf16, fp16, fp32); the arithmetic is fp32 whatever they are. Moments are fp32, or uint8 codes with ``exponents``
    (``state8``), which are rounded up or down by a hash of (``seed``, step, tensor, weight), so that their mean is right; a tensor's number there is that in ``numbers``, or its place in
    the list. ``step`` is the number of this step, from 1. With ``counter``, an int64 tensor of one element on the tensors' device, that is raised by one instead and read on the device, so that a captured
    call counts its replays; then ``lr`` may be an fp32 tensor of one element there. Values that are not finite make a weight NaN as in torch, and with 8-bit moments from the
    next step on all weights of its block. Tensors on a CPU, of fp64 or not contiguous take torch's operations, to the same codes."""
    if (step is None) == (counter is None):
        raise ValueError("either step or counter")
    if counter is None and step < 1:
        raise ValueError(f"step: from 1, got {step}")
    device_lr = lr if torch.is_tensor(lr) else None
    if counter is not None and (counter.dtype != torch.int64 or counter.numel() != 1):
        raise ValueError(f"counter: one int64, got {tuple(counter.shape)} of {counter.dtype}")
    if device_lr is not None and (counter is None or lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != counter.device):
        raise ValueError("lr: a number, or with counter one fp32 beside it")
    lr = 0.0 if device_lr is not None else float(lr)
    beta1, beta2 = (float(b) for b in betas)
    if not (0.0 <= lr and 0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0 and 0.0 <= eps and 0.0 <= weight_decay):
        raise ValueError(f"lr, eps and weight_decay are at least 0, betas in [0, 1), got {lr}, {eps}, {weight_decay}, {beta1, beta2}")
    seed = (int(seed) + (1 << 63)) % (1 << 64) - (1 << 63)      # as C's 64 bits
    params, grads, exp_avgs, exp_avg_sqs = (t if isinstance(t, (list, tuple)) else list(t) for t in (params, grads, exp_avgs, exp_avg_sqs))
    exponents = exponents if exponents is None or isinstance(exponents, (list, tuple)) else list(exponents)
    numbers = numbers if numbers is None or isinstance(numbers, (list, tuple)) else list(numbers)
    rates = (lr, beta1, beta2, float(eps), float(weight_decay), seed)
    traced = bool(params) and N.transformed(params[0])      # no memory to look at
    module = N.torch_module() if params and params[0].is_cuda and not traced else None
    if module is not None and module.adamw_step(params, grads, exp_avgs, exp_avg_sqs, exponents, *rates, 0 if step is None else int(step), counter, device_lr, numbers):
        return
    if any(t is not None and len(t) != len(params) for t in (grads, exp_avgs, exp_avg_sqs, exponents, numbers)):
        raise ValueError(f"{len(params)} params need as many gradients, moments, exponents and numbers")
    if not params:
        return
    tensors = list(zip(params, grads, exp_avgs, exp_avg_sqs, [None] * len(params) if exponents is None else exponents))
    seen = set()
    for i, t in enumerate(tensors):
        _check_state(*t, i)
        if counter is not None and t[0].device != counter.device:
            raise ValueError(f"counter: on {counter.device}, the tensors beside it on {t[0].device}")
        place = id(t[0]) if traced or t[0].device.type == "meta" else t[0].data_ptr()
        if t[0].numel() and place in seen:
            raise ValueError(f"params: tensor {i} is there twice")
        seen.add(place)
    _adamw_each(tensors, numbers or range(len(params)), rates, step, counter, device_lr, traced)


def _adamw_each(tensors, numbers, rates, step, counter, device_lr, traced):
    """The step without the C++ module, or with tensors that the kernels do not take."""
    lr, beta1, beta2, eps, wd, seed = rates
    by_kind, others = {}, []
    for i, (p, g, m, v, e) in zip(numbers, tensors):
        if p.numel() == 0:
            continue
        if p.is_cuda and not traced and p.dtype in N.DTYPE_CODE and all(t is None or t.is_contiguous() for t in (p, m, v, e)):
            by_kind.setdefault((p.device, p.dtype), []).append((i, p, g.contiguous(), m, v, e))
        else:
            others.append((i, p, g, m, v, e))
    a = N.Adamw(lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=wd, seed=seed & _M64, step=step or 0)
    scalars = None
    if counter is not None and counter.is_cuda and not traced:
        scalars = torch.empty(32, dtype=torch.uint8, device=counter.device)
        with torch.cuda.device(counter.device):
            N.check(N.load().ccf_adamw_scalars(C.byref(a), counter.data_ptr(), N.ptr(device_lr), scalars.data_ptr(), N.stream_ptr()), "ccf_adamw_scalars")
        N.count(1)
        a.scalars = scalars.data_ptr()
    elif counter is not None:
        counter += 1
    for (device, dtype), batch in by_kind.items():
        table = (N.AdamwTensor * len(batch))(*(N.AdamwTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), N.ptr(e), p.numel(), 1 if e is None else e.shape[0], i)
                                               for i, p, g, m, v, e in batch))
        a.tensors, a.count, a.type = C.addressof(table), len(batch), N.DTYPE_CODE[dtype]
        with torch.cuda.device(device):
            launches = N.load().ccf_adamw(C.byref(a), N.stream_ptr())
        N.check(min(launches, 0), "ccf_adamw")
        N.count(launches)
        for _, p, _, m, v, e in batch:
            for t in (p, m, v) + (() if e is None else (e,)):
                if not t.is_inference():
                    torch.autograd.graph.increment_version(t)
    if others:
        if counter is not None:      # the number of the step is needed on the host
            step, lr = int(counter), lr if device_lr is None else float(device_lr)
        for i, p, g, m, v, e in others:
            _adamw_torch(p, g, m, v, e, _rounding_key(seed, step, i), lr, beta1, beta2, eps, wd, step)


def _adamw_torch(p, g, m, v, e, key, lr, beta1, beta2, eps, wd, step):
    """One tensor by torch's operations."""
    wide = torch.float64 if p.dtype == torch.float64 else torch.float32
    first, second, g = (m, v, g.to(wide)) if e is None else (_decode(m, e, False), _decode(v, e, True), g.to(wide))
    first = first * beta1 + g * (1 - beta1)
    second = second * beta2 + g * g * (1 - beta2)
    update = first / (second.sqrt() / math.sqrt(1 - beta2 ** step) + eps)
    old = p.to(wide)
    p.copy_(old - (old * (lr * wd) + update * (lr / (1 - beta1 ** step))))
    if e is None:
        m.copy_(first)
        v.copy_(second)
        return
    at = torch.arange(p.numel(), device=p.device)
    h = _mix((at + key) & _M32).view(p.shape)
    for codes, x, bits, k in ((m, first, h & 0xFFFFF, 0), (v, second, h >> 12, 1)):
        c, e[..., k] = _encode(x, e.shape[0], bits.int(), k == 1)
        codes.copy_(c)


def _mix(h):
    """MurmurHash3's last step, on int64 that hold 32 bits."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & _M32
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & _M32
    return h ^ (h >> 16)


def _split_mix(x):
    x = (x + 0x9E3779B97F4A7C15) & _M64
    x = (x ^ x >> 30) * 0xBF58476D1CE4E5B9 & _M64
    x = (x ^ x >> 27) * 0x94D049BB133111EB & _M64
    return x ^ x >> 31


def _blocks(x, rows):
    """[rows, blocks, STATE_BLOCK], the last block of a row filled up with zeros."""
    x = x.reshape(rows, -1)
    return torch.nn.functional.pad(x, (0, -x.shape[1] % STATE_BLOCK)).view(rows, -1, STATE_BLOCK)


def _unblocks(x, shape):
    n = math.prod(shape)
    return x.reshape(x.shape[0], -1)[:, :n // x.shape[0]].reshape(shape)


def _power(exponent):
    """2 to the given int32, from -126 to 127, in fp32."""
    return ((exponent + 127) << 23).view(torch.float32)


# a code is the upper bits of a float: its exponent is that far below the block's, and its block's factor is split in two for the range of fp32
_FIRST, _SECOND = (120, 8), (100, 4)


def _decode(codes, e, second):
    down, near = _SECOND if second else _FIRST
    c, x = _blocks(codes, e.shape[0]).int(), e[..., int(second)].int().unsqueeze(-1)
    bits = c << 20 if second else ((c & 0x7F) << 20) | ((c & 0x80) << 24)
    finite = x < 255
    values = bits.view(torch.float32) * 2.0 ** down * _power(torch.where(finite, x.clamp(min=40) - 127 - near, 0))
    return _unblocks(torch.where(finite, values, math.nan), codes.shape)


def _encode(x, rows, bits, second):
    """Codes and their blocks' exponents."""
    down, near = _SECOND if second else _FIRST
    b = _blocks(x, rows)
    a = b.abs()
    top = a.view(torch.int32).amax(dim=-1, keepdim=True)
    e = torch.where(top < 0x7F800000, (top + 0xFFFFF) >> 23, 255).clamp(min=40)
    finite = e < 255
    y = a * _power(torch.where(finite, 127 + near - e, 0)) * 2.0 ** -down
    code = (y.view(torch.int32) + _blocks(bits, rows)) >> 20
    code = torch.where(a > 0, code.clamp(min=1), code) if second else code | (b.view(torch.int32) >> 24) & 0x80
    return _unblocks(torch.where(finite, code, 0).to(torch.uint8), x.shape), e.squeeze(-1).to(torch.uint8)


def _check_group(group):
    """What torch's AdamW can do and this one cannot is refused rather than left out."""
    for name in ("maximize", "amsgrad"):
        if group.get(name):
            raise ValueError(f"FusedAdamW has no {name}")
    if group.get("state_bits", 32) not in (8, 32):
        raise ValueError(f"state_bits: 8 or 32, got {group['state_bits']}")


def _state8_rows(group, p):
    """The rows of a parameter's exponents, 0 where its moments are not held in 8 bits."""
    if group["state_bits"] != 8 or p.numel() < STATE8_LEAST or p.dtype not in N.DTYPE_CODE:
        return 0
    # rows that move between ranks (parallel/placement.py) take their blocks along
    return p.shape[0] if p.dim() >= 2 and (getattr(p, "skip_allreduce", False) or hasattr(p, "dp_comm")) else 1


def _rounding_key(seed, step, number):
    return (_split_mix(_split_mix(seed & _M64) ^ step) >> 32) + number * 0x9E3779B9 & _M32


_PIECE = 1 << 24           # moments that are encoded at a time, a multiple of STATE_BLOCK


def _state8_of(p, first, second, rows, key):
    """Given moments of ``p`` in 8 bits on its device, rounded as by a step with this key; in pieces, for the hash takes 64 bits a weight."""
    m, v, e = state8(p, rows)
    width = p.numel() // rows
    first, second = (t.detach().reshape(rows, width) for t in (first, second))
    tall = max(1, _PIECE // width)
    for r in range(0, rows, tall):
        for c in range(0, width, _PIECE):
            cut = slice(r, r + tall), slice(c, c + _PIECE)
            at = torch.arange(r, min(r + tall, rows), device=p.device)[:, None] * width + torch.arange(c, min(c + _PIECE, width), device=p.device)
            h = _mix((at + key) & _M32)
            for k, (codes, x, bits) in enumerate(((m, first, h & 0xFFFFF), (v, second, h >> 12))):
                x = x[cut].to(device=p.device, dtype=torch.float32)
                codes.view(rows, width)[cut], part = _encode(x, x.shape[0], bits.int(), k == 1)
                e[cut[0], c // STATE_BLOCK:c // STATE_BLOCK + part.shape[1], k] = part
    return m, v, e


class FusedAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on ``adamw_step``: all tensors of a step in one launch per type (400 of them at most), moments in fp32 whatever the weights' type
    or, with ``state_bits=8``, in 8 bits (2 bytes a weight instead of 8; tensors of fewer than 4096 weights and fp64 ones keep theirs in full). The mean of what
    8 bits hold is right, so that moments go on following changes of a fraction of their steps; ``seed`` chooses the hash that decides.

    ``capturable=True``: for steps captured in a CUDA graph. The number of the step then lies on the device, one for all parameters of a group and device, and ``lr`` may be an fp32 tensor of
    one element there; the first step is taken before the capture, and a graph holds the moments that it was captured with: after ``load_state_dict`` it is captured anew. ``state_dict`` has the names of torch's (``step``, ``exp_avg``, ``exp_avg_sq``, and ``exponents`` for 8 bits), and
    loads those of ``torch.optim.AdamW``. Expert weights (and the router's) share exponents inside an expert only, so that ``rebalance_experts`` moves their moments with them."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0,
                 capturable: bool = False):
        _check_group({"state_bits": state_bits})
        if torch.is_tensor(lr) and not capturable:
            raise ValueError("lr: a tensor with capturable=True only")
        if not (torch.is_tensor(lr) or lr >= 0.0) or eps < 0.0 or weight_decay < 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"lr, eps and weight_decay are at least 0, betas in [0, 1), got {lr}, {eps}, {weight_decay}, {betas}")
        self._counters, self._saved = {}, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed, capturable=capturable))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _check_group(param_group)
        super().add_param_group(param_group)

    def __setstate__(self, state):
        saved = self.__dict__.get("_saved")      # a checkpoint that is being loaded
        for k, group in enumerate(state["param_groups"]):
            if "state_bits" not in group and saved is not None:      # another optimizer's group: it says nothing of these
                group.update((name, self.param_groups[k][name]) for name in ("state_bits", "seed", "capturable"))
            for name, v in (("state_bits", 32), ("seed", 0), ("capturable", False)):
                group.setdefault(name, v)
            if saved is not None:      # as a step reads them: numbers, or a rate beside the counter, wherever the checkpoint was read to
                group["betas"] = tuple(float(b) for b in group["betas"])
                if torch.is_tensor(group["lr"]):
                    beside = group["params"][0].device if group["params"] else group["lr"].device
                    group["lr"] = group["lr"].detach().to(device=beside, dtype=torch.float32) if group["capturable"] else float(group["lr"])
            for number, (p, i) in enumerate(zip(group["params"], saved["param_groups"][k]["params"] if saved is not None else ())):
                if saved["state"].get(i):
                    state["state"][p] = self._loaded(k, group, number, p, saved["state"][i])
        super().__setstate__(state)      # up to here nothing has changed
        self._counters, self._saved = {}, None
        if saved is not None:
            for k, group in enumerate(self.param_groups):
                if group["capturable"]:
                    for p in group["params"]:
                        if "step" in self.state.get(p, {}):
                            self._counter(k, p)

    def __getstate__(self):
        return {k: v for k, v in super().__getstate__().items() if k not in ("_counters", "_saved")}

    def _counter(self, k, p):
        """The number of the last step of group ``k`` on the parameter's device."""
        key = (k, p.device)
        if key not in self._counters:
            steps = [self.state[q]["step"] for q in self.param_groups[k]["params"] if q.device == p.device and "step" in self.state.get(q, {})]
            known = max((int(s) for s in steps), default=0)
            self._counters[key] = torch.full((1,), known, dtype=torch.int64, device=p.device)
            for q in self.param_groups[k]["params"]:
                if q.device == p.device and "step" in self.state.get(q, {}):
                    self.state[q]["step"] = self._counters[key]
        return self._counters[key]

    def _start(self, k, group, p):
        state = self.state[p]
        rows = _state8_rows(group, p)
        if rows:
            state["exp_avg"], state["exp_avg_sq"], state["exponents"] = state8(p, rows)
        else:
            kind = torch.float64 if p.dtype == torch.float64 else torch.float32
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros(p.shape, dtype=kind, device=p.device) for _ in range(2))
        state["step"] = self._counter(k, p) if group["capturable"] else 0
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        batches, started = {}, []      # by group, number of the step (or device) and width of the moments
        try:
            for k, group in enumerate(self.param_groups):
                # a parameter's number is its place in the group, whether or not those before it have gradients: replicas on several ranks round alike
                for number, p in enumerate(group["params"]):
                    if p.grad is None:
                        continue
                    state = self.state[p]
                    if capturing and not (group["capturable"] and "step" in state):
                        raise RuntimeError("FusedAdamW: a step in a CUDA graph needs capturable=True and a step before the capture")
                    if "step" not in state:
                        started.append(p)
                        state = self._start(k, group, p)
                    key = (k, p.device if group["capturable"] else state["step"] + 1, "exponents" in state)
                    batches.setdefault(key, []).append((p, p.grad, state["exp_avg"], state["exp_avg_sq"], state.get("exponents"), number, state))
            if len(batches) > 1:      # each call looks at its own tensors before it changes one
                for batch in batches.values():
                    if [t[1].layout for t in batch].count(torch.strided) != len(batch):
                        raise TypeError("FusedAdamW: gradients are strided")
            raised = set()
            for (k, at, eight), batch in batches.items():
                group = self.param_groups[k]
                p, g, m, v, e, numbers, states = zip(*batch)
                step, counter = at, None
                if group["capturable"]:
                    step, counter = None, self._counter(k, p[0])
                    again = (k, at) in raised
                    if again:      # by the batch before
                        counter -= 1
                try:
                    adamw_step(p, g, m, v, step, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                               exponents=e if eight else None, seed=group["seed"] + (k << 32), numbers=numbers, counter=counter)
                except BaseException:
                    if counter is not None and again:
                        counter += 1
                    raise
                raised.add((k, at))
                if counter is None:
                    for state in states:
                        state["step"] = at
                if started:
                    done = {id(q) for q in p}
                    started = [q for q in started if id(q) not in done]
        except BaseException:
            for p in started:      # a step that was refused leaves no trace
                self.state.pop(p, None)
            raise
        return loss

    @staticmethod
    def _loaded(k, group, number, p, saved):
        """The state of a parameter from a saved one."""
        step, first, second, rows = int(saved["step"]), saved["exp_avg"], saved["exp_avg_sq"], _state8_rows(group, p)
        if first.shape != p.shape or second.shape != p.shape:
            raise ValueError(f"moments of {tuple(first.shape)} and {tuple(second.shape)} for a parameter of {tuple(p.shape)}")
        made = {"step": step}
        if rows and "exponents" not in saved:
            made.update(zip(("exp_avg", "exp_avg_sq", "exponents"), _state8_of(p, first, second, rows, _rounding_key(group["seed"] + (k << 32), step, number))))
        kind = torch.uint8 if "exponents" in saved else torch.float64 if p.dtype == torch.float64 else torch.float32
        for name, t in saved.items():
            if name not in made:
                made[name] = t.detach().to(device=p.device, dtype=kind if name in ("exp_avg", "exp_avg_sq") else None, copy=True).contiguous() if torch.is_tensor(t) else t
        return made

    def load_state_dict(self, state_dict):
        """Options come from the saved groups, as in torch; those of ``torch.optim.AdamW`` know no ``state_bits`` and ``seed``, so that these and ``capturable`` stay the
        optimizer's own, and with ``state_bits=8`` their moments are brought into 8 bits. Else moments keep the types that they were saved in: torch's own loading would cast all of
        them, codes too, to the weights' type first, and is given none. Groups with ``maximize`` or ``amsgrad`` are refused, with nothing changed."""
        def take(_, saved):
            for group in saved["param_groups"]:
                _check_group(group)
                missing = [name for name in ("lr", "betas", "eps", "weight_decay") if name not in group]
                if missing:
                    raise ValueError(f"no checkpoint of AdamW: its groups have no {', '.join(missing)}")
            self._saved = saved
            mine = {i for group in saved["param_groups"] for i in group["params"]}
            return {**saved, "state": {i: s for i, s in saved["state"].items() if i not in mine}}

        handle = self.register_load_state_dict_pre_hook(take)      # behind the hooks that change it, before anything is taken over
        try:
            super().load_state_dict(state_dict)                    # ends in __setstate__, then hooks that look at what was loaded
        finally:
            handle.remove()
            self._saved = None
