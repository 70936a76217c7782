"""Performance cases of what a training step of a mixture of experts does around the experts' products: tokens sorted by expert and back
with the router's weights, and the AdamW step over the model's tensors with moments in 32 or 8 bits.

``run`` computes an operator in its plain form (elementary torch operations), or with ``own`` set through the library's entry points
(``ops.expert_sort``, ``ops.optim``). A training case of the sorts is one forward and one backward pass. Sizes are those of the library's
example models and benchmarks:

    GPT-MoE          d_model 2048, experts of 2048 x 8192, 64 of them on 8 GPUs or on one, top-2, 8 sequences of 1024 tokens
    Transformer-XL   d_model 512, d_inner 2048, 16 experts, 16 sequences of 512 tokens
    layer benchmark  d_model 4096 and 1024, 16384 tokens, 4 to 64 experts
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256        # weights that share the exponents of their 8-bit moments
MOST_WEIGHTS = 284_000_000
MOST_ROW_BYTES = 1 << 28


def _adamw(name, bits, layers, d, ffn, experts, dtype="bf16", lr=1e-4, weight_decay=0.01, step=100, dense=True):
    c = {"op": "adamw", "bits": bits, "layers": layers, "d": d, "ffn": ffn, "experts": experts, "dense": dense, "dtype": dtype, "lr": lr,
         "weight_decay": weight_decay, "step": step}
    return {"name": name, **c} if name else c


def _rows(op, name, train, tokens, top_k, experts, d, dtype="bf16", align=1, capacity_factor=0.0, masked=0.0, skew=1.0):
    c = {"op": op, "train": train, "tokens": tokens, "top_k": top_k, "experts": experts, "d": d, "dtype": dtype, "align": align,
         "capacity_factor": capacity_factor, "masked": masked, "skew": skew}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one decoding step: a batch of 16 tokens, latency alone
        _rows("sort", "sort_decode", False, 16, 2, 64, 2048),
        # the benchmark model's layer in training, groups on the tiles of the grouped GEMM
        _rows("sort", "sort_gpt_train", True, 8192, 2, 64, 2048, align=128),
        # many small experts of which each token takes eight, a capacity, and padding tokens that are not routed
        _rows("sort", "sort_top8_capacity", True, 16384, 8, 256, 1024, dtype="fp16", align=16, capacity_factor=1.25, masked=0.1),
        # rows that no vector width divides, in fp32
        _rows("sort", "sort_odd", True, 1021, 3, 7, 765, dtype="fp32"),
        # the same ends of the way back
        _rows("back", "back_decode", False, 16, 2, 64, 2048),
        _rows("back", "back_gpt_train", True, 8192, 2, 64, 2048, align=128),
        _rows("back", "back_top8_capacity", True, 16384, 8, 256, 1024, dtype="fp16", align=16, capacity_factor=1.25, masked=0.1),
        _rows("back", "back_wide", False, 16384, 2, 8, 4096),
        # a Transformer-XL of six layers without its experts: a hundred small tensors in fp32
        _adamw("adamw32_small", 32, 6, 512, 2048, 0, dtype="fp32", lr=2.5e-4),
        # one layer of the benchmark model on one of 8 GPUs: attention, router and 8 experts
        _adamw("adamw32_gpt_layer", 32, 1, 2048, 8192, 8),
        # one layer of a model with odd widths in fp16, 4 experts
        _adamw("adamw8_odd", 8, 1, 765, 1531, 4, dtype="fp16", step=3),
        # the benchmark model's layer with moments in 8 bits, which is what lets all of it fit one GPU
        _adamw("adamw8_gpt_layer", 8, 1, 2048, 8192, 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "back", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "adamw":
        layers, d = _log_int(rng, 1, 12), _log_int(rng, 64, 2048) if rng.random() < 0.4 else 64 * _log_int(rng, 1, 32)
        ffn = rng.choice([d, 2 * d, 4 * d, 4 * d + 3])
        experts, dense = rng.choice([0, 1, 4, 8, 64]), rng.random() < 0.7
        dense = dense or experts == 0
        while layers * (4 * d * d + max(1, experts) * 2 * d * ffn) > (MOST_WEIGHTS if dtype != "fp32" else MOST_WEIGHTS // 2):
            layers, experts = max(1, layers // 2), experts // 2
        return _adamw(None, rng.choice([8, 32]), layers, d, ffn, experts, dtype, rng.choice([1e-3, 1e-4, 3e-5]), rng.choice([0.0, 0.01, 0.1]),
                      _log_int(rng, 1, 100000), dense or experts == 0)
    tokens, top_k = _log_int(rng, 1, 16384), rng.choice([1, 2, 2, 3, 4, 6, 8])
    experts = max(top_k, _log_int(rng, 1, 256))
    d = _log_int(rng, 8, 4096) if rng.random() < 0.4 else 8 * _log_int(rng, 1, 512)
    tokens = max(1, min(tokens, MOST_ROW_BYTES // (top_k * d * (4 if dtype == "fp32" else 2))))
    return _rows(op, None, rng.random() < 0.7, tokens, top_k, experts, d, dtype, rng.choice([1, 1, 16, 128]), rng.choice([0.0, 0.0, 1.0, 1.5]),
                 rng.choice([0.0, 0.0, 0.2]), rng.choice([0.0, 1.0, 3.0]))


# ---- inputs, from the seed alone -----------------------------------------------------------------------------------
def _shapes(case):
    """The tensors of a model's layers: two norms, four projections of the attention, the router, the experts or a dense FFN."""
    d, f, e, shapes = case["d"], case["ffn"], case["experts"], []
    for _ in range(case["layers"]):
        if case["dense"]:
            shapes += [(d,)] * 4 + [(d, d), (d,)] * 4
        if e:
            shapes += [(e, d), (e,), (e, f, d), (e, f), (e, d, f), (e, d)]
        else:
            shapes += [(f, d), (f,), (d, f), (d,)]
    return shapes


def _up(n, to):
    return (n + to - 1) // to * to


def _prepare_adamw(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, shapes = DTYPES[case["dtype"]], _shapes(case)
    counts = [math.prod(s) for s in shapes]
    firsts, total = [], 0
    for n in counts:      # the tensors lie one after another, each on a block of its own
        firsts.append(total)
        total += _up(n, BLOCK)
    sizes = torch.tensor([_up(n, BLOCK) for n in counts], device="cuda")
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for first, n in zip(firsts, counts):
        used[first:first + n] = True

    def normal(std):
        return torch.empty(total, dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=g).mul_(std).mul_(used)

    # gradients differ in size from place to place, and an expert without tokens has none
    scale = torch.empty(total // BLOCK, 1, device="cuda").normal_(0.0, 1.0, generator=g).exp_().mul_(1e-3).expand(-1, BLOCK).reshape(-1)
    idle = (torch.rand(total // BLOCK, 1, generator=g, device="cuda") < 0.1).expand(-1, BLOCK).reshape(-1)
    p, grad = normal(0.02).to(dt), normal(scale).masked_fill_(idle, 0.0).to(dt)
    m = normal(scale * 0.3)
    v = normal(0.5).exp_().mul_(scale).mul_(scale).mul_(used)

    def split(flat):
        return [flat[first:first + n].view(shape) for first, n, shape in zip(firsts, counts, shapes)]

    s = {"case": case, "p": p, "g": grad, "sizes": sizes, "params": split(p), "grads": split(grad), "seed": 1000 + seed}
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        key, at = _keys(sizes, 99, case["step"])
        h = _hash(at, key)
        s["m"], em = _encode(m, h & 0xFFFFF, False)
        s["v"], ev = _encode(v, (h >> 12) & 0xFFFFF, True)
        s["exponents"] = torch.stack([em, ev], dim=1)
        s["block_exponents"] = [s["exponents"][first // BLOCK:(first + _up(n, BLOCK)) // BLOCK].unsqueeze(0) for first, n in zip(firsts, counts)]
    s["first_moments"], s["second_moments"] = split(s["m"]), split(s["v"])
    return s


def _routes(case, g):
    """Expert ids [tokens, top_k] as a router gives them: the best of scores with a preference for some experts; masked tokens have none."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    favour = torch.randn(e, generator=g, device="cuda") * case["skew"]
    score, idx = torch.topk(torch.randn(t, e, generator=g, device="cuda") + favour, k, dim=1)
    idx = idx.to(torch.int32)
    if case["masked"]:
        idx = torch.where(torch.rand(t, 1, generator=g, device="cuda") < case["masked"], torch.full_like(idx, -1), idx)
    return idx, torch.softmax(score, dim=1)


def _capacity(case):
    slots = case["tokens"] * case["top_k"]
    return min(slots, math.ceil(case["capacity_factor"] * slots / case["experts"])) if case["capacity_factor"] else None


def _row_count(case):
    """Rows that hold every slot, whatever the routing: each expert that can have tokens may add a part of a tile."""
    slots, e, a, cap = case["tokens"] * case["top_k"], case["experts"], case["align"], _capacity(case)
    kept = slots if cap is None else min(slots, e * cap)
    return (kept + min(e, kept) * (a - 1)) // a * a


def prepare(case, seed):
    if case["op"] == "adamw":
        return _prepare_adamw(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, t, d, rows = DTYPES[case["dtype"]], case["tokens"], case["d"], _row_count(case)

    def normal(*shape):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, 1.0, generator=g)

    idx, weights = _routes(case, g)
    s = {"case": case, "idx": idx}
    if case["op"] == "sort":
        s["x"] = normal(t, d).requires_grad_(case["train"])
        s["grad"] = normal(rows, d) if case["train"] else None
    else:
        s["order"] = _order(idx, case)
        s["rows"] = normal(rows, d).requires_grad_(case["train"])
        s["weights"] = weights.requires_grad_(case["train"])
        s["grad"] = normal(t, d) if case["train"] else None
    return s


# ---- the library's operators ------------------------------------------------------------------------------------------
def _run_own(s):
    case = s["case"]
    if case["op"] == "adamw":
        from ccfuser_b200.ops.optim import adamw_step, state_values
        adamw_step(s["params"], s["grads"], s["first_moments"], s["second_moments"], case["step"], lr=case["lr"], weight_decay=case["weight_decay"],
                   exponents=s.get("block_exponents"), seed=s["seed"])
        if case["bits"] == 32:
            return [s["p"], s["m"], s["v"]]
        return [s["p"], state_values(s["m"], s["exponents"]), state_values(s["v"], s["exponents"], second=True)]
    from ccfuser_b200.ops.expert_sort import ExpertOrder, return_rows, sort_by_expert
    if case["op"] == "sort":
        rows, order = sort_by_expert(s["x"], s["idx"], case["experts"], capacity=_capacity(case), align=case["align"])
        out = [rows.detach(), order.slot_row, order.row_slot, order.counts, order.base]
        return out + (list(torch.autograd.grad(rows, [s["x"]], s["grad"])) if case["train"] else [])
    y = return_rows(s["rows"], ExpertOrder(*s["order"]), s["weights"])
    return [y.detach()] + (list(torch.autograd.grad(y, [s["rows"], s["weights"]], s["grad"])) if case["train"] else [])


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _order(idx, case):
    """Row of each slot (-1: none), slot of each row (-1: none), rows of each expert, first row of each expert and behind the last."""
    e, a, cap, rows = case["experts"], case["align"], _capacity(case), _row_count(case)
    flat = idx.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < e), flat, torch.full_like(flat, e))
    sorted_key, order = torch.sort(key, stable=True)
    ends = torch.searchsorted(sorted_key, torch.arange(e + 1, device="cuda"), right=True)
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    counts = (ends - starts)[:e]
    if cap is not None:
        counts = counts.clamp(max=cap)
    base = torch.cat([ends.new_zeros(1), torch.cumsum((counts + a - 1) // a * a, 0)])
    pos = torch.arange(n, device="cuda") - starts[sorted_key]
    kept = (sorted_key < e) & (pos < torch.cat([counts, counts.new_zeros(1)])[sorted_key])
    row = torch.where(kept, base[sorted_key] + pos, torch.full_like(pos, rows))      # the others go to a row behind the last
    row_slot = torch.full((rows + 1,), -1, dtype=torch.int32, device="cuda")
    row_slot[row] = order.int()
    slot_row = torch.empty(n, dtype=torch.int32, device="cuda")
    slot_row[order] = torch.where(kept, row, torch.full_like(row, -1)).int()
    return slot_row.view(idx.shape), row_slot[:rows], counts.int(), base.int()


def _gathered(rows, slot_row):
    """Each slot's row in fp32, zeros where it has none: [tokens, top_k, d]."""
    at = slot_row.long()
    return rows.float()[at.clamp(min=0)] * (at >= 0)[..., None] if rows.shape[0] else torch.zeros(*at.shape, rows.shape[1], device="cuda")


def _to_rows(values, slot_row, rows):
    """[tokens, top_k, d] or [tokens, 1, d] to their rows, zeros elsewhere."""
    at = slot_row.reshape(-1).long()
    out = torch.zeros(rows + 1, values.shape[-1], dtype=values.dtype, device="cuda")
    out[torch.where(at < 0, torch.full_like(at, rows), at)] = values.expand(*slot_row.shape, -1).reshape(at.numel(), -1)
    return out[:rows]


def _plain_rows(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    if case["op"] == "sort":
        order = _order(s["idx"], case)
        out = [_to_rows(s["x"].detach()[:, None], order[0], _row_count(case)), *order]
        return out + ([_gathered(s["grad"], order[0]).sum(dim=1).to(dt)] if case["train"] else [])
    at, w = s["order"][0], s["weights"].detach()
    rows = _gathered(s["rows"].detach(), at)
    out = [(rows * w[..., None]).sum(dim=1).to(dt)]
    if not case["train"]:
        return out
    dy = s["grad"].float()[:, None]
    return out + [_to_rows((dy * w[..., None]).to(dt), at, _row_count(case)), (rows * dy).sum(dim=-1)]


MASK = 0xFFFFFFFF


def _mix(h):
    """The last step of MurmurHash3 on whole numbers of 32 bits."""
    h ^= h >> 16
    h = h * 0x85EBCA6B & MASK
    h ^= h >> 13
    h = h * 0xC2B2AE35 & MASK
    return h ^ h >> 16


def _split_mix(x):
    """SplitMix64's output for the state x."""
    x = (x + 0x9E3779B97F4A7C15) % (1 << 64)
    x = (x ^ x >> 30) * 0xBF58476D1CE4E5B9 % (1 << 64)
    x = (x ^ x >> 27) * 0x94D049BB133111EB % (1 << 64)
    return x ^ x >> 31


def _key(seed, step):
    return _split_mix(_split_mix(seed) ^ step) >> 32


def _int32(n):
    return n - (1 << 32) if n >= 1 << 31 else n


def _hash(at, key):
    """32 bits for each element: the mixed sum of its number in its tensor and the tensor's key, in int32 that wrap around."""
    h = at + key
    h = h ^ ((h >> 16) & 0xFFFF)
    h = h * _int32(0x85EBCA6B)
    h = h ^ ((h >> 13) & 0x7FFFF)
    h = h * _int32(0xC2B2AE35)
    return h ^ ((h >> 16) & 0xFFFF)


def _keys(sizes, seed, step):
    """For each element the key of its tensor and its number in it, for tensors one after another."""
    number = torch.arange(sizes.numel(), dtype=torch.int64, device="cuda")
    keys = (_key(seed, step) + number * 0x9E3779B9) & MASK
    keys = torch.where(keys >= 1 << 31, keys - (1 << 32), keys).int()
    first = torch.cumsum(sizes, 0) - sizes
    which = torch.repeat_interleave(number, sizes)
    return keys[which], (torch.arange(which.numel(), device="cuda") - first[which]).int()


def _power(exponent, plus):
    """2^(exponent + plus) in fp32, for results between 2^-126 and 2^127."""
    return ((exponent.int() + plus + 127) << 23).view(torch.float32)


def _encode(x, bits, second):
    """Values to 8-bit codes and the biased exponents of their blocks. The first moment: sign, 4 bits of exponent, 3 of mantissa. The second: 5 and 3, and
    what is not zero never becomes zero. 20 given bits decide between the two codes next to a value."""
    a = x.abs().view(-1, BLOCK)
    largest = a.view(torch.int32).amax(dim=1, keepdim=True)
    e = torch.where(largest < 0x7F800000, (largest + 0xFFFFF) >> 23, torch.full_like(largest, 255)).clamp(min=40)
    finite = e < 255
    e0 = torch.where(finite, e, torch.full_like(e, 127)) - 127
    # so far down that the code is what the upper bits of the float say
    y = a * _power(4 - e0, 0) * 2.0 ** -100 if second else a * _power(8 - e0, 0) * 2.0 ** -120
    code = (y.view(torch.int32) + bits.view(-1, BLOCK)) >> 20
    if second:
        code = torch.where(a > 0, code.clamp(min=1), code)
    else:
        code = code | (x.view(-1, BLOCK).view(torch.int32) >> 24) & 0x80
    return torch.where(finite, code, torch.zeros_like(code)).to(torch.uint8).view(-1), e.to(torch.uint8).view(-1)


def _decode(codes, exponents, second):
    c, e = codes.view(-1, BLOCK).int(), exponents.int()[:, None]
    e0 = torch.where(e < 255, e, torch.full_like(e, 127)) - 127
    if second:
        x = (c << 20).view(torch.float32) * 2.0 ** 100 * _power(e0.clamp(min=-87) - 4, 0)
    else:
        x = (((c & 0x7F) << 20) | ((c & 0x80) << 24)).view(torch.float32) * 2.0 ** 120 * _power(e0.clamp(min=-87) - 8, 0)
    return torch.where(e < 255, x, torch.full_like(x, math.nan)).view(-1)


def _plain_adamw(s):
    case = s["case"]
    b1, b2, eps, lr, t = 0.9, 0.999, 1e-8, case["lr"], case["step"]
    eight = case["bits"] == 8
    m = _decode(s["m"], s["exponents"][:, 0], False) if eight else s["m"]
    v = _decode(s["v"], s["exponents"][:, 1], True) if eight else s["v"]
    g = s["g"].float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    p = s["p"].float() * (1 - lr * case["weight_decay"]) - m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps) * (lr / (1 - b1 ** t))
    s["p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return [s["p"], s["m"], s["v"]]
    key, at = _keys(s["sizes"], s["seed"], t)
    h = _hash(at, key)
    for name, x, bits, second in (("m", m, h & 0xFFFFF, False), ("v", v, (h >> 12) & 0xFFFFF, True)):
        codes, e = _encode(x, bits, second)
        s[name].copy_(codes)
        s["exponents"][:, int(second)] = e
    return [s["p"], _decode(s["m"], s["exponents"][:, 0], False).bfloat16(), _decode(s["v"], s["exponents"][:, 1], True).bfloat16()]


def run(s):
    if own:
        return _run_own(s)
    return _plain_adamw(s) if s["case"]["op"] == "adamw" else _plain_rows(s)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _stored(x, bits, second):
    """What a moment stands for once it is held in 8 bits: a multiple of its binade's step, or of the smallest binade's, relative to its block's 2^e."""
    a = x.abs().view(-1, BLOCK)
    top = a.amax(dim=1, keepdim=True)
    mantissa, e = torch.frexp(top)                   # top = mantissa * 2^e, mantissa in [1/2, 1)
    e = e - 1 + (mantissa > 0.9375).to(e.dtype)      # one binade more where rounding up could leave the largest
    e = torch.where(top > 0, e, torch.full_like(e, -87)).clamp(min=-87).double()
    y = a * torch.exp2(-e)
    lowest = -30 if second else -14
    binade = (torch.frexp(y)[1] - 1).clamp(min=lowest).double()
    step = torch.exp2(binade - 3)
    q = torch.floor(y / step + bits.view(-1, BLOCK).double() / 2 ** 20) * step
    if second:
        q = torch.where(a > 0, q.clamp(min=2.0 ** (lowest - 3)), q)
    return (q * torch.exp2(e) * x.view(-1, BLOCK).sign()).view(-1)


def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    t, lr, p, g = case["step"], case["lr"], s["p"].double(), s["g"].double()
    eight = case["bits"] == 8
    m = (_decode(s["m"], s["exponents"][:, 0], False) if eight else s["m"]).double()      # exact: three bits of mantissa
    v = (_decode(s["v"], s["exponents"][:, 1], True) if eight else s["v"]).double()
    m += (g - m) / 10
    v += (g * g - v) / 1000
    update = (m / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
    p -= lr * (case["weight_decay"] * p + update)
    if eight:
        n, key = s["sizes"].tolist(), _key(s["seed"], t)
        h = torch.cat([_mix((torch.arange(k, dtype=torch.int64, device="cuda") + (key + i * 0x9E3779B9)) & MASK) for i, k in enumerate(n)])
        m, v = _stored(m, h & 0xFFFFF, False), _stored(v, h >> 12, True)
    return [p, m, v]


def _exact_rows(case, seed):
    s = prepare(case, seed)
    e, a, cap, rows, k = case["experts"], case["align"], _capacity(case), _row_count(case), case["top_k"]
    idx = s["idx"].reshape(-1).long()
    slot_row = torch.full((idx.numel(),), -1, dtype=torch.int64, device="cuda")
    first = 0
    for i in range(e):
        slots = (idx == i).nonzero()[:, 0][:cap]
        slot_row[slots] = first + torch.arange(slots.numel(), device="cuda")
        first += _up(slots.numel(), a)
    kept = (slot_row >= 0).nonzero()[:, 0]
    at, token = slot_row[kept], kept // k
    d = case["d"]

    def summed(rows_, scale):
        return torch.zeros(case["tokens"], d, dtype=torch.float64, device="cuda").index_add_(0, token, rows_.double()[at] * scale)

    def spread(values):
        out = torch.zeros(rows, d, dtype=torch.float64, device="cuda")
        out[at] = values
        return out

    if case["op"] == "sort":
        out = [spread(s["x"].detach().double()[token]), None, None, None, None]
        return out + ([summed(s["grad"], 1.0)] if case["train"] else [])
    w = s["weights"].detach().double().reshape(-1)[kept, None]
    out = [summed(s["rows"].detach(), w)]
    if not case["train"]:
        return out
    dy = s["grad"].double()[token]
    dw = torch.zeros(idx.numel(), dtype=torch.float64, device="cuda")
    dw[kept] = (dy * s["rows"].detach().double()[at]).sum(dim=1)
    return out + [spread(dy * w), dw.view(-1, k)]


def exact(case, seed):
    return _exact_adamw(case, seed) if case["op"] == "adamw" else _exact_rows(case, seed)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        # weights read and written, gradients read, moments read and written; those of 8 bits are also handed over as 16-bit values
        return {"bytes": n * (3 * size + (16 if case["bits"] == 32 else 8)), "flops": 14.0 * n}
    t, k, d, rows, cap = case["tokens"], case["top_k"], case["d"], _row_count(case), _capacity(case)
    slots = t * k
    kept = slots * (1 - case["masked"])
    if cap is not None:
        kept = min(kept, case["experts"] * cap)
    if case["op"] == "sort":
        nbytes = t * d * size + rows * d * size + 8 * slots + 4 * rows
        if case["train"]:
            nbytes += (kept + t) * d * size
        return {"bytes": nbytes, "flops": kept * d if case["train"] else 0}
    nbytes = (kept + t) * d * size + 8 * slots
    if case["train"]:
        nbytes += (kept + t + rows) * d * size + 8 * slots
    return {"bytes": nbytes, "flops": 2.0 * kept * d * (3 if case["train"] else 1)}
