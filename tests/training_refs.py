"""Tokens sorted by expert and AdamW from their definitions, on the host, by loops and in 64 bits. How far results may be off: token_refs.py."""
import math

import torch
from token_refs import U


# ---- tokens sorted by expert -------------------------------------------------------------------------------------------
def order(idx, experts, capacity, align):
    """slot_row, row_slot, counts, base as lists, and the number of rows."""
    flat = idx.reshape(-1).tolist()
    slots = [[s for s, e in enumerate(flat) if e == x][:capacity] for x in range(experts)]
    kept_most = len(flat) if capacity is None else min(len(flat), experts * capacity)
    rows = (kept_most + min(experts, kept_most) * (align - 1)) // align * align
    slot_row, row_slot, base = [-1] * len(flat), [-1] * rows, [0]
    for mine in slots:
        for p, s in enumerate(mine):
            slot_row[s], row_slot[base[-1] + p] = base[-1] + p, s
        base.append(base[-1] + -(-len(mine) // align) * align)
    assert base[-1] <= rows
    return slot_row, row_slot, [len(m) for m in slots], base


def check_order(got, idx, experts, capacity, align):
    want = order(idx, experts, capacity, align)
    assert got.slot_row.shape == idx.shape and all(t.dtype == torch.int32 and t.device == idx.device for t in got)
    for name, g, w in zip(got._fields, got, want):
        assert g.reshape(-1).tolist() == w, name


def sorted_rows(x, row_slot, k):
    """[rows, d]: each row's token, zeros in rows without a slot."""
    out = torch.zeros(row_slot.numel(), x.shape[-1], dtype=x.dtype)
    on = row_slot.cpu() >= 0
    out[on] = x.detach().cpu().reshape(-1, x.shape[-1])[row_slot.cpu().long()[on] // k]
    return out


def returned(rows, slot_row, weights=None):
    """The sum over a token's slots in 64 bits, and the sum of magnitudes."""
    at = slot_row.cpu().long()
    on = at >= 0
    w = torch.ones(at.shape, dtype=torch.float64) if weights is None else weights.detach().cpu().double()
    v = torch.zeros(*at.shape, rows.shape[1], dtype=torch.float64)
    v[on] = rows.detach().cpu().double()[at[on]] * w[on].unsqueeze(-1)
    return v.sum(dim=-2), v.abs().sum(dim=-2)


def return_grads(dy, rows, slot_row, row_slot, weights):
    """Gradients of rows and weights in 64 bits, and the magnitudes behind the second."""
    k, d = slot_row.shape[-1], dy.shape[-1]
    flat, slot = dy.detach().cpu().double().reshape(-1, d), row_slot.cpu().long()
    on = slot >= 0
    g = torch.zeros(slot.numel(), d, dtype=torch.float64)
    g[on] = flat[slot[on] // k] * weights.detach().cpu().double().reshape(-1)[slot[on]].unsqueeze(1)
    dw, size = (torch.zeros(slot_row.numel(), dtype=torch.float64) for _ in range(2))
    product = flat[slot[on] // k] * rows.detach().cpu().double()[on]
    dw[slot[on]], size[slot[on]] = product.sum(dim=1), product.abs().sum(dim=1)
    return g, dw.view(slot_row.shape), size.view(slot_row.shape)


# ---- AdamW ---------------------------------------------------------------------------------------------------------------
def adamw(p, g, m, v, step, lr, betas, eps, wd):
    """p, m, v after a step in 64 bits, and how far fp32 arithmetic may take each: betas and their complements are rounded to fp32 (U each), each product and sum
    adds U of its result; m may cancel, v cannot; the root, its factor, eps, the quotient and the rate add U of the update each."""
    p, g, m, v = (t.detach().cpu().double() for t in (p, g, m, v))
    b1, b2 = betas
    size_m = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    root = v.sqrt() / math.sqrt(1 - b2 ** step) + eps
    rate = lr / (1 - b1 ** step)
    update = rate * m / root
    new = p * (1 - lr * wd) - update
    tiny = 2.0 ** -149      # what a subnormal result is rounded to
    off_m, off_v = 4 * U * size_m + tiny, 6 * U * v + 4 * tiny
    return (new, m, v), (3 * U * p.abs() + U * new.abs() + 14 * U * update.abs() + rate * off_m / root, off_m, off_v)


def _mix(h):
    h ^= h >> 16
    h = h * 0x85EBCA6B & 0xFFFFFFFF
    h ^= h >> 13
    h = h * 0xC2B2AE35 & 0xFFFFFFFF
    return h ^ h >> 16


def _split_mix(x):
    x = (x + 0x9E3779B97F4A7C15) % (1 << 64)
    x = (x ^ x >> 30) * 0xBF58476D1CE4E5B9 % (1 << 64)
    x = (x ^ x >> 27) * 0x94D049BB133111EB % (1 << 64)
    return x ^ x >> 31


def rounding_bits(seed, step, number, n):
    """The 32 bits of each weight of a call's tensor, in Python's whole numbers."""
    key = (_split_mix(_split_mix(seed % (1 << 64)) ^ step) >> 32) + number * 0x9E3779B9
    return [_mix((i + key) & 0xFFFFFFFF) for i in range(n)]


def stored(x, rows, bits, second):
    """What 8 bits keep of the fp32 values ``x``, one value after another in Python's numbers: [rows, blocks of 256] with a power of two each."""
    x = x.detach().cpu().float()
    flat, width = x.reshape(-1).tolist(), x.numel() // rows
    lowest = -30 if second else -14
    out = []
    for r in range(rows):
        for begin in range(0, width, 256):
            block = range(r * width + begin, r * width + min(begin + 256, width))
            if not all(math.isfinite(flat[i]) for i in block):
                out += [math.nan] * len(block)
                continue
            top = max(abs(flat[i]) for i in block)
            e = -87
            if top > 0:
                mantissa, e = math.frexp(top)            # [1/2, 1)
                e = max(e - 1 + (mantissa > 0.9375), -87)
            if e > 127:      # no power of two of fp32
                out += [math.nan] * len(block)
                continue
            for i in block:
                a = abs(flat[i]) * 2.0 ** -e
                binade = max(math.frexp(a)[1] - 1 if a else lowest, lowest)
                unit = 2.0 ** (binade - 3)
                q = math.floor(a / unit + bits[i] / 2 ** 20) * unit
                if second and a > 0:
                    q = max(q, 2.0 ** (lowest - 3))
                out.append(math.copysign(q * 2.0 ** e, flat[i]))
    return torch.tensor(out, dtype=torch.float64).view(x.shape)
