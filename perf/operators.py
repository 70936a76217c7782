"""Performance cases of the operators at both ends of a training or scoring step: token embedding, log probabilities of given
tokens, and dropout on the residual stream.

``run`` computes an operator in its plain form (elementary torch operations in fp32), or with ``own`` set through the library's entry points
(``ops.embedding``, ``ops.logprobs``, ``ops.dropout``). A training case is one forward and one backward pass. Sizes are those of
the library's example models and benchmark:

    GPT-MoE          vocabulary 50257 (50304 padded), d_model 2048, 8 sequences of 1024 tokens
    Transformer-XL   vocabulary 100, d_model 512, 16 sequences of 512 tokens, embedding scaled by sqrt(d_model)
    BERT             vocabulary 30522, d_model 768, three tables added
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100


def _embed(name, train, batch, seq, vocab, d, dtype="bf16", scale=1.0, positions="none", types=0, ids="zipf", padding=False):
    c = {"op": "embed", "train": train, "batch": batch, "seq": seq, "vocab": vocab, "d": d, "dtype": dtype, "scale": scale,
         "positions": positions, "types": types, "ids": ids, "padding": padding}
    return {"name": name, **c} if name else c


def _logprobs(name, train, rows, vocab, width=0, dtype="bf16", top_k=0, temperature=1.0, entropy=False, mask="none", ignored=0.0):
    c = {"op": "logprobs", "train": train, "rows": rows, "vocab": vocab, "width": width or vocab, "dtype": dtype, "top_k": top_k,
         "temperature": temperature, "entropy": entropy, "mask": mask, "ignored": ignored}
    return {"name": name, **c} if name else c


def _dropout(name, train, rows, d, dtype="bf16", p=0.1, residual=True):
    c = {"op": "dropout", "train": train, "rows": rows, "d": d, "dtype": dtype, "p": p, "residual": residual}
    return {"name": name, **c} if name else c


def listed():
    return [
        # decoding: the newest token of 16 sequences, each at its own position
        _embed("embed_decode", False, 16, 1, 50304, 2048, positions="given"),
        # Transformer-XL training: few words, so every word's gradient is a sum over many tokens
        _embed("embed_few_words", True, 16, 512, 100, 512, scale=math.sqrt(512.0), ids="uniform"),
        # the GPT-MoE step: word and position table, a dense gradient of the whole vocabulary
        _embed("embed_gpt", True, 8, 1024, 50304, 2048, positions="order"),
        # BERT fine-tuning on a padded batch of odd length in fp16: three tables, the padding word has no gradient
        _embed("embed_padded", True, 23, 381, 30522, 768, dtype="fp16", positions="order", types=2, ids="padded", padding=True),
        # answering: the sampled tokens of 4 sequences with their 20 best alternatives
        _logprobs("score_decode", False, 4, 50257, top_k=20, temperature=0.7),
        # the same under a grammar that allows few tokens, the others at -inf, fp32 logits
        _logprobs("score_grammar", False, 61, 30522, dtype="fp32", top_k=8, mask="inf"),
        # scoring a text: every token's log probability, entropy and 5 alternatives, rows off a 16-byte boundary
        _logprobs("score_text", False, 4099, 50257, top_k=5),
        # the GPT-MoE loss over the padded vocabulary, forward and backward
        _logprobs("loss_gpt", True, 8192, 50257, width=50304, ignored=0.02),
        # policy gradient with an entropy bonus: gradients into both outputs, fp16 logits, an odd number of rows
        _logprobs("loss_entropy", True, 1025, 30522, dtype="fp16", temperature=1.3, entropy=True),
        # a small Transformer-XL block: the branch's output joins the residual stream
        _dropout("dropout_block", True, 2048, 512),
        # dropout of activations alone, fp32, a number of elements that no vector width divides
        _dropout("dropout_odd", True, 1013, 1021, dtype="fp32", p=0.25, residual=False),
        # the widest block of the layer benchmark
        _dropout("dropout_wide", True, 16384, 4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "logprobs", "dropout"])
    dtype, train = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6
    if op == "embed":
        batch, seq = _log_int(rng, 1, 64), _log_int(rng, 1, 2048)
        batch = max(1, min(batch, 32768 // seq))
        d = _log_int(rng, 16, 4096) if rng.random() < 0.3 else 8 * _log_int(rng, 2, 512)
        kind = rng.choice(["uniform", "zipf", "padded"])
        vocab = min(_log_int(rng, 50, 65536), (1 << 27) // d)
        return _embed(None, train, batch, seq, vocab, d, dtype, rng.choice([1.0, math.sqrt(d)]),
                      rng.choice(["none", "order", "given"]), rng.choice([0, 0, 2]), kind, kind == "padded" and rng.random() < 0.7)
    if op == "logprobs":
        vocab, mask = _log_int(rng, 100, 200000), rng.choice(["none", "none", "inf", "lowest"])
        rows = _log_int(rng, 1, max(2, min(8192, 200_000_000 // vocab)))
        return _logprobs(None, train, rows, vocab, vocab if rng.random() < 0.5 else (vocab + 127) // 128 * 128, dtype,
                         rng.choice([0, 0, 1, 5, 20]), rng.choice([1.0, 1.0, 1.3] + [0.7] * (mask != "lowest")), rng.random() < 0.5, mask, rng.choice([0.0, 0.1]))
    return _dropout(None, train, _log_int(rng, 1, 16384), _log_int(rng, 64, 4096), dtype, rng.choice([0.1, 0.1, 0.25, 0.5]), rng.random() < 0.7)


# ---- inputs, from the seed alone -----------------------------------------------------------------------------------
def _normal(g, dt, *shape, std=1.0):
    return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, std, generator=g)


def _word_ids(case, g):
    """Word ids: uniform; by Zipf's law in a random order of the words, as text has them; or that with a tail of padding (id 0) per row."""
    b, s, v = case["batch"], case["seq"], case["vocab"]
    if case["ids"] == "uniform":
        return torch.randint(0, v, (b, s), generator=g, device="cuda")
    u = torch.rand(b, s, generator=g, device="cuda", dtype=torch.float64)
    rank = ((v + 1.0) ** u - 1.0).floor().long().clamp_(0, v - 1)        # density proportional to 1 / (rank + 1)
    ids = torch.randperm(v, generator=g, device="cuda")[rank]
    if case["ids"] == "padded":
        length = torch.randint(max(1, s // 4), s + 1, (b, 1), generator=g, device="cuda")
        ids = torch.where(torch.arange(s, device="cuda") < length, ids, torch.zeros_like(ids))
    return ids


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]
    s = {"case": case}
    if case["op"] == "embed":
        b, n, d = case["batch"], case["seq"], case["d"]
        s["ids"] = _word_ids(case, g)
        s["weight"] = _normal(g, dt, case["vocab"], d, std=0.02).requires_grad_(train)
        s["position"] = s["position_ids"] = s["type"] = s["type_ids"] = None
        if case["positions"] != "none":
            s["position"] = _normal(g, dt, max(n, 1024), d, std=0.02).requires_grad_(train)
        if case["positions"] == "given":
            first = torch.randint(0, max(n, 1024) - n + 1, (b, 1), generator=g, device="cuda")
            s["position_ids"] = first + torch.arange(n, device="cuda")
        if case["types"]:
            s["type"] = _normal(g, dt, case["types"], d, std=0.02).requires_grad_(train)
            s["type_ids"] = (torch.arange(n, device="cuda") >= torch.randint(1, n + 1, (b, 1), generator=g, device="cuda")).long()
        s["grad"] = _normal(g, dt, b, n, d) if train else None
    elif case["op"] == "logprobs":
        rows, v, width = case["rows"], case["vocab"], case["width"]
        x = _normal(g, dt, rows, width, std=3.0)
        targets = torch.randint(0, v, (rows,), generator=g, device="cuda")
        # the model expects the right token more often than not: a few units above the others
        x.scatter_add_(1, targets[:, None], (torch.rand(rows, 1, generator=g, device="cuda") * 12.0).to(dt))
        if case["mask"] != "none":
            allowed = torch.rand(rows, width, generator=g, device="cuda") < 0.01
            allowed.scatter_(1, targets[:, None], True)
            x.masked_fill_(~allowed, -math.inf if case["mask"] == "inf" else torch.finfo(dt).min)
        if case["ignored"]:
            targets[torch.rand(rows, generator=g, device="cuda") < case["ignored"]] = IGNORE
        s["logits"], s["targets"] = x.requires_grad_(train), targets
        if train:
            k = case["top_k"]
            s["grads"] = [_normal(g, torch.float32, rows)] + ([_normal(g, torch.float32, rows, std=0.1)] if case["entropy"] else [])
            s["grads"] += [_normal(g, torch.float32, rows, k, std=0.1)] if k and case["mask"] == "none" else []
    else:
        rows, d = case["rows"], case["d"]
        s["x"] = _normal(g, dt, rows, d).requires_grad_(train)
        s["residual"] = _normal(g, dt, rows, d).requires_grad_(train) if case["residual"] else None
        s["grad"] = _normal(g, dt, rows, d) if train else None
        s["state"] = torch.tensor([0x9E3779B97F4A7C15 % (1 << 61) + seed, 17 + seed % 1000], dtype=torch.int64, device="cuda")
        s["call"] = 5
    return s


# ---- the library's operators ------------------------------------------------------------------------------------------
def _run_own(s):
    case = s["case"]
    if case["op"] == "embed":
        from ccfuser_b200.ops.embedding import embedding
        y = embedding(s["ids"], s["weight"], case["scale"], position_weight=s["position"], position_ids=s["position_ids"],
                      type_weight=s["type"], type_ids=s["type_ids"], padding_idx=0 if case["padding"] else None)
        if not case["train"]:
            return [y]
        tables = [t for t in (s["weight"], s["position"], s["type"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, tables, s["grad"])]
    if case["op"] == "logprobs":
        from ccfuser_b200.ops.logprobs import token_logprobs
        r = token_logprobs(s["logits"], s["targets"], top_k=case["top_k"], temperature=case["temperature"], vocab_size=case["vocab"],
                           ignore_index=IGNORE)
        out = [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_ids] if case["top_k"] else [])
        if not case["train"]:
            return out
        used = [r.logprobs] + ([r.entropy] if case["entropy"] else []) + ([r.top_logprobs] if len(s["grads"]) > 1 + case["entropy"] else [])
        grad, = torch.autograd.grad(used, [s["logits"]], s["grads"])
        return [t.detach() for t in out] + [grad]
    from ccfuser_b200.ops.dropout import dropout
    y = dropout(s["x"], case["p"], s["state"], s["call"], residual=s["residual"])
    if not case["train"]:
        return [y]
    inputs = [t for t in (s["x"], s["residual"]) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, inputs, s["grad"])]


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _table_grad(ids, grad, rows):
    return torch.zeros(rows, grad.shape[-1], dtype=torch.float32, device="cuda").index_add_(0, ids.reshape(-1), grad.reshape(-1, grad.shape[-1]))


def _plain_embed(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    ids, pos = s["ids"], s["position_ids"]
    y = s["weight"].detach()[ids].float() * case["scale"]
    if s["position"] is not None:
        if pos is None:
            pos = torch.arange(case["seq"], device="cuda").expand(case["batch"], case["seq"])
        y = y + s["position"].detach()[pos].float()
    if s["type"] is not None:
        y = y + s["type"].detach()[s["type_ids"]].float()
    out = [y.to(dt)]
    if case["train"]:
        grad = s["grad"].float()
        dw = _table_grad(ids, grad, case["vocab"]) * case["scale"]
        if case["padding"]:
            dw[0] = 0.0
        out.append(dw.to(dt))
        out += [_table_grad(pos, grad, s["position"].shape[0]).to(dt)] if s["position"] is not None else []
        out += [_table_grad(s["type_ids"], grad, s["type"].shape[0]).to(dt)] if s["type"] is not None else []
    return out


def _top(x, k):
    """The k largest of each row, equal ones by their index: one whole number holds the value's order and, below it, the index."""
    bits = (x.float() + 0.0).view(torch.int32).long()                    # + 0.0: -0 and 0 are equal
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device="cuda"))
    return (1 << 20) - 1 - (key.topk(k, dim=1).values & ((1 << 20) - 1))


def _plain_logprobs(s):
    case = s["case"]
    v, temp, k, t = case["vocab"], case["temperature"], case["top_k"], s["targets"]
    x = s["logits"].detach()
    z = x[:, :v].float() / temp
    z = z - z.max(dim=1, keepdim=True).values
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    lp, p = z - total.log(), e / total
    h = total.log()[:, 0] - (p * z.masked_fill(p == 0, 0.0)).sum(dim=1)
    kept = t != IGNORE
    at = torch.where(kept, t, torch.zeros_like(t))[:, None]
    out = [torch.where(kept, lp.gather(1, at)[:, 0], 0.0), h]
    if k:
        ids = _top(x[:, :v], k)
        out += [lp.gather(1, ids), torch.where(x.gather(1, ids) == -math.inf, -1, ids)]
    if case["train"]:
        g = torch.where(kept, s["grads"][0], 0.0)[:, None]
        along = g
        gh = s["grads"][1][:, None] if case["entropy"] else None
        gk = s["grads"][-1] if len(s["grads"]) > 1 + case["entropy"] else None
        if gk is not None:
            along = along + gk.sum(dim=1, keepdim=True)
        d = -p * along
        if gh is not None:
            d = d - gh * p * (lp.masked_fill(p == 0, 0.0) + h[:, None])
        d.scatter_add_(1, at, g)
        if gk is not None:
            d.scatter_add_(1, ids, gk)
        full = torch.zeros_like(x)
        full[:, :v] = (d / temp).to(x.dtype)
        out.append(full)
    return out


def _plain_keep(s, n):
    """Philox4x32-10 of (number of the group of eight, call, step) under the seed, in whole numbers of 64 bits; 16 bits an element."""
    seed, step = s["state"][0], s["state"][1]
    low = 0xFFFFFFFF
    group = torch.arange((n + 7) // 8, dtype=torch.int64, device="cuda")
    c0, c1 = group & low, group >> 32
    c2, c3 = torch.full_like(group, s["call"] & low), (step & low).expand_as(group)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    r = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    return r >= round(s["case"]["p"] * 65536)


def _plain_dropout(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    keep = _plain_keep(s, s["x"].numel()).view(s["x"].shape)
    up = 65536.0 / (65536 - round(case["p"] * 65536))
    y = torch.where(keep, s["x"].detach().float() * up, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    out = [y.to(dt)]
    if case["train"]:
        out.append(torch.where(keep, s["grad"].float() * up, 0.0).to(dt))
        out += [s["grad"]] if s["residual"] is not None else []
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"embed": _plain_embed, "logprobs": _plain_logprobs, "dropout": _plain_dropout}[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "embed":
        n, d, v = case["batch"] * case["seq"], case["d"], case["vocab"]
        tables = 1 + (case["positions"] != "none") + (case["types"] > 0)
        used = min(n, v) + (min(n, case["seq"]) if case["positions"] != "none" else 0) + case["types"]
        nbytes, flops = (used + n) * d * size + 8 * n * tables, n * d * tables
        if case["train"]:
            rows = v + (max(case["seq"], 1024) if case["positions"] != "none" else 0) + case["types"]
            nbytes, flops = nbytes + (n + rows) * d * size, flops + n * d * tables
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "logprobs":
        rows, v = case["rows"], case["vocab"]
        nbytes, flops = rows * (v * size + 16 + 12 * case["top_k"]), 8 * rows * v
        if case["train"]:
            nbytes, flops = nbytes + rows * (v + case["width"]) * size, flops + 6 * rows * v
        return {"bytes": nbytes, "flops": flops}
    n = case["rows"] * case["d"]
    arrays = 2 + case["residual"] + 2 * case["train"]
    return {"bytes": arrays * n * size, "flops": n * (12 + 12 * case["train"])}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_sum_by_row(ids, grad, rows):
    """Sums in the order of the sorted ids: differences of a running total would lose bits, so every run is added by itself."""
    order = torch.argsort(ids, stable=True)
    sorted_ids = ids[order]
    got, counts = torch.unique_consecutive(sorted_ids, return_counts=True)
    out = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // max(1, grad.shape[0]))
    for c in range(0, grad.shape[1], step):
        out[got, c:c + step] = torch.segment_reduce(grad[order, c:c + step].double(), "sum", lengths=counts, axis=0)
    return out


def _exact_embed(case, s):
    b, n, d = case["batch"], case["seq"], case["d"]
    tables = [(s["weight"], s["ids"].reshape(-1), case["scale"])]
    if s["position"] is not None:
        pos = s["position_ids"].reshape(-1) if s["position_ids"] is not None else torch.arange(b * n, device="cuda") % n
        tables.append((s["position"], pos, 1.0))
    if s["type"] is not None:
        tables.append((s["type"], s["type_ids"].reshape(-1), 1.0))
    y = torch.zeros(b * n, d, dtype=torch.float64, device="cuda")
    for w, i, scale in tables:
        y += w.detach().index_select(0, i).double() * scale
    out = [y.view(b, n, d)]
    if case["train"]:
        for k, (w, i, scale) in enumerate(tables):
            dw = _exact_sum_by_row(i, s["grad"].reshape(b * n, d), w.shape[0]) * scale
            if k == 0 and case["padding"]:
                dw[0].zero_()
            out.append(dw)
    return out


def _exact_logprobs(case, s):
    v, k, temp = case["vocab"], case["top_k"], case["temperature"]
    parts = []
    step = max(1, (1 << 26) // v)
    for r in range(0, case["rows"], step):
        x, t = s["logits"].detach()[r:r + step], s["targets"][r:r + step]
        z = x[:, :v].double() / temp
        lse = torch.logsumexp(z, dim=1)
        lp = z - lse[:, None]
        p = lp.exp()
        h = -torch.special.xlogy(p, p).sum(dim=1)
        live = t.ne(IGNORE)
        rows = torch.arange(x.shape[0], device="cuda")
        got = [torch.where(live, lp[rows, t.clamp_min(0)], 0.0), h]
        if k:
            top = torch.sort(x[:, :v].double(), dim=1, descending=True, stable=True).indices[:, :k]
            got += [torch.gather(lp, 1, top), top.masked_fill(torch.isneginf(torch.gather(x, 1, top)), -1)]
        if case["train"]:
            grads = [g[r:r + step].double() for g in s["grads"]]
            up = torch.zeros_like(lp)                                      # gradient with respect to every log probability
            up[rows[live], t[live]] += grads[0][live]
            if len(grads) > 1 + case["entropy"]:
                up.scatter_add_(1, top, grads[-1])
            d = up - p * up.sum(dim=1, keepdim=True)
            if case["entropy"]:
                d -= grads[1][:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            whole = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
            whole[:, :v] = d / temp
            got.append(whole.to(torch.float32 if x.dtype != torch.float32 else torch.float64))
        parts.append(got)
    return [torch.cat([p[i] for p in parts]) for i in range(len(parts[0]))]


def _exact_bits(seed, step, call, n):
    """The generator again, on the host in unsigned 64-bit numbers, from its published definition (Salmon et al., 2011)."""
    m0, m1, mask = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    x = [g & mask, g >> half, np.full_like(g, call & 0xFFFFFFFF), np.full_like(g, step & 0xFFFFFFFF)]
    for r in range(10):
        k0, k1 = (seed + r * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF
        p0, p1 = m0 * x[0], m1 * x[2]
        x = [(p1 >> half) ^ x[1] ^ np.uint64(k0), p1 & mask, (p0 >> half) ^ x[3] ^ np.uint64(k1), p0 & mask]
    return np.stack(x, 1).astype("<u4").view("<u2").reshape(-1)[:n].astype(np.int32)


def _exact_dropout(case, s):
    seed, step = (int(i) for i in s["state"].tolist())
    drop = round(case["p"] * 65536)
    bits = torch.from_numpy(_exact_bits(seed, step, s["call"], s["x"].numel())).cuda().view(s["x"].shape)
    keep = (bits >= drop).double() * (65536.0 / (65536 - drop))
    y = s["x"].detach().double() * keep
    out = [y if s["residual"] is None else y + s["residual"].detach().double()]
    if case["train"]:
        out.append(s["grad"].double() * keep)
        out += [s["grad"].double()] if s["residual"] is not None else []
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "logprobs": _exact_logprobs, "dropout": _exact_dropout}[case["op"]](case, s)
