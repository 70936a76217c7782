"""The operators between token ids and logits in 64 bits, on the host, from their definitions, and how far a kernel's results may be off.

A result that is rounded once to a type is off by half a step of that type, relative to it (bf16 2^-8, fp16 2^-11, fp32 2^-24), and by the error
of its fp32 arithmetic in front of that: 2^-24 of the magnitudes for every operation along the longest chain of them. Results of fp16 below its normal
range are off by half of its smallest number, 2^-25."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(got, ref, arithmetic, what=""):
    """|got - ref| <= half a step of got's type at ref + `arithmetic` (absolute, of ref's shape or a number). A rounding to the next
    value counts from the value before it, so half a step is taken of the larger of the two."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    g = got.detach().double().cpu()
    ref = ref.cpu()
    arithmetic = arithmetic.cpu() if torch.is_tensor(arithmetic) else torch.tensor(float(arithmetic), dtype=torch.float64)
    special = ~torch.isfinite(ref)
    same = (g == ref) | (torch.isnan(g) & torch.isnan(ref))
    assert bool(same[special].all()), what
    limit = half_step(got.dtype) * (ref.abs() + arithmetic) + arithmetic + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = (g - ref).abs()
    bad = ~special & ~(off <= limit)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off - limit)[bad].max())} over, at {bad.nonzero()[0].tolist()}"


# ---- embedding ---------------------------------------------------------------------------------------------------------
def embedding_sum(lookups):
    """lookups: (ids, weight, scale). Returns the sum and the sum of magnitudes."""
    y = sum(w.detach().double().cpu()[i.cpu().long()] * s for i, w, s in lookups)
    size = sum((w.detach().double().cpu()[i.cpu().long()] * s).abs() for i, w, s in lookups)
    return y, size


def table_grad(ids, dy, rows, scale, skip=None):
    """The gradient, the sum of magnitudes and the number of tokens of every row."""
    i = ids.cpu().reshape(-1).long()
    d = dy.detach().double().cpu().reshape(-1, dy.shape[-1])
    ok = (i >= 0) & (i < rows)
    if skip is not None:
        ok &= i != skip
    i, d = i[ok], d[ok]
    g = torch.zeros(rows, dy.shape[-1], dtype=torch.float64).index_add_(0, i, d) * scale
    size = torch.zeros(rows, dy.shape[-1], dtype=torch.float64).index_add_(0, i, d.abs()) * abs(scale)
    return g, size, torch.bincount(i, minlength=rows)[:, None].double()


# ---- log probabilities -------------------------------------------------------------------------------------------------
class Scores:
    """Everything that token_logprobs gives for logits [n, width] and targets [n], with its gradient, in 64 bits."""

    def __init__(self, logits, targets, vocab, top_k=0, temperature=1.0, ignore=-100):
        x = logits.detach().double().cpu()
        self.x, self.t, self.v, self.k, self.temp, self.ignore = x[:, :vocab], targets.cpu().long(), vocab, top_k, temperature, ignore
        z = self.x / temperature
        m = z.max(dim=1, keepdim=True).values
        self.none = m == -float("inf")
        m0 = torch.where(self.none, torch.zeros_like(m), m)
        e = (z - m0).exp()
        s = e.sum(dim=1, keepdim=True)
        self.lp = z - m0 - s.log()
        self.lp = torch.where(self.none, torch.full_like(self.lp, -float("inf")), self.lp)
        self.p = torch.where(self.none, torch.zeros_like(e), e / s)
        plp = torch.where(self.p == 0, torch.zeros_like(self.p), self.p * torch.where(self.p == 0, torch.zeros_like(self.p), self.lp))
        self.h = -plp.sum(dim=1)
        self.width = logits.shape[1]
        self.kept = self.t != ignore
        at = torch.where(self.kept, self.t, torch.zeros_like(self.t))
        self.picked = torch.where(self.kept, self.lp.gather(1, at[:, None])[:, 0], torch.zeros_like(self.h))
        # how far fp32 may be off: see `arithmetic`
        zz = torch.where(torch.isfinite(z), z - m0, torch.zeros_like(z)).abs()
        self.mean_z = (self.p * zz).sum(dim=1)
        if top_k:
            self.ids = torch.sort(self.x, dim=1, descending=True, stable=True).indices[:, :top_k]
            self.top = self.lp.gather(1, self.ids)
            self.top_ids = torch.where(self.x.gather(1, self.ids) == -float("inf"), -1, self.ids)

    def arithmetic(self, size):
        """fp32: the sum of 2^u has at most vocab / 512 + 64 additions in a row, terms with 2^-22 of the exponential and 3 roundings of u; the
        logarithm, the difference and the products in front add a rounding each of their magnitudes."""
        return U * (self.v / 512 + 64 + 16) * (1.0 + size)

    def of_lp(self, lp):
        return self.arithmetic(torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp)) + (self.mean_z if lp.dim() == 1 else self.mean_z[:, None]))

    def of_h(self):
        return self.arithmetic(self.h.abs() + 2 * self.mean_z)

    def grad(self, g=None, gh=None, gk=None):
        """The gradient with respect to the logits [n, width], and how far fp32 may be off."""
        n = self.x.shape[0]
        up = torch.zeros_like(self.x)
        rows = torch.arange(n)
        live = self.kept & ~self.none[:, 0]
        if g is not None:
            up[rows[live], self.t[live]] += g.double().cpu()[live]
        if gk is not None:
            w = torch.where(self.top_ids >= 0, gk.double().cpu(), torch.zeros_like(self.top))
            up.scatter_add_(1, self.ids, w)
        total = up.sum(dim=1, keepdim=True)
        d = up - self.p * total
        lp0 = torch.where(self.p == 0, torch.zeros_like(self.p), self.lp)
        size = up.abs() + self.p * (up.abs().sum(dim=1, keepdim=True)) * (1 + lp0.abs())
        if gh is not None:
            gh = gh.double().cpu()[:, None]
            d = d - gh * self.p * (lp0 + self.h[:, None])
            size = size + gh.abs() * self.p * (lp0.abs() + self.h[:, None] + 1) * (1 + lp0.abs())
        out = torch.zeros(n, self.width, dtype=torch.float64)
        off = torch.zeros_like(out)
        out[:, :self.v] = torch.where(self.none, torch.zeros_like(d), d) / self.temp
        off[:, :self.v] = U * (self.v / 512 + 64 + 16) * size / self.temp + 1e-37
        return out, off


# ---- dropout -----------------------------------------------------------------------------------------------------------
def philox_bits(seed, step, call, n, first=0):
    """16 bits an element from Philox4x32-10, in Python's whole numbers, of n elements from group `first` of eight on."""
    low = 0xFFFFFFFF
    out = []
    for group in range(first, first + (n + 7) // 8):
        c = [group & low, group >> 32, call & low, step & low]
        k0, k1 = seed & low, (seed >> 32) & low
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k0, b & low, (a >> 32) ^ c[3] ^ k1, a & low]
            k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
        for w in c:
            out += [w & 0xFFFF, w >> 16]
    return torch.tensor(out[:n])
