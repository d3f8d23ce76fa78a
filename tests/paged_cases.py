"""Inputs and 64-bit references for the operators of batched serving (paged cache, attention over it)."""
import torch

BF16_STEP = 2.0 ** -8  # half a step of bf16, relative: torch.finfo(torch.bfloat16).eps / 2


class Batch:
    """A paged cache with the sequences of a call: `new` rows each, `lens` tokens each (the new ones counted).  Slots that hold
    no token of a sequence, and pages that nobody has, are NaN.  order: 'hsd' ([page, head, slot, dim] in memory) or 'shd'."""

    def __init__(self, new, lens, Hq, Hk, D, page, seed=0, order="hsd", extra_rows=0, spare_width=2, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.new, self.lens, self.Hq, self.Hk, self.D, self.page = list(new), list(lens), Hq, Hk, D, page
        B, need = len(lens), [-(-max(n, 0) // page) for n in lens]
        n_pages = sum(need) + 3
        ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(1, max(need) + spare_width)
        table = torch.full((B, width), -1, dtype=torch.int32)
        shape = (n_pages, Hk, page, D) if order == "hsd" else (n_pages, page, Hk, D)
        nan = lambda: torch.full(shape, float("nan"), dtype=torch.bfloat16, device=device)
        self.cache_k, self.cache_v = nan(), nan()
        if order == "shd":
            self.cache_k, self.cache_v = self.cache_k.transpose(1, 2), self.cache_v.transpose(1, 2)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
            for i in range(n):
                used = min(page, lens[b] - i * page)
                for c in (self.cache_k, self.cache_v):
                    c[int(table[b, i]), :, :used] = torch.randn(Hk, used, D, device=device, generator=g).to(torch.bfloat16)
        self.table = table.to(device)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.starts = [sum(new[:b]) for b in range(B + 1)]
        self.cu = torch.tensor(self.starts, dtype=torch.int32, device=device)
        self.T = sum(new) + extra_rows
        self.q = (1.5 * torch.randn(self.T, Hq * D, device=device, generator=g)).to(torch.bfloat16)
        self.heads = (Hq, Hk, D)

    def sequence(self, table, n):
        """Keys and values 0 .. n - 1 of a table's pages, [Hk, n, D] in 64 bits, and which of them are there."""
        j = torch.arange(n, device=table.device)
        col = j // self.page
        page = torch.where(col < table.numel(), table.long()[col.clamp(max=table.numel() - 1)], -1)
        there = (page >= 0) & (page < self.cache_k.shape[0])
        rows = lambda c: c[page.clamp(0, self.cache_k.shape[0] - 1), :, j % self.page].transpose(0, 1).double()
        return rows(self.cache_k), rows(self.cache_v), there


def attention_64(q, k, v, seen, scale):
    """q [n, Hq, D], k, v [Hk, L, D], seen [n, L]: the result, and what bounds its rounding: the same average of |v|, and the
    largest sum of |q| |k| scale of a visible pair."""
    n, Hq, D = q.shape
    rep = Hq // k.shape[0]
    k, v = (torch.where(seen.any(0)[None, :, None], x, 0.0) for x in (k, v))  # nobody's keys may hold anything
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    most = 0.0
    some = seen.any(1)
    for h in range(Hq):
        s = (q[:, h] @ k[h // rep].T) * scale
        s = torch.where(seen, s, -torch.inf)
        p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
        p = torch.where(some[:, None], p / p.sum(-1, keepdim=True), 0.0)
        out[:, h], size[:, h] = p @ v[h // rep], p @ v[h // rep].abs()
        if some.any():
            most = max(most, float(torch.where(seen, q[:, h].abs() @ k[h // rep].abs().T * scale, 0.0).max()))
    return out, size, most


def tolerance(ref, size, most, D):
    """What separates a result from the 64-bit one: its rounding to bf16 (half a step of |ref|); each weight rounded to bf16 for
    the second product (half a step of the average of |v|); the scores, D + 2 roundings to 32 bits of sums no larger than `most`,
    in the weight and in the denominator; and the exponential with its argument (2^-24 of up to 2^6 and 2^-22, both twice: 2^-16)."""
    slack = 2 * (D + 2) * 2.0 ** -24 * most + 2.0 ** -16
    return BF16_STEP * ref.abs() + (BF16_STEP + slack) * (1 + BF16_STEP) * size + 1e-30


def visible(n, length, L, window, sinks, device):
    pos = torch.arange(length - n, length, device=device)[:, None]
    j = torch.arange(L, device=device)[None]
    seen = j <= pos
    if window:
        seen = seen & ((j > pos - window) | (j < sinks))
    return seen


def paged_reference(b: Batch, window=0, sinks=0, scale=None, cu=True):
    scale = b.D ** -0.5 if scale is None else scale
    q = b.q.double().view(b.T, b.Hq, b.D)
    ref, tol = torch.zeros_like(q), torch.zeros_like(q)
    for i, (n, length) in enumerate(zip(b.new, b.lens)):
        if n == 0:
            continue
        L = max(length, 1)
        k, v, there = b.sequence(b.table[i], L)
        seen = visible(n, length, L, window, sinks, q.device) & there[None]
        rows = slice(b.starts[i], b.starts[i] + n)
        ref[rows], size, most = attention_64(q[rows], k, v, seen, scale)
        tol[rows] = tolerance(ref[rows], size, most, b.D)
    return ref.view(b.T, -1), tol.view(b.T, -1)


def check(got, ref, tol):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol)[bad].max()), bad.nonzero()[0].tolist())
