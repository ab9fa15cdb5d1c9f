"""Plain attention in 64 bits, the tolerances of its comparison, and paged caches for the tests."""
import numpy as np
import torch

# half a step relative to the value: 2^-24, 2^-11, 2^-8
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def attend(q, keys, values, scale):
    """One sequence in 64 bits: q [n][heads][hd], keys and values [m][kv][hd]; row i sees keys 0..m-n+i.

    Returns the outputs and, per row and head, a bound of the error that f32 arithmetic in any order of
    summation can make: every score is off by at most (hd + 8) 2^-24 sum|q k| scale, which with the sums of
    m terms (m 2^-24), the exponential (its argument rounded below 2^6 in size, two roundings of its own)
    moves each weight by a relative e, and a quotient of weighted sums by 2 e max|v|.
    """
    q, keys, values = (x.detach().cpu().double() for x in (q, keys, values))
    n, heads, hd = q.shape
    m, group = keys.shape[0], heads // keys.shape[1]
    out, tol = torch.zeros(n, heads, hd, dtype=torch.float64), torch.zeros(n, heads, 1, dtype=torch.float64)
    for i in range(n):
        seen = m - n + i + 1
        if seen <= 0:
            continue
        for h in range(heads):
            k, v = keys[:seen, h // group], values[:seen, h // group]
            s = k @ q[i, h] * scale
            w = torch.exp(s - s.max())
            out[i, h] = w @ v / w.sum()
            off = (hd + 8) * (k.abs() @ q[i, h].abs()).max() * abs(scale)
            tol[i, h] = 2 * 2.0**-24 * (off + seen + 80) * v.abs().max()
    return out, tol


def close(got, want, tol, where=""):
    """got is want within tol and one rounding to got's type (a subnormal's half step in 16 bits)."""
    tiny = {torch.float16: 2.0**-25, torch.bfloat16: 0.0, torch.float32: 0.0}[got.dtype]
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= tol + HALF_STEP[got.dtype] * (want.abs() + tol) + tiny)
    assert not bad.any(), (where, int(bad.sum()), off[bad].max().item(), bad.nonzero()[:4].tolist())


def weights_rounded(tol, values, dtype):
    """Room for weights rounded to a 16-bit type before they meet the values: 2 half steps of max|v|."""
    return tol if dtype == torch.float32 else tol + 2 * HALF_STEP[dtype] * values.detach().abs().max().cpu().double()


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


class Pages:
    """A shuffled paged cache of sequences of the given lengths, its free places filled with NaN.

    order: the order in memory of (page, position, head), of the pools' view [page][position][head][hd]."""

    def __init__(self, lens, page, kv, hd, dtype, seed, order=(0, 1, 2), spare=2, width=1, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        self.page, self.lens = page, list(lens)
        sizes = (total, page, kv)
        back = [order.index(i) for i in range(3)]
        self.k, self.v = (torch.full([sizes[i] for i in order] + [hd], float("nan"), dtype=dtype, device=device).permute(*back, 3) for _ in range(2))
        perm = torch.randperm(total, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(need + [0]) + width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = perm[at:at + n]
            at += n
        self.table_host, self.table = table, table.to(device)

    def place(self, s, p):
        return int(self.table_host[s, p // self.page]), p % self.page

    def fill(self, s, keys, values, first=0):
        """Writes positions first.. of sequence s."""
        p = torch.arange(first, first + keys.shape[0])
        pg, at = self.table_host[s, (p // self.page).long()].long().to(self.k.device), (p % self.page).to(self.k.device)
        self.k[pg, at] = keys.to(self.k)
        self.v[pg, at] = values.to(self.v)

    def read(self, s, n):
        p = torch.arange(n)
        pg, at = self.table_host[s, (p // self.page).long()].long().to(self.k.device), (p % self.page).to(self.k.device)
        return self.k[pg, at], self.v[pg, at]


def ints(x, device="cuda"):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)
