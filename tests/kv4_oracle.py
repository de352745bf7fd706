"""64-bit statements of the cache's rounding, of attention over it and of the beam selection, without the package's code."""
import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E4M3 = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64)


def nearest_even(x, grid):
    """x >= 0 to the nearest of the ascending grid, ties to the entry with the even index, saturating."""
    grid = grid.to(x.device)
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    a, b = x - grid[hi - 1], grid[hi] - x
    return grid[torch.where((b < a) | ((a == b) & (hi % 2 == 0)), hi, hi - 1)]


def rounded64(x, unit):
    """What finite x [..., head] stands for once it has been in the cache."""
    b = x.double().unflatten(-1, (-1, 16))
    s = nearest_even(b.abs().amax(-1, keepdim=True) / 6.0 / unit, E4M3) * unit
    y = nearest_even(b.abs() / torch.where(s > 0, s, torch.ones_like(s)), LEVELS) * s
    return torch.where(b < 0, -y, y).flatten(-2)


class Dense:
    """Keys and values that a cache of one layer stands for, dense per slot, float64."""

    def __init__(self, S, H, T, hd, unit=2.0 ** -4, device="cpu"):
        self.k, self.v = (torch.zeros(S, T, H, hd, dtype=torch.float64, device=device) for _ in range(2))
        self.unit, self.T = unit, T

    def append(self, k, v, start, counts):
        bad = ~(torch.isfinite(k.double()).all(-1, keepdim=True) & torch.isfinite(v.double()).all(-1, keepdim=True))
        for d, x in ((self.k, k), (self.v, v)):
            y = torch.where(bad, torch.full_like(x, float("nan")).double(), rounded64(x.nan_to_num(0.0, 0.0, 0.0), self.unit))
            for s, (a, n) in enumerate(zip(start, counts)):
                n = min(n, self.T - a)
                d[s, a:a + n] = y[s, :n]

    def reorder(self, src):
        self.k, self.v = self.k[src].clone(), self.v[src].clone()


def attention64(q, dense, lens, counts, scale=None):
    """(out, sum_j p_j |v_j|) [S, n, heads, head] in float64; rows behind the counts are zeros."""
    S, n, heads, hd = q.shape
    group = heads // dense.k.shape[2]
    out, mag = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for s in range(S):
        L, c = min(lens[s], dense.T), counts[s]
        k, v = (x[s, :L].repeat_interleave(group, 1) for x in (dense.k, dense.v))
        w = torch.einsum("chd,lhd->hcl", q[s, :c].double(), k) * (1 / math.sqrt(hd) if scale is None else scale)
        see = L - c + 1 + torch.arange(c, device=q.device)
        w = w.masked_fill(torch.arange(L, device=q.device) >= see.view(-1, 1), float("-inf"))
        p = torch.softmax(w, -1)
        p = torch.where((see <= 0).view(1, -1, 1), torch.zeros_like(p), p)
        visible_nan = torch.isnan(p).any(-1)
        o = torch.einsum("hcl,lhd->chd", p.nan_to_num(0.0), v.nan_to_num(0.0))
        out[s, :c] = torch.where(visible_nan.t().unsqueeze(-1), torch.full_like(o, float("nan")), o)
        mag[s, :c] = torch.einsum("hcl,lhd->chd", p.nan_to_num(0.0), v.nan_to_num(0.0).abs())
    return out, mag


def select64(logits, scores, V, finished=None, eos=-1):
    B, K = scores.shape
    x = logits[:, :V].double().view(B, K, V)
    base = scores.double().unsqueeze(-1)
    lse = torch.logsumexp(x, -1, keepdim=True)
    alive = torch.isfinite(base) & torch.isfinite(lse)
    c = torch.where(alive, base + (x - lse), torch.full_like(x, float("-inf")))
    if finished is not None:
        for b, k in finished.nonzero().tolist():
            c[b, k] = float("-inf")
            if math.isfinite(float(scores[b, k])):
                c[b, k, eos] = float(scores[b, k])
    best, at = torch.sort(c.view(B, -1), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    fin = at % V == eos
    if finished is not None:
        fin = fin | finished.gather(1, at // V)
    return best, at % V, at // V, fin
