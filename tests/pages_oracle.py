"""The exact paged cache in plain 64-bit torch on the CPU: what tests/test_gpu_pages.py compares with."""

import math

import torch


def rows(table, n, page):
    """Row of each of the first n slots of a sequence in the planes' flattened (block, token) dimension."""
    t = torch.arange(n)
    return table[t // page].long() * page + t % page


def gather(plane, table, n, page):
    return plane.flatten(0, 1)[rows(table, n, page)].double()


def attention(q, k, v, scale=None, last=None, there=None):
    """q (R, H, G, D), k / v (n, H, D) doubles; row r sees slots up to last[r] whose page exists -> out (R, H, G, D) and the
    weights (R, H, G, n); rows that see nothing are zero."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    n = k.shape[0]
    if n == 0:
        return torch.zeros_like(q), q.new_zeros(*q.shape[:3], 0)
    s = torch.einsum("rhgd,nhd->rhgn", q, torch.nan_to_num(k, nan=0.0) if there is not None else k) * scale
    seen = torch.ones(q.shape[0], n, dtype=torch.bool) if last is None else torch.arange(n)[None] <= last[:, None]
    if there is not None:
        seen = seen & there[None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    return torch.einsum("rhgn,nhd->rhgd", p, torch.nan_to_num(v, nan=0.0) if there is not None else v), p


def order_key(x):
    """Descending order of masses: NaN above everything."""
    return (0, 0.0) if math.isnan(x) else (1, -x)


def evict(mass, positions, held, seen, n, budget, recent):
    """One (sequence, kv head): mass (n,), positions (n,) as lists -> source slot of every slot that is left, and its position."""
    pos = [positions[t] if t < held else seen + t - held for t in range(n)]
    m = min(n, budget)
    if n <= budget:
        return list(range(n)), pos
    late = seen + n - held - recent
    kept = set(sorted(range(n), key=lambda t: (pos[t] < late, *order_key(mass[t]), t))[:m])
    movers = iter(sorted(t for t in kept if t >= m))
    source = [t if t in kept else next(movers) for t in range(m)]
    return source, [pos[t] for t in source]
