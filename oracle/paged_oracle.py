"""Oracle of the paged 8-bit key/value cache in 64 bits: plain loops over sequences and tokens, test infrastructure only."""
from __future__ import annotations

import math

import torch


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (fp64) rounded to e4m3 values, half to even, saturating at 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.nan_to_num(torch.round(x / step) * step, nan=math.nan).clamp(-448.0, 448.0)


def scale_of(largest: float) -> float:
    """Smallest power of two s with largest <= 448 s, within 2^-100 .. 2^119."""
    if not largest > 0.0:
        return 2.0 ** -100
    s = 2.0 ** min(max(math.ceil(math.log2(largest / 448.0)), -100), 119)
    while s < 2.0 ** 119 and largest > 448.0 * s:  # the logarithm is rounded
        s *= 2.0
    while s > 2.0 ** -100 and largest <= 224.0 * s:
        s /= 2.0
    return s


def rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [heads, D] by one position's tables [D / 2], in the dtype given (fp32 gives the products' and sums' own roundings)."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def spans(starts, T, lens):
    """(first row, rows) of every sequence; ``starts`` None: as many for each."""
    B = len(lens)
    if starts is None:
        return [(b * (T // B), T // B) for b in range(B)]
    return [(int(starts[b]), int(starts[b + 1]) - int(starts[b])) for b in range(B)]


class Cache:
    """Values of the pages as [page, head, place, D] (fp64), scales as [page, head]."""

    def __init__(self, pages):
        heads_first = pages.layout == "bhsd"
        self.codes = [(t if heads_first else t.transpose(1, 2)).cpu().to(torch.float32).double().clone() for t in (pages.k, pages.v)]
        self.scales = [t.cpu().double().clone() for t in (pages.k_scale, pages.v_scale)]

    def append(self, k, v, table, lens, starts=None, rope=None):
        """The values before their rounding of what was written: {(page, head, place): (key, value)} (fp64)."""
        size = self.codes[0].shape[2]
        wrote = {}
        for b, (row, n) in enumerate(spans(starts, k.shape[0], lens)):
            first = int(lens[b]) - n
            new = {}
            for i in range(n):
                pos = first + i
                if pos < 0 or (rope is not None and pos >= rope[0].shape[0]) or pos >= table.shape[1] * size:
                    continue
                x = k[row + i].float().cpu()
                if rope is not None:
                    x = rotated(x, rope[0][pos].cpu(), rope[1][pos].cpu())
                new.setdefault(pos // size, []).append((pos % size, x.double(), v[row + i].cpu().double()))
            for block, tokens in new.items():
                page = int(table[b, block])
                if not 0 <= page < self.codes[0].shape[0]:
                    continue
                for h in range(k.shape[1]):
                    fine = [bool(torch.isfinite(x[h]).all() and torch.isfinite(y[h]).all()) for _, x, y in tokens]
                    for which in (0, 1):
                        codes, scales = self.codes[which], self.scales[which]
                        largest = max([float(t[1 + which][h].abs().max()) for t, ok in zip(tokens, fine) if ok], default=0.0)
                        earlier, old = tokens[0][0], float(scales[page, h])
                        s = max(scale_of(largest), old if earlier else 0.0)
                        if earlier and s > old:
                            codes[page, h, :earlier] = e4m3(codes[page, h, :earlier] * (old / s))
                        for t, ok in zip(tokens, fine):
                            value = t[1 + which][h] / s
                            codes[page, h, t[0]] = e4m3(value) if ok else (math.nan if which == 0 else 0.0)
                        scales[page, h] = s
                    for t, ok in zip(tokens, fine):
                        wrote[page, h, t[0]] = (t[1][h], t[2][h], ok)
        return wrote

    def dense(self, which, table_row, length, h):
        size = self.codes[0].shape[2]
        out = torch.full((length, self.codes[0].shape[3]), math.nan, dtype=torch.float64)
        seen = torch.zeros(length, dtype=torch.bool)
        for block in range(-(-length // size)):
            page = int(table_row[block])
            if 0 <= page < self.codes[0].shape[0]:
                end = min(size, length - block * size)
                out[block * size:block * size + end] = self.codes[which][page, h, :end] * self.scales[which][page, h]
                seen[block * size:block * size + end] = True
        return out, seen


def attend(q, cache, table, lens, starts=None, causal=True, scale=None):
    """(O, LSE, and three error scales: sum p |v| / sum p, keys x twice the largest |v| / sum exp(s - max), the scores' own) in fp64."""
    T, Hq, D = q.shape
    Hkv, size = cache.codes[0].shape[1], cache.codes[0].shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    mean, spread = torch.zeros_like(out), torch.zeros_like(out)
    score_tol = torch.zeros_like(lse)
    q = q.cpu().double()
    for b, (row, n) in enumerate(spans(starts, T, lens)):
        length = min(max(int(lens[b]), 0), table.shape[1] * size)
        if n <= 0:
            continue
        for h in range(Hkv):
            k, seen = cache.dense(0, table[b], length, h)
            v, _ = cache.dense(1, table[b], length, h)
            v_ref = v[seen].abs().max() if seen.any() else 0.0
            pos = torch.arange(length - n, length)
            visible = seen[None, :].expand(n, -1) & ((torch.arange(length)[None, :] <= pos[:, None]) | (not causal))
            for hq in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                rows = q[row:row + n, hq]
                s = torch.where(visible, rows @ torch.where(seen[:, None], k, 0.0).T * scale, -math.inf)
                top = s.amax(-1, keepdim=True) if length else torch.full((n, 1), -math.inf, dtype=torch.float64)
                top = torch.where(top == -math.inf, 0.0, top)
                p = torch.exp(s - top)
                total = p.sum(-1, keepdim=True)
                safe = torch.where(total == 0, 1.0, total)
                vz = torch.where(seen[:, None], v, 0.0)
                out[row:row + n, hq] = torch.where(visible.any(-1)[:, None], (p @ vz) / safe, 0.0)
                lse[row:row + n, hq] = (top + torch.log(total))[:, 0]
                mean[row:row + n, hq] = (p @ vz.abs()) / safe
                spread[row:row + n, hq] = visible.double().sum(-1)[:, None] * v_ref * 2 / safe
                if seen.any():
                    kabs = torch.where(seen[:, None], k, 0.0).abs()
                    score_tol[row:row + n, hq] = scale * (rows.abs() @ kabs.T).amax(-1) * D * 2.0 ** -23  # D sums in fp32, cut off or rounded
    return out, lse, mean, spread, score_tol
