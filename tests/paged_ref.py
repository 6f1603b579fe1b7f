"""Plain 64-bit restatements of the paged-cache operators, and the error that
a kernel of a given element type may show against them."""

import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def page_tables(table, ctx, new, free, page, T):
    """The step's tables, request by request and token by token."""
    table = np.array(table)
    R, W = table.shape
    slots, positions = np.full(T, -1), np.full(T, -1)
    start, seq, used, t = [0], [], 0, 0
    for r in range(R):
        c, n = max(int(ctx[r]), 0), max(int(new[r]), 0)
        have = min(-(-c // page), W)
        for j in range(have, min(-(-(c + n) // page), W)):
            table[r, j] = free[used] if used < len(free) else -1
            used += 1
        for i in range(n):
            pos = c + i
            if t < T:
                positions[t] = pos
                if pos // page < W and table[r, pos // page] >= 0:
                    slots[t] = table[r, pos // page] * page + pos % page
            t += 1
        start.append(t)
        seq.append(c + n)
    return table, slots, positions, start, seq, used


def rows(q, k, v, n, window, first, scale, sinks, seen=None):
    """Attention of the last L of n rows in float64: q (L, H, D), k (n, Hkv,
    D), v (n, Hkv, V) CPU tensors; `seen` (n,) hides rows. Returns (out (L, H,
    V), tolerance of the same shape)."""
    dtype, (L, H, D), V = q.dtype, q.shape, v.shape[2]
    Hkv = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    pos = torch.arange(n - L, n)[:, None]
    key = torch.arange(n)[None]
    see = key <= pos
    if window:
        see = see & ((key > pos - window) | (key < first))
    if seen is not None:
        see = see & seen[None]
    out = torch.zeros(L, H, V, dtype=torch.float64)
    tol = torch.zeros(L, H, V, dtype=torch.float64)
    if n == 0:
        return out, tol
    u, f32 = UNIT[dtype], 2.0 ** -24
    for h in range(H):
        kh, vh = k[:, h * Hkv // H], v[:, h * Hkv // H]
        # A row hidden from all may hold anything.
        kh = torch.where(see.any(0)[:, None], kh, 0.0)
        vh = torch.where(see.any(0)[:, None], vh, 0.0)
        s = q[:, h] @ kh.T * scale
        mag = (q[:, h].abs() @ kh.abs().T * abs(scale)).masked_fill(~see, 0).amax(1)
        s = s.masked_fill(~see, -float("inf"))
        top = s.amax(1)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        e = torch.exp(s - top[:, None])
        den = e.sum(1)
        if sinks is not None:
            den = den + torch.exp(sinks[h].double() - top)
        w = torch.where(den[:, None] > 0, e / den.clamp(min=1e-300)[:, None], 0.0)
        out[:, h] = w @ vh
        # A score is off by its fp32 sum (D roundings of at most `mag`), the
        # scaling and the subtraction of the base (3 of at most mag) and exp2
        # (2); a weight's numerator and denominator by that each. The sums over
        # n keys cost n roundings each, numerator and denominator; the weights
        # are rounded once to the type (f16: below 2^-14 by 2^-25 against a
        # denominator of at least 2^-4), the result once more. The rounded
        # weights p (1 + e), |e| <= u, stand in numerator and denominator alike:
        # sum p (1 + e) v / sum p (1 + e) is off by sum w e (v - out) / (1 + e'),
        # at most u (sum w |v| + |out|) to first order, so |out| counts u once
        # for this and once for the result's own rounding.
        delta = (D + 5) * f32 * mag + 2 * f32
        part = u + 2 * delta + 2 * n * f32
        tol[:, h] = 2.02 * u * out[:, h].abs() + 1.01 * part[:, None] * (w @ vh.abs()) + 1e-30
        if dtype == torch.float16:
            big = torch.where(see.any(0)[:, None], vh.abs(), 0.0).amax()
            tol[:, h] += n * 2.0 ** -21 * big + 2.0 ** -25  # the result's own half step
    return out, tol


class Cache:
    """Requests of given lengths in a paged cache with shuffled pages, on the
    GPU, and their contiguous keys and values on the CPU."""

    def __init__(self, seq, Hkv, D, V, page, dtype, seed, device, order="phtd", spare=3, width=None,
                 fill=0.0, kv=None):
        g = torch.Generator().manual_seed(seed)
        self.seq, self.page = list(seq), page
        need = [-(-n // page) for n in seq]
        W = max(need + [1]) if width is None else width
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(seq), W), -1, dtype=torch.int32)
        kc = torch.full((pages, page, Hkv, D), fill, dtype=dtype)
        vc = torch.full((pages, page, Hkv, V), fill, dtype=dtype)
        self.k, self.v = [], []
        at = 0
        for r, n in enumerate(seq):
            table[r, :need[r]] = perm[at:at + need[r]]
            at += need[r]
            if kv is None:
                k = torch.randn(n, Hkv, D, generator=g).to(dtype)
                v = torch.randn(n, Hkv, V, generator=g).to(dtype)
            else:
                k, v = kv[r]
            self.k.append(k)
            self.v.append(v)
            i = torch.arange(n)
            p = table[r][i // page].long()
            kc[p, i % page], vc[p, i % page] = k, v
        if order == "phtd":
            kc, vc = kc.transpose(1, 2).contiguous(), vc.transpose(1, 2).contiguous()
            self.kc, self.vc = kc.to(device), vc.to(device)
        else:
            self.kc, self.vc = kc.to(device).transpose(1, 2), vc.to(device).transpose(1, 2)
        self.table = table.to(device)
        self.lens = torch.tensor(list(seq), dtype=torch.int32, device=device)


def starts(new, device):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=device)
