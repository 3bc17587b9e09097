"""Plain 64-bit implementations of the several-sequence operators
(include/rdl_attention.h), and the rounding bounds their tests use."""
import math

import torch

STEP32 = 2.0 ** -24  # half a step of f32 rounding, relative


def plan(cached, new, free, page, tables, m):
    """(tables, row_start, kv_len, row_seq, positions, slots, summary) as lists, one sequence after the other."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    start, kv_len, flags, taken, wanted = [0], [], 0, 0, 0
    seqs, poss, slots = [], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        if c < 0 or n < 0:
            flags |= 1
        c, n = max(c, 0), max(n, 0)
        if c + n > 2**31 - 1:
            flags |= 1
            n = 2**31 - 1 - c
        have, upto = -(-c // page), -(-(c + n) // page)
        if upto > width:
            flags |= 2
        for p in range(min(have, width), min(upto, width)):
            tables[b][p] = free[wanted] if wanted < len(free) else -1
            wanted += 1
        for i in range(min(n, max(0, m - start[-1]))):
            p = (c + i) // page
            pg = tables[b][p] if p < width else -1
            seqs.append(b)
            poss.append(c + i)
            slots.append(pg * page + (c + i) % page if pg >= 0 else -1)
        start.append(start[-1] + n)
        kv_len.append(c + n)
    taken = min(wanted, len(free))
    flags |= (4 if wanted > len(free) else 0) | (8 if start[-1] > m else 0)
    pad = m - len(seqs)
    return (tables, start, kv_len, seqs + [-1] * pad, poss + [0] * pad, slots + [-1] * pad,
            [start[-1], taken, flags, max(kv_len, default=0)])


def rope(x, cos, sin):
    """x [rows, heads, hd], cos / sin [rows, hd / 2]; also what rounding in 32 bits can move each value by."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h].double(), x[..., h:].double(), cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, a * s + b * c], -1)
    # two products and a sum, each rounded once
    most = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
    return y, 2 * STEP32 * most


def attention(q, k, v, first, scale):
    """q [rows, heads, hd]; k, v [keys, kv heads, hd] (64 bits); row i sees the
    keys 0 .. first + i.  Returns (out, bound): the exact outputs and how far
    a 32-bit evaluation from products of 22-bit parts may be from them.

    bound: a score is a sum of hd products, whose parts are off by at most
    2^-21 together (two of 22 bits) and whose f32 sum by (hd + 4) steps: off by
    e <= scale * sum|q k| * (2^-21 + (hd + 4) 2^-23), beside which the running
    maximum's subtraction and the exponent's own rounding move a weight by at
    most (|s - max| + 4) 2^-23.  Weights off by a factor 1 + w move the quotient by 2 w
    sum p|v|, the f32 sums over n keys and the 22 bits of weights and values by
    (n + 16) 2^-23 sum p|v| more."""
    rows, heads, hd = q.shape
    keys, kvh = k.shape[:2]
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if keys == 0 or rows == 0:
        return out, bound
    g = heads // kvh
    j = torch.arange(keys, device=q.device)
    sees = j <= (first + torch.arange(rows, device=q.device))[:, None]
    some = sees.any(1)
    for h in range(heads):
        qh, kh, vh = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        kh = torch.where(torch.isfinite(kh), kh, 0.0)
        clean = torch.where(torch.isfinite(vh), vh, 0.0)
        s = (qh @ kh.T.contiguous()) * scale
        mag = (qh.abs() @ kh.abs().T.contiguous()) * scale
        s = torch.where(sees, s, -math.inf)
        top = torch.where(some, s.amax(1), 0.0)[:, None]
        e = torch.where(sees, (s - top).exp(), 0.0)
        p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
        out[:, h] = p @ clean
        w = (torch.where(sees, mag, 0.0).amax(1) * (2.0**-21 + (hd + 4) * 2.0**-23) +
             (torch.where(sees, top - s, 0.0).clamp(max=104).amax(1) + 4) * 2.0**-23)
        n = sees.sum(1)
        bound[:, h] = (p @ clean.abs()) * (2 * w + (n + 16) * 2.0**-23)[:, None]
        if not torch.isfinite(vh).all():  # what a row sees
            wide = torch.where(torch.isfinite(vh), 0.0, vh)
            for r in range(rows):
                out[r, h] += wide[sees[r]].sum(0)
    return out, bound


def gather(pool, table, n, page):
    """Positions 0 .. n - 1 of a sequence from a pool viewed as [pages, kv heads, positions, hd]."""
    ids = table[: -(-n // page)].long()
    return pool[ids].permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:n]
