"""Plain 64-bit forms of the attention operators, written from their definitions, for the tests."""
import math

import torch


def round_bits(s, bits):
    """fp64 to `bits` significant bits, ties to even."""
    m, e = torch.frexp(s)
    return torch.ldexp(torch.round(m * 2.0 ** bits), e - bits)


def quantised(x):
    """What the cache holds of x [..., D], in fp64: s = rn5(amax / 7) in [2^-60, 2^60], s * clamp(rint(x / s), -7, 7)."""
    g = x.double().unflatten(-1, (-1, 64))
    amax = g.abs().amax(-1, keepdim=True)
    s = round_bits(amax / 7, 5).clamp(2.0 ** -60, 2.0 ** 60)
    y = s * torch.round(g / s).clamp(-7, 7)
    return torch.where(torch.isfinite(g).all(-1, keepdim=True), y, math.nan).flatten(-2)


def norm_rope(x, w, table, positions, eps, interleaved, unit):
    y = x.double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (w.double() + (1 if unit else 0))
    R = table.shape[1]
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        c, s = table[positions.long(), i].double()[:, None], table[positions.long(), R // 2 + i].double()[:, None]
        y0, y1 = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = y0 * c - y1 * s, y1 * c + y0 * s
    return y


def attention(q, keys, values, starts, window, scale):
    """q [T, H, D]; keys, values: one [len, K, D] for each request. Output, log-sum-exp, and sum of p |v|, in fp64."""
    T, H, D = q.shape
    out, size = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    for b, (k, v) in enumerate(zip(keys, values)):
        n, rows = len(k), slice(starts[b], starts[b + 1])
        place = n - starts[b + 1] + torch.arange(starts[b], starts[b + 1], device=q.device)
        if not len(place) or not n:
            continue
        j = torch.arange(n, device=q.device)
        seen = j <= place[:, None]
        if window:
            seen &= j > place[:, None] - window
        for h in range(H):
            kk, vv = (x[:, h * x.shape[1] // H].double() for x in (k, v))
            s = (q[rows, h].double() @ kk.t() * scale).masked_fill(~seen, -math.inf)
            lse[rows, h] = torch.logsumexp(s, -1)
            p = torch.where(seen, torch.softmax(s, -1), 0.0)
            # a value that is not a number reaches only the rows that see it
            bad = torch.isnan(vv)
            for o, x in ((out, vv), (size, vv.abs())):
                o[rows, h] = p @ x.masked_fill(bad, 0.0) + torch.where(seen.double() @ bad.double() > 0, math.nan, 0.0)
    return out, lse, size


def plan(cached, new, table, free, taken, page, tokens):
    """Lists and lists of lists of whole numbers; the table is changed in place."""
    start, pos, slot, req = [0], [], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(-(-c // page), -(-(c + n) // page)):
            table[b][j] = free[taken]
            taken += 1
        for p in range(c, c + n):
            pos.append(p)
            slot.append(table[b][p // page] * page + p % page)
            req.append(b)
        start.append(start[-1] + n)
    pad = tokens - len(pos)
    return start, [c + n for c, n in zip(cached, new)], pos + [0] * pad, slot + [-1] * pad, req + [-1] * pad, taken
