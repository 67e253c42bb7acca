"""The weights that cached keys receive, restated in 64 bits: what the kernels are compared with."""

from __future__ import annotations

import math

import torch


def received(case, chunk=0, window=0, temper=0.0, floor=1.0, sink=None, slopes=None, cap=0.0, add=None, width=None, rows=None):
    """(sums, how far a kernel's may be) in float64 on the CPU, [R, Hkv, width].  ``rows``: query rows of every request that count, the
    last ones of ``case.n`` (None: all).

    The bound of a weight w: relative, twice the scores' error (numerator and sum): 2 dh 2^-24 of the largest sum of |q k| for the order
    of dh products in 32 bits, and 2^-18 for the exponent's argument and the exponential; of the sum of a key's weights 2^-24 an
    addition; of `add` its half step."""
    G = case.Hq // case.Hkv
    R = len(case.n)
    width = width or max(a + b for a, b in zip(case.n, case.held))
    out, tol = torch.zeros((R, case.Hkv, width), dtype=torch.float64), torch.zeros((R, case.Hkv, width), dtype=torch.float64)
    q, positions, table = case.q.cpu().double(), case.positions.cpu().long(), case.table.cpu().long()
    sink = None if sink is None else sink.cpu().double()
    slopes = None if slopes is None else slopes.cpu().double()
    at = 0
    for r, (m, c) in enumerate(zip(case.n, case.held)):
        place = torch.arange(m + c)
        keys = case.rows[table[r][place // case.page], 0, :, place % case.page]  # [L, Hkv, dh]
        for i in range(m - min(m, m if rows is None else rows), m):
            p = int(positions[at + i])
            lo = max(p - p % chunk if chunk else 0, p - window + 1 if window else 0)
            seen = (place <= p) & (place >= lo)
            if not seen.any():
                continue
            temp = 1 + temper * math.log1p(math.floor((p + 1) / floor)) if temper else 1.0
            for h in range(case.Hq):
                k, x = keys[seen, h // G], q[at + i, h]
                s = k @ x * case.scale * temp
                size = float(torch.nan_to_num(k.abs() @ x.abs()).max()) * case.scale * temp
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s - slopes[h] * (p - place[seen]).double()
                    size += float(slopes[h]) * (p + 1)
                total = torch.logsumexp(s, 0) if sink is None else torch.logaddexp(torch.logsumexp(s, 0), sink[h])
                w = torch.exp(s - total)
                out[r, h // G, place[seen]] += w
                tol[r, h // G, place[seen]] += w * (2 * (2 * case.dh * 2.0 ** -24 * size + 2.0 ** -18) + (m * G + 2) * 2.0 ** -24)
        at += m
    if add is not None:
        out += add.cpu().double()
        tol += 2.0 ** -24 * out.abs()
    return out, tol
