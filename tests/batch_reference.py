"""Plain implementations of a batch's steps around the products: page tables
step by step in Python, adapters and sampling in 64 bits."""
from __future__ import annotations

import math

import torch


def step(tables, lens, free, page, tokens, new=None, keep=None):
    """PageTables.step on lists, the stack `free` of the pages that count; returns (q_starts, taken, slots,
    positions, seq) and changes its arguments."""
    row = len(tables[0]) if tables else 0
    cap = row * page
    back = []
    for b, table in enumerate(tables):
        lens[b] = max(0, min(lens[b], cap))
        held = -(-lens[b] // page)
        if keep is not None and 0 <= keep[b] <= lens[b]:
            lens[b] = keep[b]
        for j in range(-(-lens[b] // page), held):
            back.append(table[j])
            table[j] = -1
    free += back[::-1]
    starts, taken, slots, positions, seq = [0], [], [], [], []
    asked, out_of_pages = 0, False
    for b, table in enumerate(tables):
        n = max(0, new[b]) if new is not None else 0
        asked += n
        fits = asked <= tokens and lens[b] + n <= cap
        have = -(-lens[b] // page)
        want = -(-(lens[b] + n) // page) if fits else have
        if want > have:
            out_of_pages = out_of_pages or want - have > len(free)
            fits = not out_of_pages
        if fits:
            for j in range(have, want):
                table[j] = free.pop()
        for i in range(min(n, tokens - len(slots))):
            p = lens[b] + i
            at = table[p // page] if fits else -1
            slots.append(at * page + p % page if at >= 0 else -1)
            positions.append(p if fits else -1)
            seq.append(b)
        starts.append(len(slots))
        taken.append(n if fits else 0)
        lens[b] += taken[-1]
    rest = [-1] * (tokens - len(slots))
    return starts, taken, slots + rest, positions + rest, seq + rest


def adapters(y, x, ids, a, b, scales):
    """y + scales[i] (x a[i]^T) b[i]^T row by row in 64 bits, and a bound on what 32-bit sums may be off."""
    out, bound = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    k, rank = x.shape[1], a.shape[1]
    half = 2.0 ** -24
    for i in ids.unique().tolist():
        if not 0 <= i < a.shape[0]:
            continue
        rows = torch.nonzero(ids == i)[:, 0]
        xr, ai, bi = x[rows].double(), a[i].double(), b[i].double()
        s = float(scales[i]) if scales is not None else 1.0
        mid, mags = xr @ ai.T, xr.abs() @ ai.abs().T
        out[rows] += s * (mid @ bi.T)
        # a sum of n terms in f32, in any order: n half steps of the sum of their sizes
        off = (k + 40) * half * mags
        bound[rows] = abs(s) * ((off + (rank + 4) * half * (mid.abs() + off)) @ bi.abs().T)
    return out, bound + half * (out.abs() + bound)


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The weights (64 bits) of one row's logits that its settings leave, 0 for the others; None for a row
    without a token."""
    x = torch.where(x.isnan(), -math.inf, x.double())
    top = x.max()
    if top == -math.inf:
        return None
    w = torch.zeros_like(x)
    if not temperature > 0.0:
        w[int(torch.nonzero(x == top)[0])] = 1.0
        return w
    if top == math.inf:
        w[x == top] = 1.0
    else:
        w = torch.where(x == -math.inf, 0.0, torch.exp((x - top) / temperature))
    order = torch.sort(x, descending=True, stable=True).indices
    ws = w[order]
    if 0 < top_k < len(x):
        ws[top_k:] = 0.0
    if top_p < 1.0:
        before = ws.cumsum(0) - ws
        stay = before < max(top_p, 0.0) * ws.sum()
        stay[0] = True
        ws = torch.where(stay, ws, 0.0)
    if min_p > 0.0:
        ws = torch.where(ws >= min(min_p, 1.0), ws, 0.0)
    return torch.zeros_like(w).scatter_(0, order, ws)


def token(w, u):
    """The token of a row of weights for the number u, and its chance."""
    if w is None:
        return -1, 0.0
    u = 0.0 if math.isnan(u) else min(max(u, 0.0), 1.0)
    sums = w.cumsum(0)
    hits = torch.nonzero((sums > u * sums[-1]) & (w > 0))
    i = int(hits[0]) if len(hits) else int(torch.nonzero(w > 0)[-1])
    return i, float(w[i] / sums[-1])
