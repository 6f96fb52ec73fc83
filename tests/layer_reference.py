"""Plain 64-bit forms that the tests of the cache and the attention share."""
import numpy as np
import torch


def cache_values(kv):
    """Every slot's keys and values [slots, heads, hd] of a KvCache, in 64 bits."""
    kc, ks, vc, vs = (t.double() for t in kv.planes)
    k = kc.unflatten(3, (-1, 32)) * ks[..., None]
    v = vc.unflatten(2, (-1, 32)) * vs[:, :, :, None, :]
    return k.flatten(3).transpose(1, 2).flatten(0, 1), v.flatten(2, 3).permute(0, 3, 1, 2).flatten(0, 1)


def attend64(kv, q, q_starts, kv_lens, tables, scale, window=0, sinks=None, max_kv=None):
    """(outputs, allowed error) of the attention, in 64 bits, rows of no
    sequence NaN.

    The allowed error, with u = 2^-11 (half an f16 step): q and each key round
    once to f16 (2 u of sum |q k|, and half an f16 subnormal step, 2^-25, where
    they are tiny) and the score's f32 sum adds hd + 8 steps of 2^-24, so a score is off by at most
    delta, the weights and their sum by a factor exp(2 delta); a weight
    exp(s - m) rounds to f16 (u, or 2^-25 below 2^-14), a value to f16 (u).
    f32 sums over n positions add n / 64 + 64 steps of 2^-24 (a matrix product of
    64, then one addition a tile). The output's own rounding comes on top."""
    u = 2.0**-11
    keys, vals = cache_values(kv)
    tokens, heads, hd = q.shape
    group = heads // kv.kv_heads
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    starts, lens, tab = q_starts.tolist(), kv_lens.tolist(), tables.cpu()
    for b, n in enumerate(lens):
        new = starts[b + 1] - starts[b]
        rows = slice(starts[b], starts[b + 1])
        n_all = n
        if max_kv is not None:
            n = min(n, max_kv)
        if new == 0:
            continue
        j = torch.arange(n)
        pages = tab[b].long()[j // kv.page] if n else torch.zeros(0, dtype=torch.long)
        there = ((pages >= 0) & (pages < kv.pages)).to(q.device)
        slots = (pages.clamp(0, kv.pages - 1) * kv.page + j % kv.page).to(q.device)
        j = j.to(q.device)
        pos = (n - new + torch.arange(new, device=q.device))[:, None]
        seen = (j <= pos) & there
        if window:
            seen &= j > pos - window
        for h in range(heads):
            k, v, x = keys[slots, h // group], vals[slots, h // group], q[rows, h].double()
            s = (x @ k.T * scale).masked_fill(~seen, float("-inf"))
            size = x.abs() @ k.abs().T * abs(scale)
            delta = ((2 * u + (hd + 8) * 2.0**-24) * size + 2.0**-24 * (x.abs().sum(1, keepdim=True) * abs(scale) + k.abs().sum(1)))
            delta = delta.masked_fill(~seen, 0.0).amax(1, keepdim=True) if n else torch.zeros(new, 1, device=q.device, dtype=torch.float64)
            top = s.amax(1, keepdim=True) if n else torch.full((new, 1), float("-inf"), device=q.device, dtype=torch.float64)
            if sinks is not None:
                top = torch.maximum(top, sinks[h].double())
            p = torch.where(seen, torch.exp(s - top), 0.0)
            total = p.sum(1, keepdim=True)
            some = total > 0
            if sinks is not None:
                total = total + torch.exp(sinks[h].double() - top)
            total = torch.where(some, total, 1.0)
            out[rows, h] = torch.where(some, p @ v / total, 0.0)
            rel = torch.expm1(2 * delta) + 2 * u * (1 + u) + (n / 64 + 64) * 2.0**-24
            tol[rows, h] = rel * (p @ v.abs()) / total + 2.0**-25 * (seen.double() @ v.abs()) / total
    return out, tol


def rounding(t):
    return torch.finfo(t).eps / 2


def wire_blocks(x):
    """Codes [.., hd] and scales [.., hd / 32] of the Q8_0 wire blocks of f32 values, from the CPU oracle."""
    from oracle import qref
    b = qref.wire_encode(np.ascontiguousarray(x, dtype=np.float32).ravel()).reshape(-1, 34)
    return b[:, 2:].copy().view(np.int8).reshape(x.shape), b[:, :2].copy().view(np.float16).reshape(*x.shape[:-1], -1)
