"""Rotary positions and attention over a paged cache in 64 bits, and how far an fp32 computation with 16-bit weights may be off."""
import math

import torch


def rotate(x, positions, freq, scale=1.0, interleaved=False):
    """(x (tokens, heads, dim) rotated, the bound of its rounding in fp32): freq in radians per position, 64 bits."""
    pairs = freq.numel()
    x = x.double().cpu()
    y, mag = x.clone(), torch.zeros_like(x)
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        t = positions.double().cpu() * float(freq[i])
        c, s = (torch.cos(t) * scale)[:, None], (torch.sin(t) * scale)[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        # sine and cosine off by 2^-22 (their argument 2^-24 of at most pi, the function 2 ulp), the scale, two products and a sum
        mag[..., a] = mag[..., b] = abs(scale) * (x[..., a].abs() + x[..., b].abs()) * 2.0 ** -21
    return y, mag


def attend(query, keys, values, pages, lengths, offsets, scale=None, causal=True, window=0):
    """(out (tokens, heads, dim), bound): rows of no sequence are NaN in `out`.  All on the host; a page outside the cache is zeros."""
    query, keys, values = query.double().cpu(), keys.cpu(), values.cpu()
    tokens, heads, dim = query.shape
    size, kv = keys.shape[1:3]
    scale = dim ** -0.5 if scale is None else scale
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[keys.dtype]
    out, bound = torch.full_like(query, math.nan), torch.zeros_like(query)
    for i, n in enumerate(int(v) for v in lengths):
        n = max(0, min(n, pages.shape[1] * size))
        first, last = int(offsets[i]), int(offsets[i + 1])
        ids = [int(p) for p in pages[i, :-(-n // size)]] if n else []
        zero = torch.zeros(size, kv, dim, dtype=keys.dtype)
        pick = lambda c: torch.cat([c[p] if 0 <= p < c.shape[0] else zero for p in ids])[:n].double() if n else torch.zeros(0, kv, dim).double()
        k, v = pick(keys), pick(values)
        for r in range(first, last):
            at = n - (last - first) + (r - first)
            hi = min(n, max(0, at + 1)) if causal else n
            lo = min(hi, max(0, at + 1 - window)) if window else 0
            if hi <= lo:
                out[r] = 0
                continue
            for h in range(heads):
                kk, vv = k[lo:hi, h // (heads // kv)], v[lo:hi, h // (heads // kv)]
                z = kk @ query[r, h] * scale
                p = torch.softmax(z, 0)
                out[r, h] = p @ vv
                reach = p @ vv.abs()
                # fp32 scores: dim products and sums, 2^-23 each where the tensor cores cut off; in a weight's exponent and in their sum
                off = float((kk.abs() @ query[r, h].abs()).max()) * scale * (dim + 4) * 2.0 ** -23 if hi > lo else 0.0
                bound[r, h] = u * reach + u * out[r, h].abs() + (2 * off + (hi - lo) * 2.0 ** -22 + 2.0 ** -19) * reach
    return out, bound
