"""Plain 64-bit forms of the sequence operators (after_amd.attention) for their tests, with the bounds of their rounding errors."""
import math

import torch

from oracle.denoiser import band_bounds

GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def bounds(n, keys, causal, window, chunk):
    """[first, last) per query; the queries are the newest n of `keys` tokens (band_bounds is the denoiser's own mask)."""
    if not causal:
        return [(0, keys)] * n
    out = []
    for p in range(keys - n, keys):
        lo, hi = band_bounds(p, chunk, window, keys)
        out.append((max(lo, 0), max(hi, 0)))
    return out


def attention(q, k, v, seen, scale):
    """q [n, H, D], k / v [m, KV, D] (any type, on any device), seen [n, m] bool -> (out, tolerance) in 64 bits, before the output's
    own rounding.  What is not seen has no part in it, NaN included."""
    n, H, D = q.shape
    m, KV, _ = k.shape
    G = H // KV
    q, k, v = (t.double().cpu() for t in (q, k, v))
    out, tol = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    probs = torch.zeros(n, H, m, dtype=torch.float64)
    for h in range(H):
        for i in range(n):
            at = seen[i].nonzero()[:, 0]
            if not len(at):
                continue
            kk, vv = k[at, h // G], v[at, h // G]
            p = torch.softmax(kk @ q[i, h] * scale, 0)
            probs[i, h, at] = p
            out[i, h] = p @ vv
            # scores: D products and sums in 32 bits; a score's error moves p by its double (its own and the sum's)
            d = (D + 4) * 2.0 ** -24 * scale * (kk.abs() @ q[i, h].abs()).max()
            tol[i, h] = (2 * d + (len(at) + 32) * 2.0 ** -24) * (p @ vv.abs())
    return out, tol, probs


def tolerance(out, tol, probs, v, dtype, p_half):
    """... with the rounding of the probabilities (p_half each, relative; fp16 keeps 2^-25 of the largest absolutely) and of the output."""
    G = out.shape[1] // v.shape[1]
    va = v.double().cpu().abs().nan_to_num(0, 0, 0).repeat_interleave(G, 1)  # [m, H, D]
    spread = torch.einsum("nhm,mhd->nhd", probs, va)
    least = (2.0 ** -25 * va.sum(0) if dtype == torch.float16 and p_half >= 2.0 ** -12 else 0)
    t = tol + p_half * spread + least
    return t + HALF[dtype] * (out.abs() + t) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)


def round4(x):
    """[..., D] -> (codes uint8 [..., D], scale bytes [..., D / 32]) by distance to the grid, ties to the even code."""
    x = x.double().cpu().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    byte = torch.full(top.shape, 255, dtype=torch.int64)
    fine = torch.isfinite(top)
    for b in range(252, 15, -1):  # the smallest power with which the largest is <= 6
        fits = top <= 6 * 2.0 ** (b - 127)
        byte = torch.where(fine & (fits | (b == 252)), b, byte)
    y = (x.abs() / 2.0 ** (byte.unsqueeze(-1) - 127.0)).nan_to_num(0, 6, 0).clamp(max=6)
    far = (y.unsqueeze(-1) - GRID).abs()
    far[..., 1::2] += 1e-13  # an odd code loses a tie
    code = far.argmin(-1) + 8 * torch.signbit(x)
    code = torch.where(fine.unsqueeze(-1), code, 0)
    return code.to(torch.uint8).flatten(-2), byte.to(torch.uint8)


def value4(code, byte):
    v = GRID[(code & 7).long()] * (1 - 2 * (code >> 3).double())
    p = torch.where(byte == 255, math.nan, 2.0 ** (byte.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * p.unsqueeze(-1)).flatten(-2)


def key_codes(keys):
    """The codes of a cache's `keys` buffer, [R, H, C, D]."""
    k = keys.cpu()
    return torch.stack([k & 15, k >> 4], -1).flatten(-2)


def value_codes(values):
    """... and of its `values` buffer (include/after_hip.h: after_kv4)."""
    v = values.cpu()
    R, H, B, D, _ = v.shape
    out = torch.empty(R, H, B * 8, D, dtype=torch.uint8)
    for s in range(8):
        for d in range(D):
            out[:, :, s::8, d] = v[:, :, :, (d // 2 % 16) * (D // 16) + d // 32 * 2 + d % 2, s // 2] >> 4 * (s % 2) & 15
    return out


def cache_values(c):
    """(keys, values) [R, H, C, D] of a KVCache4 in 64 bits."""
    return value4(key_codes(c.keys), c.key_scales.cpu()), value4(value_codes(c.values), c.value_scales.cpu())


def evict(weights, length, keep, recent):
    """The slots that stay, for one row and head."""
    if length <= keep:
        return list(range(length))
    old = length - recent
    w = [(-math.inf if math.isnan(x) else x, not math.isnan(x)) for x in weights[:old].tolist()]
    order = sorted(range(old), key=lambda i: (not w[i][1], -w[i][0], i))
    return sorted(order[:keep - recent] + list(range(old, length)))
