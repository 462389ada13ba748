"""64-bit references of the attention operators and the bounds their outputs are held to.

A logit is a sum of D products in 32 bits: off by at most (D + 2) 2^-24 of its products' magnitudes, fp32 products made of
two parts 2^-20 more, and a few roundings of itself.  An error dz of every logit changes a softmax weight by a factor of at
most exp(2 dz); rounding weights to f16 or bf16 by 1 + 2^-11 or 1 + 2^-8.  The output, a weighted mean, moves by that factor
of the mean of |v|, by the roundings of its n additions, and by its own rounding.
"""

import math

import torch

from serving_reference import HALF, PARTS, U

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 16


def attention64(q, k, v, visible, scale=None, weight_half=0.0, out_dtype=None):
    """One sequence: q [n, Hq, D], k and v [m, Hk, D], the first visible[i] keys for row i.  (out, lse, out's bound, lse's, [largest logit])."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    qd, kd, vd = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
    err, lse_err, largest = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros(1, dtype=torch.float64, device=q.device)
    seen = torch.arange(len(k), device=q.device)[None, :] < visible[:, None]
    if len(k):
        for h in range(hq):
            z = (qd[:, h] @ kd[:, h].t()) * scale
            size = (qd[:, h].abs() @ kd[:, h].abs().t()) * abs(scale)
            dz = torch.where(seen, ((d + 2) * U + PARTS) * size + 6 * U * z.abs(), 0).amax(1)   # of a row, at most
            if n:
                largest = torch.maximum(largest, torch.where(seen, z, 0).abs().amax().nan_to_num(0, 0, 0)[None])
            z = torch.where(seen, z, -math.inf)
            top = z.amax(1)
            some = top > -math.inf
            p = torch.where(seen, torch.exp(z - torch.where(some, top, 0)[:, None]), 0)
            l = p.sum(1)
            lse[:, h] = torch.where(some, top + l.log(), -math.inf)
            p = p / torch.where(some, l, 1)[:, None]
            # what a row does not see does not enter, infinities and NaN included
            odd = ~vd[:, h].isfinite()
            plain = torch.where(odd, 0, vd[:, h])
            out[:, h] = p @ plain
            mean = p @ plain.abs()
            if odd.any():
                for i in range(n):
                    for j, c in odd[:int(visible[i])].nonzero().tolist():
                        out[i, h, c] = out[i, h, c] + vd[j, h, c]
            m = visible.clamp_max(len(k)).double()
            rel = 2 * dz + weight_half + (m + 64) * U + 2.0 ** -22 * (m / 16).ceil()
            err[:, h] = rel[:, None] * mean + 2.0 ** -24 * (m / len(k))[:, None] * plain.abs().amax(0)
            lse_err[:, h] = 2 * dz + (m + 64) * U + 4 * U * lse[:, h].abs().nan_to_num(0, 0, 0)
    dt = out_dtype or q.dtype
    return out, lse, err + HALF[dt] * (out.abs().nan_to_num(0, 0, 0) + err) + 1e-30, lse_err + 1e-30, largest


def norm_bound(out_dtype, bf16_weights, largest):
    """For check_norm.  fp32: 3e-6 of sums in random signs, and what a logit's own last place (its sum is cut, not rounded: up
    to 2 U of it, and the scale's rounding as much) makes of its weight.  bf16: the result's rounding, 2^-9 to 2^-8 of a value
    evenly spread (root mean square 0.0017), and weights rounded to bf16 as much again on their own."""
    z = 4 * U * float(largest.max()) if largest.numel() else 0.0
    return z + (3e-6 if out_dtype == torch.float32 else 0.004 if bf16_weights else 0.003)


def quantise64(x, unit=1.0):
    """What the cache holds for x [..., D], from the definition: (code's value, scale), both 64-bit, by nearest of all numbers."""
    x = x.double().unflatten(-1, (-1, GROUP)) / unit
    dev = x.device
    bytes_ = torch.arange(0, 127, dtype=torch.uint8, device=dev)
    e4m3 = bytes_.view(torch.float8_e4m3fn).double()          # 0 .. 448, ascending
    scale = _nearest(x.abs().amax(-1) / 6, e4m3)
    q = x.abs() / torch.where(scale > 0, scale, 1)[..., None]
    code = torch.where(scale[..., None] > 0, _nearest(q, torch.tensor(GRID, dtype=torch.float64, device=dev)), 0)
    bad = x.isnan().any(-1)
    return (torch.sign(x) * code * torch.where(bad, math.nan, scale)[..., None] * unit).flatten(-2)


def _nearest(x, grid):
    """The grid's number nearest to x, of two the one with the even index; x NaN gives 0."""
    x = x.nan_to_num(0.0, posinf=1e300)
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, len(grid) - 1)
    lo = hi - 1
    up, down = grid[hi] - x, x - grid[lo]
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    return torch.where(take_hi, grid[hi], grid[lo])


def cache64(cache, slots):
    """Keys and values that the cache's bytes stand for, [N, heads, D] in 64 bits; slots below zero give zeros."""
    outs = []
    at = slots.clamp_min(0).long()
    page, row = at // cache.page_size, at % cache.page_size
    grid = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device=slots.device)
    for codes, scales, unit in ((cache.k_codes, cache.k_scales, cache.k_unit), (cache.v_codes, cache.v_scales, cache.v_unit)):
        c = codes[page, :, row]
        s = scales.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).double()
        x = grid[torch.stack((c & 15, c >> 4), -1).flatten(-2).long()].unflatten(-1, (-1, GROUP)) * s[..., None] * unit
        outs.append(torch.where((slots >= 0)[:, None, None], x.flatten(-2), 0.0))
    return outs


def slots_of(table, lengths, page_size):
    """Slots of the first lengths[b] tokens of every sequence, one list for each."""
    out = []
    for row, n in zip(table.tolist(), lengths):
        out.append(torch.tensor([row[i // page_size] * page_size + i % page_size for i in range(n)], dtype=torch.int64))
    return out
