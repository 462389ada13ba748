"""64-bit references of the serving operators and the bounds their outputs are held to.

Bounds, for a sum of K products in 32 bits in any order: the error is at most (K + 2) 2^-24 times the sum of the
products' magnitudes (one rounding per product and addition).  fp32 products made of tf32 parts add 2^-20 of the
magnitudes (two operands of 22 bits, the product of the low parts dropped).  A bf16 output is off by at most half a step
of its value, 2^-8; a bf16 hidden activation carries 2^-8 of itself through |W2|.  An activation multiplies the error of
its argument by its largest slope (1.13 for GELU, 1.1 for SiLU) and adds a few roundings of its own value.
"""

import math

import torch

U = 2.0 ** -24        # half a step of fp32
PARTS = 2.0 ** -20    # fp32 products of tf32 parts
HALF = {torch.float32: torch.finfo(torch.float32).eps / 2, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}
SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}


def act64(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def product64(x, w, bias, act):
    """act(x w^T + bias) in 64 bits and a bound of a 32-bit evaluation's error, before the result's rounding."""
    x, w = x.double(), w.double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    err = ((x.shape[1] + 2) * U + PARTS) * mag
    if act == "swiglu":
        f = w.shape[0] // 2
        g, u, eg, eu = z[:, :f], z[:, f:], err[:, :f], err[:, f:]
        s = g * torch.sigmoid(g)
        return s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 16 * U * (s * u).abs()
    y = act64(z, act)
    return y, SLOPE[act] * err + 16 * U * (y.abs() + (z.abs() if act != "none" else 0))


def linear64(x, weight, bias=None, act="none", residual=None, out_dtype=None):
    """(value, bound) of linear()."""
    y, err = product64(x, weight, bias, act)
    if residual is not None:
        y = y + residual.double()
        err = err + U * (y.abs() + residual.double().abs())
    return y, err + HALF[out_dtype or x.dtype] * (y.abs() + err) + 1e-30


def route64(x, router_w, top_k, gate_mode, router_b=None, block_mask=None):
    """ids, gates and the smallest distance between a token's neighbouring logits around its choices."""
    logits = (x.double() @ router_w.double().t()).cpu()
    if router_b is not None:
        logits = logits + router_b.double().cpu()
    T, E = logits.shape
    mask = torch.zeros(T, E, dtype=torch.bool) if block_mask is None else block_mask.bool().cpu().expand(T, E)
    ids = torch.full((T, top_k), -1, dtype=torch.int32)
    gates = torch.zeros(T, top_k, dtype=torch.float64)
    gap = math.inf
    for t in range(T):
        l = logits[t].tolist()
        free = [e for e in range(E) if not mask[t, e] and l[e] != -math.inf]
        order = sorted(free, key=lambda e: (math.isnan(l[e]), 0.0 if math.isnan(l[e]) else -l[e], e))
        chosen = order[:top_k]
        for a, b in zip(order[:top_k], order[1:top_k + 1]):
            if l[a] != l[b]:
                gap = min(gap, abs(l[a] - l[b]))
        pool = order if gate_mode == "softmax" else chosen
        for j, e in enumerate(chosen):
            ids[t, j] = e
            if gate_mode == "none":
                gates[t, j] = 1.0
            elif any(math.isnan(l[o]) for o in pool):
                gates[t, j] = math.nan
            else:
                gates[t, j] = 1.0 / sum(math.exp(min(l[o] - l[e], 700.0)) for o in pool)
    return ids, gates, gap


def moe64(x, router_w, w1, w2, *, top_k, act, gate_mode, router_b=None, b1=None, b2=None, block_mask=None, residual=None,
          out_dtype=None):
    """(out, bound, ids, gates, gate bound, gap) of moe_few_tokens()."""
    ids, gates, gap = route64(x, router_w, top_k, gate_mode, router_b, block_mask)
    T, O = x.shape[0], w2.shape[1]
    out = torch.zeros(T, O, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    size = torch.zeros_like(out)
    # a gate's error: the logits' errors (absolute) go through a softmax, and a few roundings
    logit_err = ((x.shape[1] + 2) * U * (x.double().abs() @ router_w.double().abs().t())).max().item() if T else 0.0
    if router_b is not None:
        finite = router_b[router_b.abs() < 1e30].double().abs()  # a logit of the lowest value has a gate of 0 whatever its error
        logit_err += 2 * U * (finite.max().item() if finite.numel() else 0.0)
    gate_rel = 0.0 if gate_mode == "none" else 4 * logit_err + 64 * U
    for e in range(router_w.shape[0]):
        rows, slot = (ids == e).nonzero(as_tuple=True)
        if not len(rows):
            continue
        rows, slot = rows.to(x.device), slot.to(x.device)
        h, eh = product64(x[rows], w1[e], None if b1 is None else b1[e], act)
        eh = eh + HALF[x.dtype] * (h.abs() + eh)
        w = w2[e].double()
        y, mag = h @ w.t(), (h.abs() + eh) @ w.abs().t()
        ey = eh @ w.abs().t() + ((w.shape[1] + 2) * U + PARTS) * mag
        if b2 is not None:
            y, ey = y + b2[e].double(), ey + U * b2[e].double().abs()
        g = gates.to(x.device)[rows, slot][:, None]
        out[rows] += g * y
        err[rows] += g * (ey + (gate_rel + 4 * U) * (y.abs() + ey))
        size[rows] += g * (y.abs() + ey)
    if residual is not None:
        out = out + residual.double()
        size = size + residual.double().abs()
    err = err + (top_k + 2) * U * size
    return out, err + HALF[out_dtype or x.dtype] * (out.abs() + err) + 1e-30, ids, gates, gate_rel, gap


def check_close(got, want, bound):
    """Elementwise within the bound; NaN where the reference has it."""
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    off = (got - want).abs()[ok]
    far = off > bound[ok]
    assert not far.any(), f"{int(far.sum())} of {far.numel()} outside the bound, worst {float((off / bound[ok]).max()):.3g} x"


def check_norm(got, want, most):
    """2-norm of the difference over 2-norm of the reference.  Rounding errors of random sign grow with the square root
    of their number: in 32 bits far below the elementwise bounds, which could not tell fp32 products from tf32's."""
    rel = float((got.double() - want).norm() / want.norm())
    assert rel <= most, f"relative error {rel:.3g} over {most:.3g}"
