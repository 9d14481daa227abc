"""Attention in 64 bits, with element-wise bounds on what a kernel may be off.

The bounds follow the arithmetic that the kernels document. u = 2^-24 is half a
step of fp32 relative to the value, h = 2^-8 that of bf16. A sum of n products in
fp32, in any order, is off by at most n u times the sum of the magnitudes
(first order; n + 2 below also covers the rounding of what enters it).
"""
from __future__ import annotations

import math

import torch

U, HB = 2.0 ** -24, 2.0 ** -8
LOG2E = math.log2(math.e)


def rounding(dtype):
    return torch.finfo(dtype).eps / 2


def scores(q, k, scale, seen):
    """S, its weights, and the bound on a weight's relative error. The score's
    dot product is off by (D + 2) u sum |q||k|; log2 e times it enters 2^x
    together with its rounding (2 u |S| log2 e, the constant's included), the
    maximum's likewise, and 2^x itself is good to 2 u."""
    S = (q @ k.T) * scale
    mag = (q.abs() @ k.abs().T) * scale
    dS = (q.shape[1] + 2) * U * mag + 2 * U * S.abs()
    S = S.masked_fill(~seen, -math.inf)
    none = ~seen.any(1, keepdim=True)
    W = torch.softmax(S.masked_fill(none, 0.0), 1).masked_fill(none, 0.0)
    big = torch.where(seen, dS, torch.zeros_like(dS)).amax(1, keepdim=True)
    top = torch.where(seen, S.abs(), torch.zeros_like(S)).amax(1, keepdim=True)
    return S, W, dS + 2 * big + 6 * U * top + 8 * U


def forward(q, k, v, scale, seen, out_dtype, p_bf16):
    """Output rows and the bound on them, one head."""
    _, W, eW = scores(q, k, scale, seen)
    n = k.shape[0]
    out = W @ v
    bound = (W * (eW + (2 * n + 4) * U + (HB if p_bf16 else 0.0))) @ v.abs()
    # The weights' sum is off like the weights themselves.
    bound = bound + (W * eW).sum(1, keepdim=True) * out.abs()
    return out, bound + rounding(out_dtype) * (out.abs() + bound) + 1e-30


def backward(q, k, v, scale, seen, out_bound, dout, bf16):
    """dq, dk, dv of one head and the bounds on them. P comes back from lse,
    which is off like a weight and its sum; bf16 rounds P and dS, and delta is taken from the rounded out."""
    S, W, eW = scores(q, k, scale, seen)
    n, D = k.shape
    h = HB if bf16 else 0.0
    out = W @ v
    lse = torch.logsumexp(S, 1, keepdim=True)
    lse = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))
    eP = 2 * eW + (n + 4) * U + 4 * U * lse.abs()
    dP, magP = dout @ v.T, dout.abs() @ v.abs().T
    delta = (dout * out).sum(1, keepdim=True)
    e_delta = (dout.abs() * (out_bound + (D + 2) * U * out.abs())).sum(1, keepdim=True)
    slope = dP - delta
    dS = W * slope
    e_dS = W * (eP * slope.abs() + (D + 2) * U * magP + e_delta + 2 * U * slope.abs())
    e_dS = e_dS + (h + U) * (dS.abs() + e_dS)
    rows = q.shape[0]
    dv = W.T @ dout
    e_dv = (W * (eP + h + (rows + 2) * U)).T @ dout.abs()
    dq = dS @ k * scale
    e_dq = (e_dS + (n + 3) * U * dS.abs()) @ k.abs() * scale
    dk = dS.T @ q * scale
    e_dk = (e_dS + (rows + 3) * U * dS.abs()).T @ q.abs() * scale
    return (dq, dk, dv), (e_dq, e_dk, e_dv)


def packed(q, k, v, starts, scale, causal, dout=None):
    """Whole tensors [rows, heads, D] (any dtype, any device): values and bounds in a dict."""
    dtype = q.dtype
    bf16 = dtype == torch.bfloat16
    q, k, v = q.double(), k.double(), v.double()
    H, KVH = q.shape[1], k.shape[1]
    G = H // KVH
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else [])
    val = {n: torch.zeros_like(k if n in ("dk", "dv") else q) for n in names}
    bnd = {n: torch.zeros_like(t) for n, t in val.items()}
    starts = [int(s) for s in starts]
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril()
        for h in range(H):
            g = h // G
            args = q[a:b, h].contiguous(), k[a:b, g].contiguous(), v[a:b, g].contiguous(), scale, seen
            o, eo = forward(*args, dtype, bf16)
            val["out"][a:b, h], bnd["out"][a:b, h] = o, eo
            if dout is None:
                continue
            d, e = backward(*args, eo, dout[a:b, h].double().contiguous(), bf16)
            for name, x, ex, at in zip(("dq", "dk", "dv"), d, e, (h, g, g)):
                val[name][a:b, at] += x
                # the sum over the group's heads runs on in the same accumulator
                bnd[name][a:b, at] += ex + (G - 1) * n * U * x.abs()
    for name in ("dq", "dk", "dv"):
        if name in val:
            bnd[name] = bnd[name] + rounding(dtype) * (val[name].abs() + bnd[name]) + 1e-30
    return val, bnd


def decode(q, kcache, vcache, pages, lens, scale, p_bf16):
    """[nseq, H, D] and the bound; positions of pages that do not exist are left out."""
    dtype, page = q.dtype, kcache.shape[2]
    H, KVH = q.shape[1], kcache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bnd = torch.zeros_like(out)
    for s, n in enumerate(lens):
        pos = torch.arange(min(max(int(n), 0), pages.shape[1] * page), device=q.device)
        ids = pages[s].long()[pos // page]
        there = (ids >= 0) & (ids < kcache.shape[0])
        ids, pos = ids[there], pos[there]
        if not len(pos):
            continue
        seen = torch.ones(1, len(pos), dtype=torch.bool, device=q.device)
        for h in range(H):
            k, v = (c[ids, h // (H // KVH), pos % page].double() for c in (kcache, vcache))
            o, e = forward(q[s, h:h + 1].double(), k, v, scale, seen, dtype, p_bf16)
            out[s, h], bnd[s, h] = o[0], e[0]
    return out, bnd


def assert_within(got, want, bound, what=""):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst "
                           f"{float(((got.double() - want).abs() / bound).nan_to_num(nan=math.inf).max()):.3g} times the bound")
