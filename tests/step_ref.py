"""The operators of a training step around its linears in 64 bits, with bounds for what 32 may lose, element by element.

u = 2^-24 is fp32's rounding. A sum of n terms that goes through a chain of k additions is off by at most k u times the sum of
the terms' magnitudes; CHAIN covers the kernels' rows: 32 elements of a lane, 4 + 2 steps over a wave, 16 waves, the
product before and the division behind it. What rounds to the rows' type adds half a step of it."""
from __future__ import annotations

import torch

U = 2.0 ** -24
CHAIN = 64
F64 = torch.float64


def half(dtype):
    return torch.finfo(dtype).eps / 2


def layer_norm(x, w, b, eps):
    """(y, mean, rstd, bound of y) from rows x as held, everything in 64 bits."""
    x, w = x.to(F64), w.to(F64)
    b = torch.zeros_like(w) if b is None else b.to(F64)
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    d = x - mean
    var = (d * d).sum(1, keepdim=True) / n
    rstd = 1 / torch.sqrt(var + eps)
    y = d * rstd * w + b
    dmean = CHAIN * U * x.abs().sum(1, keepdim=True) / n
    # mean((d + e)^2) = var + 2 e mean(d) + e^2, mean(d) = 0; 1 / sqrt halves a relative error.
    rel = (CHAIN + 8) * U + rstd * rstd * dmean * dmean
    err = w.abs() * (rstd * (dmean + U * d.abs()) + (d * rstd).abs() * (rel + 4 * U)) + 2 * U * (y.abs() + b.abs())
    return y, mean.view(-1), rstd.view(-1), err, (dmean.view(-1) + U * mean.abs().view(-1), rel.view(-1) * rstd.view(-1))


def layer_norm_bwd(x, mean, rstd, w, dy, dsum, chain):
    """(dx, dw, db, their bounds) from fp32 mean and rstd as given. chain: additions that a column's sum goes through."""
    x, mean, rstd, w, dy = x.to(F64), mean.to(F64)[:, None], rstd.to(F64)[:, None], w.to(F64), dy.to(F64)
    n = x.shape[1]
    xh, g = (x - mean) * rstd, dy * w
    s1, s2 = g.sum(1, keepdim=True) / n, (g * xh).sum(1, keepdim=True) / n
    dx = rstd * (g - s1 - xh * s2)
    e = 3 * U * xh.abs()
    d1 = (CHAIN + 1) * U * g.abs().sum(1, keepdim=True) / n
    d2 = (CHAIN + 1) * U * (g * xh).abs().sum(1, keepdim=True) / n + (g.abs() * e).sum(1, keepdim=True) / n
    err = rstd * (4 * U * (g.abs() + s1.abs() + (xh * s2).abs()) + d1 + xh.abs() * d2 + e * s2.abs())
    if dsum is not None:
        dx = dx + dsum.to(F64)
        err = err + 2 * U * (dx.abs() + dsum.to(F64).abs())
    ew = chain * U * (dy * xh).abs().sum(0) + (dy.abs() * e).sum(0)
    return dx, (dy * xh).sum(0), dy.sum(0), err + U * dx.abs(), ew, chain * U * dy.abs().sum(0)


def cross_entropy(z, targets, scale, row_scale=None):
    """(loss, lse, dz, their bounds). The power of two of a rounded product: e^(z - m) is off by 3 |z - m| u for
    the difference and the product, and 4 u for the constant and the instruction."""
    z = z.to(F64)
    m = z.max(1, keepdim=True).values
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    away = torch.where(p > 0, (z - m).abs(), torch.zeros_like(z))
    wrong = p * (3 * away + 4) * U
    rel = wrong.sum(1, keepdim=True) / total + 2 * CHAIN * U      # up to 128 elements of a lane
    lse = (torch.log(total) + m).view(-1)
    held = targets >= 0
    at = targets.long().clamp(min=0)
    row = torch.arange(z.shape[0], device=z.device)
    zt = z[row, at]
    loss = torch.where(held, lse - zt, torch.zeros_like(lse))
    k = torch.full_like(lse, scale) if row_scale is None else scale * row_scale.to(F64)
    q = p / total
    hot = torch.zeros_like(z)
    hot[row, at] = 1
    dz = torch.where(held[:, None], (q - hot) * k[:, None], torch.zeros_like(z))
    dlse = 4 * U + 4 * U * lse.abs() + rel.view(-1)
    ddz = k.abs()[:, None] * (wrong / total + q * (rel + 4 * U) + 2 * U * hot) + 2 * U * dz.abs()
    return loss, lse, dz, dlse + 2 * U * (zt.abs() + loss.abs()), dlse, torch.where(held[:, None], ddz, torch.zeros_like(z))


def embed_bwd(tokens, dy, V, scale):
    """(sums [V, C], bound): a chain of a token's rows, 64 at a time, then the product and the sum with what was there."""
    dy = dy.to(F64)
    met = (tokens >= 0) & (tokens < V)
    ids = tokens[met].long()
    zeros = torch.zeros(V, dy.shape[1], dtype=F64, device=dy.device)
    sums = zeros.index_add(0, ids, dy[met]) * scale
    most = zeros.index_add(0, ids, dy[met].abs()) * abs(scale)
    count = torch.bincount(ids, minlength=V).to(F64)[:, None]
    return sums, (torch.minimum(count, 64 + count / 64) + 3) * U * most


# ---- moments in 8 bits, with numpy's fp32 (each operation rounded) and borders in 64 bits ---------

LEAST = 2.0 ** -120


def decode_m(c, scale):
    import numpy as np
    c = c.astype(np.float32).reshape(-1, 256)
    return (c * np.abs(c) * scale[:, None]).reshape(-1)


def decode_v(c, scale):
    import numpy as np
    c = c.astype(np.float32).reshape(-1, 256)
    root = c * c * scale[:, None]
    return (root * root).reshape(-1)


def encode(x, second):
    """Codes and scales of fp32 moments (a multiple of 256 of them), by the nearest root, ties up."""
    import numpy as np
    x = x.reshape(-1, 256)
    top = np.abs(x).max(1)
    most, power = (255, 4) if second else (127, 2)
    border = ((np.arange(most) + 0.5) / most) ** power
    c = np.zeros(x.shape, np.int64)
    for i, t in enumerate(top):
        if t >= LEAST and np.isfinite(t):
            c[i] = np.searchsorted(border, np.abs(x[i]).astype(np.float64) / np.float64(t), side="right")
            if second:
                c[i] = np.where((x[i] > 0) & (c[i] == 0), 1, c[i])
            else:
                c[i] = np.where(x[i] < 0, -c[i], c[i])
    f = np.float32
    with np.errstate(invalid="ignore"):
        scale = np.sqrt(top) * (f(1) / f(65025)) if second else top * (f(1) / f(16129))
    scale = np.where(np.isfinite(top), np.where(top >= LEAST, scale, f(0)), f("nan")).astype(f)
    return c.reshape(-1), scale


def adam(w, g, m, v, factor, lr, b1, b2, eps, wd, inv1, inv2):
    """dgm_adam in numpy's fp32."""
    import numpy as np
    f = np.float32
    lr, b1, b2, eps, wd, inv1, inv2 = (f(t) for t in (lr, b1, b2, eps, wd, inv1, inv2))
    g = g * f(factor)
    m = b1 * m + (f(1) - b1) * g
    v = b2 * v + (f(1) - b2) * g * g
    w = w - lr * ((m * inv1) / (np.sqrt(v * inv2) + eps) + wd * w)
    return w, m, v
