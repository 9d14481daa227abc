"""One step of AdamW with moments in 8 bits in numpy's fp32: the nearest codes, two of them moved by one where rounding would hold
what they stand for."""
from __future__ import annotations

import numpy as np

import step_ref as ref

F = np.float32


def zeros(blocks):
    """(codes and scales of m, codes and scales of v) of nothing yet."""
    return (np.zeros(256 * blocks, np.int64), np.zeros(blocks, F)) * 2


def values(state):
    """What the codes stand for; a v of a code above 0 is above 0."""
    cm, sm, cv, rv = state
    v = ref.decode_v(cv, rv)
    return ref.decode_m(cm, sm), np.where((v == 0) & (cv > 0) & np.repeat(rv > 0, 256), F(2.0 ** -149), v).astype(F)


def follow(state, m, v, b1, b2):
    """Codes and scales of m and v (fp32), whose codes and scales were `state` a step ago, and where they are not the nearest ones."""
    cm0, sm0, cv0, rv0 = state
    m0, v0 = values(state)
    with np.errstate(all="ignore"):
        (cm, sm), (cv, rv) = ref.encode(m, False), ref.encode(v, True)
        up = (cv == cv0) & (cv < 255) & np.repeat(rv <= rv0, 256) & np.repeat(rv > 0, 256)
        up &= v > max(F(9) - F(8) * F(b2), F(1)) * v0
        cv = cv + up
        c = np.abs(cm)
        held = (c > 0) & (cm == cm0) & np.repeat((sm >= sm0) & (sm <= F(1.125) * sm0), 256) & (np.abs(m) < np.abs(m0))
        held &= (c.astype(F) * (F(1) - F(b1)) < F(1)) & (cv.astype(F) * (F(1) - F(b2)) < F(4))
        cm = cm - np.sign(cm) * held
    return (cm, sm, cv, rv), (held, up)


def step(w, g, state, factor=1.0, *, lr, b1, b2, eps, wd, inv1, inv2):
    """(w, state, (where m's code is not the nearest, where v's))."""
    m, v = values(state)
    g = g * F(factor)
    with np.errstate(all="ignore"):
        w, m, v = ref.adam(w, g, m, v, 1.0, lr, b1, b2, eps, wd, inv1, inv2)
    return (w, *follow(state, m, v, b1, b2))
