"""Training with 8-bit moments against 32-bit ones, by the coding's numpy form: weights that lose their gradients
come to rest, steps stay of AdamW's size where gradients are small beside their block's, and others move as they do in 32 bits."""
from __future__ import annotations

import numpy as np
import pytest

import adam8_ref as a8
import step_ref as ref

LR = 1e-3
BLOCKS = 4
HALF = np.tile(np.arange(256) < 128, BLOCKS)      # of each block, the elements that the gradients below make different


def train(gradient, steps, b1, b2, mark):
    """What weights moved by from step `mark` on, in units of the learning rate: (in 8 bits, in 32)."""
    n = 256 * BLOCKS
    w8, w32 = np.zeros(n, a8.F), np.zeros(n, a8.F)
    m, v, state = np.zeros(n, a8.F), np.zeros(n, a8.F), a8.zeros(BLOCKS)
    rng = np.random.default_rng(1)
    for t in range(steps):
        g = gradient(rng, t).astype(a8.F)
        hyper = dict(lr=LR, b1=b1, b2=b2, eps=1e-8, wd=0.0, inv1=1 / (1 - b1 ** (t + 1)), inv2=1 / (1 - b2 ** (t + 1)))
        w8, state, _ = a8.step(w8, g, state, **hyper)
        w32, m, v = ref.adam(w32, g, m, v, 1.0, *hyper.values())
        if t + 1 == mark:
            from8, from32 = w8.copy(), w32.copy()
    return (w8 - from8) / LR, (w32 - from32) / LR


def gradients(part):
    """Random ones of size 1, and in HALF part(rng, t) times those."""
    def g(rng, t):
        x = rng.standard_normal(256 * BLOCKS)
        return np.where(HALF, part(rng, t) * x, x)
    return g


@pytest.mark.parametrize("b1,b2", [(0.9, 0.95), (0.9, 0.999), (0.9, 0.9)])
def test_weights_without_gradients_come_to_rest(b1, b2):
    """From step 100 on HALF has none. A code from 10 on is within half a code, 1 / c of its moment, so that the steps that a moment still makes
    as it decays are AdamW's within a factor of 2; smaller codes go one down a step, 9 + 8 + ... squared are 2% of the block's largest, less than a step.
    Held moments would make some hundreds."""
    eight, wide = train(gradients(lambda rng, t: float(t < 100)), 1100, b1, b2, 100)
    assert (np.abs(eight[HALF]) <= 2 * np.abs(wide[HALF]).max() + 1).all()
    rms = [np.sqrt(np.mean(x[HALF] ** 2)) for x in (eight, wide)]
    assert rms[0] <= 1.25 * rms[1]


def test_a_weight_whose_gradient_ends():
    """One weight among others with gradients: 0.1 for 100 steps, then none for 5000."""
    def g(rng, t):
        x = rng.standard_normal(256 * BLOCKS)
        x[::256] = 0.1 if t < 100 else 0.0
        return x
    eight, wide = train(g, 5100, 0.9, 0.95, 100)
    assert (np.abs(eight[::256]) <= 2 * np.abs(wide[::256]) + 1).all()


@pytest.mark.parametrize("b2", [0.95, 0.999])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2])
def test_small_random_gradients_move_no_further(b2, size):
    """HALF's are `size` of the others' from step 100 on. In 32 bits such weights wander, by at most one step each way; in 8 bits no further: their v
    is at least a ninth of g^2 or its moments 0. Twice the root mean square, or 3 steps while they get there."""
    eight, wide = train(gradients(lambda rng, t: 1.0 if t < 100 else size), 1100, 0.9, b2, 100)
    rms = [np.sqrt(np.mean(x[HALF] ** 2)) for x in (eight, wide)]
    assert rms[0] <= 2 * rms[1] + 3


@pytest.mark.parametrize("b2", [0.95, 0.999])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1e-1])
def test_small_steady_gradients_make_steps_of_adamw_s_size(b2, size):
    """HALF's are `size` of the others', the same each step, from the first one on: AdamW makes a step of 1 each time, 8 bits at most of 3 (v is
    at least a ninth of g^2 once it has followed)."""
    share = np.tile(np.linspace(0.3, 3, 256), BLOCKS)

    def g(rng, t):
        return np.where(HALF, size * share, rng.standard_normal(256 * BLOCKS))
    eight, wide = train(g, 600, 0.9, b2, 200)
    assert np.allclose(wide[HALF], -400, rtol=1e-2)
    assert (eight[HALF] >= -1200).all() and (eight[HALF] <= 0).all()


@pytest.mark.parametrize("b2", [0.95, 0.999])
def test_weights_with_gradients_move_as_in_32_bits(b2):
    """Codes are moved where rounding would hold them, and there alone: the others' weights are those of 32 bits. b2 0.999: v follows by whole
    codes (2% and more of it), later than AdamW's."""
    eight, wide = train(gradients(lambda rng, t: float(t < 100)), 1100, 0.9, b2, 100)
    x, y = eight[~HALF], wide[~HALF]
    assert np.corrcoef(x, y)[0, 1] >= (0.999 if b2 == 0.95 else 0.99)
    assert 0.8 <= np.sqrt(np.mean(x ** 2) / np.mean(y ** 2)) <= 1.1
