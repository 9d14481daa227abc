"""8-bit moments that rounding would hold: the kernel's codes against numpy's, and its weights against 32-bit moments'."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import adam8_ref as a8

pytestmark = pytest.mark.gpu
BLOCKS = 6
N = 256 * BLOCKS


class Moments:
    def __init__(self, dgm, gpu, n, g, decay=False):
        blocks = -(-n // 256)
        z = lambda dtype, count: torch.zeros(count, dtype=dtype, device="cuda")
        self.w, self.m, self.v = torch.full((n,), 0.01, device="cuda"), z(torch.int8, n), z(torch.uint8, n)
        self.ms, self.vs = z(torch.float32, blocks), z(torch.float32, blocks)
        self.plan = gpu.adamMany_plan([dgm.adam_tensor(self.w, g, self.m, self.v, self.ms, self.vs, decay=decay)], 8)


@pytest.mark.parametrize("b1,b2", [(0.9, 0.95), (0.9, 0.999), (0.0, 0.95), (0.95, 0.99)])
def test_codes_are_numpy_s(dgm, gpu, torch_cuda, b1, b2):
    """Blocks with halves that lose their gradients, keep small ones, or have steady small ones: every step's bits."""
    rng = np.random.default_rng(3)
    g, factor = torch.zeros(N, device="cuda"), torch.tensor([0.5], device="cuda")
    s = Moments(dgm, gpu, N, g)
    w, state = s.w.cpu().numpy(), a8.zeros(BLOCKS)
    at = np.arange(N)
    half, block = at % 256 < 128, at // 256
    steady = 1e-3 * (1 + at % 256 / 64)
    moved = np.zeros(2, np.int64)
    for t in range(60):
        x = rng.standard_normal(N)
        quiet = np.choose(block, [x if t < 5 else 0 * x, x * (1 if t < 5 else 1e-3), steady, steady if t > 20 else 1e-9 * x, x, 1e-4 * x])
        x = np.where(half, quiet, x).astype(a8.F)
        g.copy_(torch.from_numpy(x))
        hyper = dict(lr=1e-3, b1=b1, b2=b2, eps=1e-8, wd=0.0)
        inv = 1 / (1 - b1 ** (t + 1)), 1 / (1 - b2 ** (t + 1))
        w, state, where = a8.step(w, x, state, 0.5 if t % 2 else 1.0, **hyper, inv1=inv[0], inv2=inv[1])
        moved += [k.sum() for k in where]
        gpu.begin()
        gpu.adamMany(s.plan, **hyper, invBC1=inv[0], invBC2=inv[1], factor=factor if t % 2 else None)
        gpu.end()
        assert np.array_equal(s.w.cpu().numpy(), w), t
        for got, want in zip((s.m, s.ms, s.v, s.vs), state):
            assert np.array_equal(got.cpu().numpy(), want), t
    assert moved[1] > 0 and (moved[0] > 0) == (b1 > 0.0)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_codes_of_tensors_at_any_element(dgm, gpu, torch_cuda, offset):
    """The same where buffers begin between 16-byte boundaries, and end inside a lane's 8 elements."""
    n, pad = N - 77, lambda x: np.concatenate([x, np.zeros(-len(x) % 256, x.dtype)])
    rng = np.random.default_rng(offset)
    part = lambda dtype, count: torch.full((count + offset + 8,), 3, dtype=dtype, device="cuda")[offset:offset + count].zero_()
    w8, g, m, v, ms, vs = (part(t, k) for t, k in ((torch.float32, n), (torch.float32, n), (torch.int8, n), (torch.uint8, n),
                                                   (torch.float32, BLOCKS), (torch.float32, BLOCKS)))
    plan = gpu.adamMany_plan([dgm.adam_tensor(w8, g, m, v, ms, vs, decay=False)], 8)
    w, state, moved = np.zeros(N, a8.F), a8.zeros(BLOCKS), 0
    for t in range(40):
        x = rng.standard_normal(n).astype(a8.F)
        x[rng.permutation(n) % 3 == 0] *= a8.F(1e-3)
        if t > 5:
            x[np.arange(n) % 5 == 0] = 0
        g.copy_(torch.from_numpy(x))
        hyper, inv = dict(lr=1e-3, b1=0.9, b2=0.95, eps=1e-8, wd=0.0), (1 / (1 - 0.9 ** (t + 1)), 1 / (1 - 0.95 ** (t + 1)))
        w, state, where = a8.step(w, pad(x), state, **hyper, inv1=inv[0], inv2=inv[1])
        moved += where[0].sum()
        gpu.begin()
        gpu.adamMany(plan, **hyper, invBC1=inv[0], invBC2=inv[1])
        gpu.end()
        assert np.array_equal(w8.cpu().numpy(), w[:n])
        for got, want, k in zip((m, ms, v, vs), state, (n, BLOCKS, n, BLOCKS)):
            assert np.array_equal(got.cpu().numpy(), want[:k]), t
    assert moved > 0


@pytest.mark.parametrize("b2", [0.95, 0.999])
def test_weights_without_gradients_come_to_rest(dgm, gpu, torch_cuda, b2):
    """From step 100 on the first half of each block has no gradients: over 1000 steps its weights move within a factor of 2 of
    those with 32-bit moments, or a step (test_adam8_rule.py has why); the others' weights stay near theirs."""
    n, lr = 256 * 64, 1e-3
    gen = torch.Generator("cuda").manual_seed(2)
    g = torch.zeros(n, device="cuda")
    s = Moments(dgm, gpu, n, g)
    wide = {k: torch.zeros(n, device="cuda") for k in "wmv"}
    plan = gpu.adamMany_plan([dgm.adam_tensor(wide["w"], g, wide["m"], wide["v"], decay=False)])
    half = torch.arange(n, device="cuda") % 256 < 128
    gpu.begin()
    for t in range(1100):
        g.normal_(generator=gen)
        if t >= 100:
            g.masked_fill_(half, 0.0)
        for p in (s.plan, plan):
            gpu.adamMany(p, lr, 0.9, b2, 1e-8, 0.0, 1 / (1 - 0.9 ** (t + 1)), 1 / (1 - b2 ** (t + 1)))
        if t == 99:
            start = s.w.clone(), wide["w"].clone()
    gpu.end()
    eight, full = (s.w - start[0]) / lr, (wide["w"] - start[1]) / lr
    assert (eight[half].abs() <= 2 * full[half].abs().max() + 1).all()
    assert eight[half].norm() <= 1.25 * full[half].norm()
    x = torch.corrcoef(torch.stack([eight[~half], full[~half]]))[0, 1]
    assert x >= (0.999 if b2 == 0.95 else 0.99)
    assert 0.8 <= eight[~half].norm() / full[~half].norm() <= 1.1


def test_second_moments_of_the_smallest_blocks(dgm, gpu, torch_cuda):
    """Blocks whose largest v is 2^-120 and a little more: code 1 stands for 2^-32 of that, less than half the smallest fp32 number. It is above 0
    all the same, so that a step with an eps of 0 is finite."""
    n = 256 * 8
    g = torch.full((8, 256), 2.0 ** -74.5, device="cuda")       # v 2^-149
    g[:, 1::3] = 2.0 ** -70
    g[:, 0] = torch.tensor([2.0 ** (-60 + k / 8) for k in range(8)], device="cuda")
    g = g.view(-1)
    s = Moments(dgm, gpu, n, g)
    w, state = s.w.cpu().numpy(), a8.zeros(8)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    hyper = dict(lr=1e-3, b1=0.0, b2=0.0, eps=0.0, wd=0.0)
    for t in range(3):
        if t:      # what the codes stand for, nothing new
            hyper.update(b1=0.5, b2=0.96875)
            g.zero_()
        w, state, _ = a8.step(w, g.cpu().numpy(), state, **hyper, inv1=1.0, inv2=1.0)
        gpu.begin()
        gpu.adamMany(s.plan, **hyper, invBC1=1.0, invBC2=1.0)
        gpu.adamMany_states(s.plan, m, v)
        gpu.end()
        want = a8.values(state)
        assert np.array_equal(m.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])
        assert np.array_equal(s.w.cpu().numpy(), w, equal_nan=True)
        if t == 0:
            assert (s.v > 0).all() and (v > 0).all() and (s.v == 1).any()
    assert torch.isfinite(s.w.view(8, 256)[1:]).all()      # the first one's largest fell below 2^-120, where all are zeros
