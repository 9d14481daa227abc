"""Rows of up to 128 elements round each operation on its own, as the formula is written: rows of two are numpy's bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_layer_norm import BF16, F32, code

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_of_two(dgm, gpu, torch_cuda, dtype, residual):
    """All but eps / variance of dx cancels there, so that what remains shows where an operation was fused with the next."""
    rows, eps = 3001, F(1e-5)
    gen = torch.Generator("cuda").manual_seed(5)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    x, res, dy, dsum = (rand(rows, 2).to(dtype) for _ in range(4))
    w, b = 1 + 0.1 * rand(2), 0.1 * rand(2)
    h, y, dx = (torch.zeros_like(x) for _ in range(3))
    mean, rstd, dw, db = (torch.zeros(n, device="cuda") for n in (rows, rows, 2, 2))
    cfg = dgm.NormCfg(type=code(dgm, dtype), eps=float(eps), rows=rows, cols=2)
    ws = torch.empty(max(gpu.layerNormBwd_ws_bytes(cfg), 16), dtype=torch.uint8, device="cuda")
    gpu.begin()
    gpu.layerNormFwd(cfg, x, res if residual else None, w, b, h if residual else None, y, mean, rstd)
    gpu.layerNormBwd(cfg, h if residual else x, mean, rstd, w, dy, dsum if residual else None, dx, dw, db, ws, ws.numel())
    gpu.end()

    def of(t):
        return t.float().cpu().numpy()

    def same(got, want):
        return torch.equal(got.cpu(), torch.from_numpy(want.astype(F)).to(got.dtype))
    held = (x.float() + res.float()).to(dtype) if residual else x
    assert not residual or torch.equal(h, held)
    v, W, B, g0 = of(held), of(w), of(b), of(dy)
    m = (v[:, :1] + v[:, 1:]) / F(2)
    d = v - m
    ss = d * d
    r = F(1) / np.sqrt((ss[:, :1] + ss[:, 1:]) / F(2) + eps)
    assert same(mean, m[:, 0]) and same(rstd, r[:, 0])
    assert same(y, d * r * W + B)
    xh, g = d * r, g0 * W
    s1 = (g[:, :1] + g[:, 1:]) / F(2)
    gx = g * xh
    s2 = (gx[:, :1] + gx[:, 1:]) / F(2)
    inner = -xh * s2 + (g - s1)
    assert same(dx, r * inner + of(dsum) if residual else r * inner)


@pytest.mark.parametrize("rows,cols", [(1024, 128), (1023, 33), (2048, 512), (77, 1000), (5, 7), (1, 3)])
def test_sums_over_rows_of_unlike_sizes(dgm, gpu, torch_cuda, rows, cols):
    """A row of 2^24 first and rows of 1 behind it, which a running sum that holds the first would lose one by one. The rows are in 16 shares, which
    add eights of rows, then those, and at last the shares and what was there: u of the sum of magnitudes for each addition in a row."""
    dy = torch.ones(rows, cols, device="cuda")
    dy[0] = 2.0 ** 24
    x = torch.randn(rows, cols, device="cuda")
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    w, dx, dw, db = torch.ones(cols, device="cuda"), torch.zeros_like(x), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=1e-5, rows=rows, cols=cols)
    assert gpu.layerNormBwd_ws_bytes(cfg) == 0
    gpu.begin()
    gpu.layerNormBwd(cfg, x, mean, rstd, w, dy, None, dx, dw, db, None, 0)
    gpu.end()
    u = 2.0 ** -24
    for got, terms in ((db, dy.double()), (dw, dy.double() * x.double())):
        adds = 8 + -(-rows // 128) + 16 + 1
        assert ((got.double() - terms.sum(0)).abs() <= adds * u * terms.abs().sum(0)).all()
