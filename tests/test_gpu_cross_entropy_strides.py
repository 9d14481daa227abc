"""Logits at the largest row stride that the header names, and at the first that is refused."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref

pytestmark = pytest.mark.gpu


def test_logits_2_30_apart(dgm, gpu, torch_cuda):
    """Rows 2^30 elements apart are taken, and right; one element more is refused."""
    ld, V = 1 << 30, 100
    flat = torch.zeros(ld + V, device="cuda")
    z = torch.randn(2, V, device="cuda")
    flat[:V], flat[ld:] = z[0], z[1]
    targets = torch.tensor([3, 99], dtype=torch.int32, device="cuda")
    loss, lse, dz = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(ld + V, device="cuda")

    def cfg(rows, ld):
        return dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=0.5, rows=rows, V=V, ld=ld)
    gpu.begin()
    gpu.crossEntropy(cfg(2, ld), flat, targets, loss, None, lse, dz)
    gpu.crossEntropy(cfg(0, ld), None, None, None)
    gpu.end()
    for got, (want, bound) in zip((loss, lse, torch.stack([dz[:V], dz[ld:]])),
                                  (lambda e: ((e[0], e[3]), (e[1], e[4]), (e[2], e[5])))(ref.cross_entropy(z, targets, 0.5))):
        assert ((got.double() - want).abs() <= bound + ref.U * want.abs()).all()
    assert not dz[V:ld].any()
    for rows in (0, 1):
        gpu.begin()
        with pytest.raises(dgm.DgmError) as e:
            gpu.crossEntropy(cfg(rows, ld + 1), flat.data_ptr(), targets, loss)
        assert e.value.code == dgm.DGM_ERR_UNSUPPORTED
        with pytest.raises(dgm.DgmError):
            gpu.end()
