"""Losses that are small beside their logits: rows that a model is sure of, and rows far from 0."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref
from test_gpu_layer_norm import BF16, F32, code

pytestmark = pytest.mark.gpu
U = ref.U


def losses(dgm, gpu, z, targets, gradient):
    rows, V = z.shape
    cfg = dgm.LossCfg(type=code(dgm, z.dtype), scale=1.0, rows=rows, V=V)
    loss = torch.zeros(rows, device="cuda")
    gpu.begin()
    gpu.crossEntropy(cfg, z, targets, loss, dlogits=torch.zeros_like(z) if gradient else None)
    gpu.end()
    return loss.double()


def exact(z, targets, adds):
    """(losses in 64 bits, bound). (m - z_t) is off by u of itself; e^(z - m) as step_ref has it; `adds` additions of positive terms by u of the
    sum each; the logarithm's instruction, its constant and product 4 u and 2 u of the result; the last sum u of the loss."""
    z = z.double()
    m = z.max(1, keepdim=True).values
    p = torch.exp(z - m)
    total = p.sum(1)
    wrong = (p * (3 * (z - m).abs() + 4) * U).sum(1) / total
    # The largest term's own error: e^0 by the power of two is exact.
    wrong -= (p == 1).sum(1) * 4 * U / total
    far = m[:, 0] - z.gather(1, targets.long()[:, None])[:, 0]
    rest = p.masked_fill(p == 1, 0).sum(1) + (p == 1).sum(1) - 1
    ln = torch.log1p(rest)
    loss = far + ln
    return loss, U * far + wrong + (adds + 4) * U + 2 * U * ln + U * loss


# Lanes of 16, 64 and 256 threads, a workgroup of 512, and the loop (without a gradient); with the additions of a lane, its wave and
# those of the waves.
KERNELS = [(16, True, 4 + 4), (100, True, 9 + 4), (1000, True, 17 + 6), (5000, True, 33 + 6 + 4), (20000, True, 33 + 6 + 16),
           (50000, False, 52 + 6 + 16 + 4)]


@pytest.mark.parametrize("V,gradient,adds", KERNELS)
@pytest.mark.parametrize("shift", [0.0, 100.0, -100.0, 1000.0, 1e4])
def test_rows_that_are_sure(dgm, gpu, torch_cuda, shift, V, gradient, adds):
    """Losses of about 1e-5, of logits around `shift`. One taken from a rounded lse would be off by up to half a step of the logits: 4e-6 at 100, 6e-5 at 1000."""
    gen = torch.Generator("cuda").manual_seed(V)
    rows = 64
    low = torch.log(torch.tensor((V - 1) / 1e-5)).item()
    z = (torch.randn(rows, V, generator=gen, device="cuda") * 0.3 - low).clamp(max=-8) + shift
    targets = torch.randint(0, V, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    z.scatter_(1, targets.long()[:, None], shift)
    got = losses(dgm, gpu, z, targets, gradient)
    want, bound = exact(z, targets, adds)
    assert (want > 5e-6).all() and (want < 1e-4).all()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,gradient,adds", [(200, True, 64), (3000, True, 64), (70000, False, 128)])
def test_a_shift_of_all_logits_changes_nothing(dgm, gpu, torch_cuda, dtype, V, gradient, adds):
    """Logits at multiples of 1/2 stay exact under a shift that is one, too: the same bits."""
    gen = torch.Generator("cuda").manual_seed(V)
    z = torch.randint(-20, 1, (33, V), generator=gen, device="cuda") / 2
    targets = torch.randint(0, V, (33,), generator=gen, device="cuda", dtype=torch.int32)
    shifts = (0.0, 64.0, -50.5) if dtype == BF16 else (0.0, 64.0, -50.5, 4096.5, -65536.0)
    got = [losses(dgm, gpu, (z + s).to(dtype), targets, gradient) for s in shifts]
    assert all(torch.equal(got[0], x) for x in got[1:])
    want, bound = exact(z, targets, adds)
    assert ((got[0] - want).abs() <= bound).all()
