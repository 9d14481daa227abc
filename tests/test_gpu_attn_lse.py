"""lse of the packed forward against its definition: the base-2 logarithm of the row's sum of 2^(score log2 e)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref
from test_gpu_attn_packed import FORWARD, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_,H,KVH,D,lens,causal,fused,front,back", FORWARD + [
    ("f32", 2, 1, 256, [70, 1, 200], True, False, 0, 2), ("bf16", 4, 2, 136, [33, 150], False, True, 0, 0),
    ("bf16", 2, 1, 64, [1] * 300, True, False, 0, 0)])
@pytest.mark.parametrize("scale", [None, 3.0])
def test_lse(gpu, dgm, type_, H, KVH, D, lens, causal, fused, front, back, scale):
    """attn_ref.scores bounds a weight's relative error, which holds the score's and the maximum's; the sum of n of them is
    off by (n + 2) U more; the logarithm is good to 2 U, and it and the maximum are rounded and added (2 U of each)."""
    c = Case(dgm, type_, H, KVH, D, lens, causal, fused, front, back, scale=scale)
    gpu.begin()
    c.forward(gpu)
    gpu.end()
    q, k = c.q.double(), c.k.double()
    for a, b in zip(c.starts_list[:-1], c.starts_list[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda")
        seen = seen.tril() if causal else seen
        for h in range(H):
            S, _, off = attn_ref.scores(q[a:b, h].contiguous(), k[a:b, h * KVH // H].contiguous(), c.scale, seen)
            want = torch.logsumexp(S, 1) * attn_ref.LOG2E
            off = off.masked_fill(~seen, 0.0).amax(1)
            top = S.masked_fill(~seen, -math.inf).amax(1).abs() * attn_ref.LOG2E
            bound = (off + (n + 2) * attn_ref.U) * attn_ref.LOG2E + 2 * attn_ref.U * (2 * want.abs() + top + 2)
            attn_ref.assert_within(c.lse[h, a:b], want, bound, f"head {h}")
