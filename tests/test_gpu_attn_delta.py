"""Rows that see few keys in the backward: their delta is the sum of P dP, whatever else is in the batch and however its
rows are laid over waves (attn_ref.py derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import attn_ref
from test_gpu_attn_packed import Case

pytestmark = pytest.mark.gpu

FEW = {"f32": 16, "bf16": 64}     # keys


def run(gpu, c):
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    return c


# fp32 heads to 32 in few workgroups take dq, dk and dv in one launch; the others, a launch for dq.
@pytest.mark.parametrize("type_,H,KVH,D,lens", [
    ("f32", 4, 4, 32, [1, 200]), ("f32", 4, 4, 32, [200, 1, 150]), ("f32", 4, 2, 24, [1, 1, 300]), ("f32", 8, 2, 32, [900, 1]),
    ("f32", 4, 2, 64, [1, 300]), ("f32", 2, 2, 128, [700, 1]), ("bf16", 4, 4, 32, [1, 200]), ("bf16", 4, 2, 128, [1, 1000]),
    ("bf16", 8, 2, 96, [600, 1, 30]), ("bf16", 72, 8, 64, [300, 1, 640])])
@pytest.mark.parametrize("causal", [True, False])
def test_one_key_has_no_slope_beside_long_sequences(gpu, dgm, type_, H, KVH, D, lens, causal):
    """A softmax over one key is 1 whatever the score: dq and dk are 0. Causal: the first row of any sequence."""
    c = run(gpu, Case(dgm, type_, H, KVH, D, lens, causal))
    for s, n in enumerate(lens):
        at = c.starts_list[s]
        if n == 1:
            assert not c.dq[at].any() and not c.dk[at].any(), s
        if causal:
            assert not c.dq[at].any(), s
    c.check(True)


@pytest.mark.parametrize("H,KVH,D", [(4, 4, 32), (4, 4, 8), (3, 3, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_short_sequences_keep_their_bits_beside_long_ones(gpu, dgm, H, KVH, D, causal):
    """fp32, in one launch beside a long sequence and in two without it: the same products, the same delta."""
    long = run(gpu, Case(dgm, "f32", H, KVH, D, [2, 5, 16, 150], causal))
    short = Case(dgm, "f32", H, KVH, D, [2, 5, 16], causal)
    for name in ("q", "k", "v", "dout"):
        getattr(short, name).copy_(getattr(long, name)[:23])
    run(gpu, short)
    for name in ("out", "dq", "dk", "dv"):
        assert torch.equal(getattr(short, name), getattr(long, name)[:23]), name


def tight(c, few):
    """dq, dk and their bounds where rows that see `few` keys or less have a delta as exact as the products, and the others
    one from the output as it was rounded. bf16: dS in two pieces, off by 2^-8 of what one is."""
    bf16 = c.q.dtype == torch.bfloat16
    q, k, v, dout = (t.double() for t in (c.q, c.k, c.v, c.dout))
    H, KVH, D = q.shape[1], k.shape[1], q.shape[2]
    val, off = ([torch.zeros_like(q), torch.zeros_like(k)] for _ in range(2))
    for a, b in zip(c.starts_list[:-1], c.starts_list[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda")
        seen = seen.tril() if c.causal else seen
        for h in range(H):
            g = h * KVH // H
            args = [t.contiguous() for t in (q[a:b, h], k[a:b, g], v[a:b, g])]
            S, W, eW = attn_ref.scores(args[0], args[1], c.scale, seen)
            lse = torch.logsumexp(S, 1, keepdim=True)
            eP = 2 * eW + (n + 4) * attn_ref.U + 4 * attn_ref.U * lse.abs()
            near = (W * (eP + (D + n + 4) * attn_ref.U)) @ args[2].abs()    # the sum of P dP, as an error of out
            _, rounded = attn_ref.forward(*args, c.scale, seen, c.q.dtype, bf16)
            of_out = torch.where(seen.sum(1, keepdim=True) <= few, near, rounded)
            grad = dout[a:b, h].contiguous()
            (dq, dk, _), e0 = attn_ref.backward(*args, c.scale, seen, of_out, grad, False)
            _, e1 = attn_ref.backward(*args, c.scale, seen, of_out, grad, True)
            for i, (x, at) in enumerate(((dq, h), (dk, g))):
                val[i][a:b, at] += x
                off[i][a:b, at] += e0[i] + (2.0 ** -8 * (e1[i] - e0[i]) if bf16 else 0.0) + 4 * n * attn_ref.U * x.abs()
    return val, [e + attn_ref.rounding(c.q.dtype) * (x.abs() + e) + 1e-30 for x, e in zip(val, off)]


# In each layout of a block of queries: whole waves, pairs, and narrow blocks; tiles of 64 and of 32 keys.
@pytest.mark.parametrize("H,KVH,lens", [(4, 2, [128]), (4, 2, [40, 1000]), (2, 1, [33, 64, 500, 65]), (24, 8, [300, 50, 640]),
                                        (72, 8, [300, 50, 640]), (8, 4, [100] * 9)])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_few_keys_keep_the_precision_of_bf16(gpu, dgm, H, KVH, lens, D, causal):
    c = run(gpu, Case(dgm, "bf16", H, KVH, D, lens, causal))
    val, bound = tight(c, FEW["bf16"])
    for name, x, e in zip(("dq", "dk"), val, bound):
        attn_ref.assert_within(getattr(c, name), x, e, name)


@pytest.mark.parametrize("H,KVH,D,lens", [(4, 4, 32, [3, 200, 16, 17]), (4, 2, 64, [128, 9]), (2, 1, 128, [12, 500])])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_few_keys_in_fp32(gpu, dgm, H, KVH, D, lens, causal):
    c = run(gpu, Case(dgm, "f32", H, KVH, D, lens, causal))
    val, bound = tight(c, FEW["f32"])
    for name, x, e in zip(("dq", "dk"), val, bound):
        attn_ref.assert_within(getattr(c, name), x, e, name)
