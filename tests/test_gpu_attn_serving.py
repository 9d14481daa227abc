"""Prompt attention, cache and decode together, as a decoder's layer uses them."""
from __future__ import annotations

import pytest
import torch

import attn_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
def test_prompts_then_tokens(gpu, dgm, bits):
    """Quantized fused projections of prompts, their attention, their keys and
    values into an fp32 cache, then four tokens per sequence: every row equals the
    attention over all rows so far, within the forward's bound."""
    torch.manual_seed(bits)
    H, KVH, D, C, page, group = 4, 2, 32, 128, 16, 32
    lens, new = [37, 1, 64], 4
    N = (H + 2 * KVH) * D
    w = torch.randn(N, C, device="cuda") * 0.2
    codes = torch.zeros(N * C * bits // 8, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(N * C // group, device="cuda")
    need = [-(-(n + new) // page) for n in lens]
    pages = torch.full((3, max(need)), -1, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(sum(need), device="cuda").int(), 0
    for i, n in enumerate(need):
        pages[i, :n] = order[at:at + n]
        at += n
    cfg = dgm.CacheCfg(type=dgm.DGM_TYPE_F32, KVH=KVH, D=D, pageSize=page, numPages=sum(need), maxPages=max(need))
    kc, vc = (torch.full((sum(need), KVH, page, D), float("nan"), device="cuda") for _ in range(2))
    seen = [[] for _ in lens]          # every row of the projection, by sequence
    cut = lambda t: (t[:, :H], t[:, H:H + KVH], t[:, H + KVH:])  # noqa: E731

    def project(x):
        y = torch.zeros(x.shape[0], H + 2 * KVH, D, device="cuda")
        gpu.gemmNT(bits, None, codes, scale, x, None, y, x.shape[0], N, C, group)
        return y

    def check(out, y, s):
        """Rows `out` of sequence s, whose last rows are y, against attention over all."""
        seen[s].append(y.clone())
        q, k, v = cut(torch.cat(seen[s]))
        val, bnd = attn_ref.packed(q, k, v, [0, q.shape[0]], D ** -0.5, True)
        attn_ref.assert_within(out, val["out"][-len(out):], bnd["out"][-len(out):], f"sequence {s}")

    rows = sum(lens)
    starts = torch.tensor([0, 37, 38, 102], dtype=torch.int32, device="cuda")
    gpu.begin()
    gpu.quantize(w, codes, scale, N, C, bits, group)
    y = project(torch.randn(rows, C, device="cuda"))
    q, k, v = cut(y)
    out = torch.zeros(rows, H, D, device="cuda")
    a = dgm.AttnCfg(type=dgm.DGM_TYPE_F32, H=H, KVH=KVH, D=D, causal=1, scale=D ** -0.5, rows=rows, nseq=3,
                    ldq=N, ldk=N, ldv=N, ldo=0)
    gpu.attnPackedFwd(a, q, k, v, starts, out)
    gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, starts, None, pages, kc, vc, rows, 3, N, N)
    gpu.end()
    for s in range(3):
        check(out[starts[s]:starts[s + 1]], y[starts[s]:starts[s + 1]], s)
    size = gpu.attnPagedDecode_ws_bytes(cfg, 3, H)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    have = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for _ in range(new):
        out = torch.zeros(3, H, D, device="cuda")
        gpu.begin()
        y = project(torch.randn(3, C, device="cuda"))
        q, k, v = cut(y)
        gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, None, have, pages, kc, vc, 3, 3, N, N)
        gpu.end()
        have += 1
        gpu.begin()
        gpu.attnPagedDecode(cfg, dgm.DGM_TYPE_F32, q, kc, vc, pages, have, out, ws, size, 3, H, N)
        gpu.end()
        for s in range(3):
            check(out[s:s + 1], y[s:s + 1], s)
