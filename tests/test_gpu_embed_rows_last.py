"""The last of a token's gradient rows: in a segment of its own, and beyond element 2^31."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_token_of_many_rows_takes_the_last_one_too(dgm, gpu, torch_cuda):
    """A token of 66 rows, of which the last lies in a segment of its own behind 64 others: its sum is exact in whole numbers."""
    rows, C, V = 66 * 80, 8, 100_000
    cfg = dgm.RowsCfg(type=dgm.DGM_TYPE_F32, tableType=dgm.DGM_TYPE_F32, scale=1.0, rows=rows, C=C, V=V)
    ws = torch.empty(gpu.embedRowsBwd_ws_bytes(cfg), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0      # sorted
    tokens = (torch.arange(rows, device="cuda") % 80 * 7).to(torch.int32)
    dy = torch.randint(-100, 101, (rows, C), device="cuda").float()
    dtable = torch.full((V, C), 7.0, device="cuda")
    gpu.begin()
    gpu.embedRowsBwd(cfg, tokens, dy, dtable, ws, ws.numel())
    gpu.end()
    want = torch.zeros(V, C, device="cuda").index_add_(0, tokens.long(), dy)
    assert torch.equal(dtable, want)


def test_last_rows_beyond_32_bits_reach_their_tokens(dgm, gpu, torch_cuda):
    """Gradient rows that lie beyond element 2^31, each to its token, and to one of two million rows of zeros and one of 64: whole numbers, exact."""
    rows, C = 2_100_000, 1030
    tokens = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    tokens[-7:] = torch.arange(7, device="cuda")
    dy = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    dy[-7:] = torch.randint(-9, 10, (7, C), device="cuda").bfloat16()
    dy[17] = 64
    want = dy[-7:].float()
    want[5] += 64
    dtable = torch.full((3000, C), 7.0, device="cuda")
    cfg = dgm.RowsCfg(type=dgm.DGM_TYPE_BF16, tableType=dgm.DGM_TYPE_F32, scale=1.0, rows=rows, C=C, V=3000)
    ws = torch.empty(gpu.embedRowsBwd_ws_bytes(cfg), dtype=torch.uint8, device="cuda")
    gpu.begin()
    gpu.embedRowsBwd(cfg, tokens, dy, dtable, ws, ws.numel())
    gpu.end()
    assert torch.equal(dtable[:7], want) and not dtable[7:].any()
