"""Lookup of token embeddings and its gradient by sorted tokens, against 64 bits."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref
from test_gpu_layer_norm import BF16, F32, code, within

pytestmark = pytest.mark.gpu


def rows_cfg(dgm, dtype, rows, C, V, scale=1.0, table=F32):
    return dgm.RowsCfg(type=code(dgm, dtype), tableType=code(dgm, table), scale=scale, rows=rows, C=C, V=V)


def text(rows, V, seed, none=True):
    """Few tokens often, many seldom; some rows without one."""
    gen = torch.Generator("cuda").manual_seed(seed)
    t = (torch.rand(rows, generator=gen, device="cuda") ** 4 * V).to(torch.int32).clamp(max=V - 1)
    if none and rows > 3:
        t[1::9] = -1
        t[-1] = -1
    return t


@pytest.mark.parametrize("table", [F32, BF16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,V", [(1, 1, 1), (5, 3, 2), (17, 8, 9), (100, 33, 65), (64, 128, 65), (9, 1000, 7), (33, 2047, 50),
                                      (4, 2048, 300), (7, 4099, 100), (1030, 72, 500)])
def test_lookup(dgm, gpu, torch_cuda, rows, C, V, dtype, table):
    offset = (rows + C) % 3
    wte = torch.randn(V * C + 3, device="cuda").to(table)[offset:offset + V * C].view(V, C)
    flat = torch.full((rows * C + 16,), 7.0, device="cuda").to(dtype)
    y = flat[offset:offset + rows * C].view(rows, C)
    t = text(rows, V, rows)
    scale = 11.3
    gpu.begin()
    gpu.embedRows(rows_cfg(dgm, dtype, rows, C, V, scale, table), t, wte, y)
    gpu.end()
    want = torch.where((t >= 0)[:, None], wte.double()[t.long().clamp(min=0)] * torch.tensor(scale).item(), torch.zeros((), device="cuda").double())
    within(y, want, ref.U * want.abs(), dtype)
    assert (y[t < 0] == 0).all()
    assert (flat[:offset] == 7).all() and (flat[offset + rows * C:] == 7).all()


def backward(dgm, gpu, cfg, t, dy, dtable, add):
    size = gpu.embedRowsBwd_ws_bytes(cfg)
    ws = torch.full((size + 64,), 0x7F, dtype=torch.uint8, device="cuda")
    gpu.embedRowsBwd(cfg, t, dy, dtable, ws, size, accumulate=add)
    gpu.end()
    gpu.begin()
    assert (ws[size:] == 0x7F).all()


# Without a sort by the vocabulary's rows or by the batch's (up to 4096 rows, the fewer of them x columns / 256 up to 2048; 512 with
# wide workgroups), sorted by one workgroup (4096 rows) or several;
# digits of up to 9 bits (V of 511, 512: one pass or two); segments of 8 to 64 sorted rows.
SIZES = [(1, 1, 1), (2, 5, 1), (63, 7, 3), (64, 8, 3), (65, 33, 4), (130, 260, 1), (1000, 20, 65), (4096, 12, 511), (4097, 12, 512),
         (5000, 130, 40), (9000, 9, 50257), (20000, 4, 2), (3000, 515, 200), (300, 2050, 31), (70000, 3, 262143), (70001, 3, 262144),
         (33, 64, 2 ** 27), (1, 9, 5000), (1025, 5, 3000), (2500, 260, 5000), (4096, 12, 70000), (3500, 8, 2 ** 24), (4100, 4096, 2000),
         (30000, 1028, 300), (511, 9, 700), (2047, 8, 5000), (2048, 33, 2049), (700, 700, 800), (1500, 300, 1000), (4096, 12, 2049)]


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,V", SIZES)
def test_gradient(dgm, gpu, torch_cuda, rows, C, V, dtype, add):
    if V * C > 1 << 30:
        C = 1
    offset = (rows + C) % 4
    flat = torch.full((V * C + 8,), 3.0, device="cuda")
    dtable = flat[offset:offset + V * C].view(V, C)
    dy = torch.randn(rows * C + 3, device="cuda").to(dtype)[offset % 3:offset % 3 + rows * C].view(rows, C)
    t = text(rows, V, rows + V)
    cfg = rows_cfg(dgm, dtype, rows, C, V, 0.7)
    gpu.begin()
    backward(dgm, gpu, cfg, t, dy, dtable, add)
    first = dtable.clone()
    if add:
        dtable.fill_(3.0)
    backward(dgm, gpu, cfg, t, dy, dtable, add)
    gpu.end()
    assert torch.equal(first, dtable)
    met = torch.unique(t[t >= 0].long())
    sums, err = ref.embed_bwd(torch.searchsorted(met, t.long()).where(t >= 0, -1), dy, len(met), torch.tensor(0.7).item())
    base = 3.0 if add else 0.0
    within(dtable[met], base + sums, err + 2 * ref.U * (base + sums.abs()))
    rest = torch.ones(V, dtype=torch.bool, device="cuda")
    rest[met] = False
    assert (dtable[rest] == base).all()
    assert (flat[:offset] == 3).all() and (flat[offset + V * C:] == 3).all()


@pytest.mark.parametrize("rows", [64, 500, 4096, 10000])
def test_one_token_and_all_different(dgm, gpu, torch_cuda, rows):
    """Runs over every segment; runs of one. Whole numbers, whose sums are exact in any order."""
    C, V = 37, 10000
    dy = torch.randint(-8, 9, (rows, C), device="cuda").float()
    dtable = torch.zeros(V, C, device="cuda")
    cfg = rows_cfg(dgm, F32, rows, C, V)
    for t in (torch.full((rows,), V - 1, device="cuda"), torch.randperm(V, device="cuda")[:rows], torch.arange(rows, device="cuda") // 64,
              torch.arange(rows, device="cuda").flip(0) // 65, torch.full((rows,), -1, device="cuda")):
        t = t.to(torch.int32)
        gpu.begin()
        backward(dgm, gpu, cfg, t, dy, dtable, False)
        gpu.end()
        want = torch.zeros(V, C, device="cuda")
        met = t >= 0
        want.index_add_(0, t[met].long(), dy[met])
        assert torch.equal(dtable, want)


def test_order_of_a_token_s_rows(dgm, gpu, torch_cuda):
    """2^24 takes up no 1 that comes after it, and two that came before."""
    t = torch.tensor([4, 9, 4, 4], dtype=torch.int32, device="cuda")
    dy = torch.tensor([[2.0 ** 24], [5.0], [1.0], [1.0]], device="cuda")
    dtable = torch.zeros(12, 1, device="cuda")
    cfg = rows_cfg(dgm, F32, 4, 1, 12)
    gpu.begin()
    backward(dgm, gpu, cfg, t, dy, dtable, False)
    assert dtable[4, 0] == 2.0 ** 24 and dtable[9, 0] == 5
    backward(dgm, gpu, cfg, t.flip(0).contiguous(), dy.flip(0).contiguous(), dtable, False)
    gpu.end()
    assert dtable[4, 0] == 2.0 ** 24 + 2 and dtable[9, 0] == 5


@pytest.mark.parametrize("rows,V", [(100, 65), (100, 70000), (3000, 70000), (5000, 300), (5000, 70000)])
def test_tokens_beyond_the_vocabulary(dgm, gpu, torch_cuda, rows, V):
    C = 24
    t = text(rows, V, 5)
    bad = t.clone()
    bad[3], bad[rows - 2] = V, -2
    t[3] = t[rows - 2] = -1
    table, dy = torch.randn(V, C, device="cuda"), torch.randn(rows, C, device="cuda")
    cfg = rows_cfg(dgm, F32, rows, C, V)
    out = []
    for tokens in (t, bad):
        y, dtable = torch.ones(rows, C, device="cuda"), torch.ones(V, C, device="cuda")
        for what in ("lookup", "gradient"):
            gpu.begin()
            if what == "lookup":
                gpu.embedRows(cfg, tokens, table, y)
            else:
                size = gpu.embedRowsBwd_ws_bytes(cfg)
                gpu.embedRowsBwd(cfg, tokens, dy, dtable, torch.zeros(size, dtype=torch.uint8, device="cuda"), size)
            if tokens is bad:
                with pytest.raises(dgm.DgmError, match="beyond the vocabulary") as e:
                    gpu.end()
                assert e.value.code == dgm.DGM_ERR_SHAPE
            else:
                gpu.end()
        out.append((y, dtable))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_no_rows(dgm, gpu, torch_cuda):
    dtable = torch.ones(5, 8, device="cuda")
    cfg = rows_cfg(dgm, F32, 0, 8, 5)
    gpu.begin()
    gpu.embedRows(cfg, None, None, None)
    gpu.embedRowsBwd(cfg, None, None, dtable, None, 0, accumulate=True)
    assert (dtable == 1).all()
    gpu.embedRowsBwd(cfg, None, None, dtable, None, 0)
    gpu.end()
    assert (dtable == 0).all()


def test_lookup_and_gradient_are_adjoint(dgm, gpu, torch_cuda):
    """<lookup(W), dY> = <W, gradient(dY)>, the lookup being linear in W: differences of it are its gradient."""
    rows, C, V = 777, 96, 130
    t, w, dy = text(rows, V, 2), torch.randn(V, C, device="cuda"), torch.randn(rows, C, device="cuda")
    cfg = rows_cfg(dgm, F32, rows, C, V, 3.0)
    y, dtable = torch.zeros(rows, C, device="cuda"), torch.zeros(V, C, device="cuda")
    gpu.begin()
    gpu.embedRows(cfg, t, w, y)
    backward(dgm, gpu, cfg, t, dy, dtable, False)
    gpu.end()
    a, b = (y.double() * dy.double()), (w.double() * dtable.double())
    _, err = ref.embed_bwd(t, dy, V, 3.0)
    assert abs(a.sum() - b.sum()) <= (ref.U * a.abs()).sum() + (err * w.double().abs()).sum()


def test_offsets_beyond_32_bits(dgm, gpu, torch_cuda):
    """Rows of a table and of a batch of more than 2^31 elements."""
    V, C = 524300, 4100
    table = torch.zeros(V, C, dtype=BF16, device="cuda")
    dtable = torch.ones(V, C, device="cuda")
    t = torch.tensor([V - 1, 3, V - 2, V - 1], dtype=torch.int32, device="cuda")
    table[t.long()] = torch.randn(4, C, device="cuda").bfloat16()
    table[V - 1] = 2.5
    dy, y = torch.randint(-9, 9, (4, C), device="cuda").float(), torch.zeros(4, C, device="cuda")
    cfg = rows_cfg(dgm, F32, 4, C, V, 2.0, BF16)
    gpu.begin()
    gpu.embedRows(cfg, t, table, y)
    backward(dgm, gpu, cfg, t, dy, dtable, False)
    assert torch.equal(y, 2 * table[t.long()].float())
    assert torch.equal(dtable[V - 1], 2 * (dy[0] + dy[3])) and torch.equal(dtable[V - 2], 2 * dy[2]) and torch.equal(dtable[3], 2 * dy[1])
    assert not dtable[V - 1000:V - 2].any() and not dtable[:3].any()
    gpu.end()
    del dtable, table
    rows, C = 2100000, 1030
    t = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    t[-7:] = torch.arange(7, device="cuda")
    dy = torch.zeros(rows, C, dtype=BF16, device="cuda")
    dy[-7:] = torch.randint(-9, 9, (7, C), device="cuda").bfloat16()
    dy[17] = 64
    dtable = torch.zeros(3000, C, device="cuda")
    cfg = rows_cfg(dgm, BF16, rows, C, 3000, 1.0)
    gpu.begin()
    backward(dgm, gpu, cfg, t, dy, dtable, False)
    gpu.embedRows(cfg, t, dtable, dy)
    gpu.end()
    assert torch.equal(dy[-7:].float(), dtable[:7]) and torch.equal(dy[1].float(), dtable[5]) and not dtable[7:].any()
    assert (dtable[5] >= 64 - 9).all() and (dtable[5] <= 64 + 9).all()


def test_repeats_streams_and_graphs(dgm, gpu, torch_cuda):
    rows, C, V = 6000, 65, 1000
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)
    cfg = rows_cfg(dgm, BF16, rows, C, V, 2.0, BF16)
    table, dy = torch.randn(V, C, device="cuda").bfloat16(), torch.randn(rows, C, device="cuda").bfloat16()
    t, other = text(rows, V, 1), text(rows, V, 77)
    y, dtable = torch.zeros(rows, C, device="cuda").bfloat16(), torch.zeros(V, C, device="cuda")
    size = own.embedRowsBwd_ws_bytes(cfg)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def step(g):
        g.embedRows(cfg, t, table, y)
        g.embedRowsBwd(cfg, t, dy, dtable, ws, size)
        return y.clone(), dtable.clone()
    torch.cuda.synchronize()
    own.begin()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(own)
    first = t.clone()
    for i in range(4):
        t.copy_(other if i % 2 else first)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in out]
        with torch.cuda.stream(side):
            eager = step(own)
        own.end()
        own.begin()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))
    own.end()
    own.close()


def test_refusals(dgm, gpu, torch_cuda):
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    big = torch.zeros(1 << 16, device="cuda")
    addr = {"tokens": t.data_ptr(), "table": big.data_ptr(), "y": big.data_ptr(), "dy": big.data_ptr(), "dtable": big.data_ptr() + (1 << 14),
            "ws": big.data_ptr() + (1 << 15)}

    def refused(status, cfg={}, which="both", ws_bytes=1 << 16, **over):
        a = {**addr, **over}
        c = dgm.RowsCfg(**{**dict(type=0, tableType=0, scale=1.0, rows=4, C=8, V=16), **cfg})
        for k in ("lookup", "gradient"):
            if which not in ("both", k):
                continue
            gpu.begin()
            with pytest.raises(dgm.DgmError) as e:
                if k == "lookup":
                    gpu.embedRows(c, a["tokens"], a["table"], a["y"])
                else:
                    gpu.embedRowsBwd(c, a["tokens"], a["dy"], a["dtable"], a["ws"], ws_bytes)
            assert e.value.code == status
            with pytest.raises(dgm.DgmError):
                gpu.end()
    for bad in (dict(type=9), dict(tableType=9), dict(rows=-1), dict(C=0), dict(V=0), dict(scale=float("nan"))):
        refused(dgm.DGM_ERR_ARG, bad)
    for bad in (dict(rows=(1 << 30) + 1), dict(V=1 << 31), dict(C=(1 << 24) + 1)):
        refused(dgm.DGM_ERR_UNSUPPORTED, bad)
    for k in ("tokens", "table", "y"):
        refused(dgm.DGM_ERR_ARG, which="lookup", **{k: None})
        refused(dgm.DGM_ERR_UNSUPPORTED, which="lookup", **{k: addr[k] + 2})
    large = dict(rows=5000, V=1 << 22)         # too many for each to look for its own: they are sorted, in a workspace
    for k in ("tokens", "dy", "dtable", "ws"):
        refused(dgm.DGM_ERR_ARG, large, which="gradient", ws_bytes=1 << 20, **{k: None})
        refused(dgm.DGM_ERR_UNSUPPORTED, large, which="gradient", ws_bytes=1 << 20, **{k: addr[k] + 2})
    c = dgm.RowsCfg(type=0, tableType=0, scale=1.0, rows=5000, C=8, V=1 << 22)
    refused(dgm.DGM_ERR_ARG, large, which="gradient", ws_bytes=gpu.embedRowsBwd_ws_bytes(c) - 1)
    refused(dgm.DGM_ERR_UNSUPPORTED, dict(rows=1 << 30, C=1 << 24), which="gradient", ws_bytes=1 << 62)
