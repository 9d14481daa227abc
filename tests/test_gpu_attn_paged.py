"""The paged cache's write (exact) and the attention of one new token over it,
against 64 bits (attn_ref.py derives the bounds)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def code(dgm, name):
    return dgm.DGM_TYPE_F32 if name == "f32" else dgm.DGM_TYPE_BF16


def table(lens, page, gen, spare=2):
    """Pages of the sequences in no order; -1 where none is needed. Number of pages, table."""
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    t = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return total, t


def cache_case(dgm, io, cache, H, KVH, D, page, lens, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed + D + page + len(lens))
    total, pages = table(lens, page, gen)
    kc, vc = (torch.randn(total, KVH, page, D, generator=gen, device="cuda").to(TYPES[cache]) for _ in range(2))
    q = torch.randn(len(lens), H, D, generator=gen, device="cuda").to(TYPES[io])
    cfg = dgm.CacheCfg(type=code(dgm, cache), KVH=KVH, D=D, pageSize=page, numPages=total, maxPages=pages.shape[1])
    return cfg, q, kc, vc, pages, torch.tensor(lens, dtype=torch.int32, device="cuda")


def decode(gpu, dgm, cfg, io, q, kc, vc, pages, lens, scale=None):
    n, H, D = q.shape
    out = torch.full((n, H, D), 7.0, device="cuda").to(q.dtype)
    size = gpu.attnPagedDecode_ws_bytes(cfg, n, H)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")     # NaN in every float
    gpu.attnPagedDecode(cfg, code(dgm, io), q, kc, vc, pages, lens, out, ws, size, n, H, scale=scale)
    return out


def blank(cfg, kc, vc, pages, lens):
    """NaN in every slot that no position has."""
    used = torch.zeros(kc.shape[0], kc.shape[2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens.tolist()):
        pos = torch.arange(n, device="cuda")
        used[pages[s].long()[pos // cfg.pageSize], pos % cfg.pageSize] = True
    for c in (kc, vc):
        c.permute(0, 2, 1, 3)[~used] = math.nan


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("H,KVH,D,page,lens", [
    (4, 4, 32, 16, [1, 17, 64, 65, 0]),
    (4, 1, 48, 16, [3]),
    (32, 8, 128, 16, [1000, 1, 129, 128]),
    (16, 1, 64, 1, [31, 5]),
    (20, 1, 80, 100, [250, 99, 100, 101]),
    (34, 2, 8, 8, [40, 0, 0, 7]),
    (6, 2, 256, 24, [77, 300]),
    (3, 1, 136, 7, [29]),
    (8, 2, 96, 64, [0, 0]),
    (2, 2, 128, 16, [5000]),
])
def test_decode(gpu, dgm, io, cache, H, KVH, D, page, lens):
    cfg, q, kc, vc, pages, n = cache_case(dgm, io, cache, H, KVH, D, page, lens)
    want, bound = attn_ref.decode(q, kc, vc, pages, lens, D ** -0.5, io == "bf16" and cache == "bf16")
    blank(cfg, kc, vc, pages, n)
    gpu.begin()
    out = decode(gpu, dgm, cfg, io, q, kc, vc, pages, n)
    again = decode(gpu, dgm, cfg, io, q, kc, vc, pages, n)
    gpu.end()
    attn_ref.assert_within(out, want, bound)
    assert torch.equal(out, again)
    for s, length in enumerate(lens):
        assert length > 0 or (out[s] == 0).all()


def test_decode_many_sequences(gpu, dgm):
    """More sequences than workers, lengths from none to some hundreds."""
    lens = [(i * i * 7 + 3 * i) % 257 * (i % 5 != 0) for i in range(700)]
    cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", "bf16", 4, 2, 64, 16, lens)
    gpu.begin()
    out = decode(gpu, dgm, cfg, "f32", q, kc, vc, pages, n)
    gpu.end()
    want, bound = attn_ref.decode(q, kc, vc, pages, lens, 64 ** -0.5, False)
    attn_ref.assert_within(out, want, bound)


def test_decode_strided_and_sharp(gpu, dgm):
    """Query and output rows inside wider ones; scores of hundreds."""
    cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", "bf16", 4, 2, 64, 16, [300, 20])
    wide, out = torch.zeros(2, 8, 64, device="cuda"), torch.full((2, 6, 64), 7.0, device="cuda")
    wide[:, 2:6] = q
    size = gpu.attnPagedDecode_ws_bytes(cfg, 2, 4)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    gpu.begin()
    gpu.attnPagedDecode(cfg, dgm.DGM_TYPE_F32, wide[:, 2:6], kc, vc, pages, n, out[:, 1:5], ws, size, 2, 4,
                        wide.stride(0), out.stride(0), 20.0)
    gpu.end()
    want, bound = attn_ref.decode(q, kc, vc, pages, [300, 20], 20.0, False)
    attn_ref.assert_within(out[:, 1:5], want, bound)
    assert (out[:, 0] == 7).all() and (out[:, 5] == 7).all()


@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_bad_pages_and_lengths_are_left_out(gpu, dgm, cache):
    """A page number that the cache does not have, and a length beyond the table: the other positions count, and the region's end reports it."""
    cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", cache, 4, 2, 64, 16, [100, 90, 40, 10])
    pages[0, 2] = -1
    pages[1, 0] = kc.shape[0]
    pages[2, :3] = 2 ** 31 - 1
    gpu.begin()
    out = decode(gpu, dgm, cfg, "f32", q, kc, vc, pages, n)
    with pytest.raises(dgm.DgmError) as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    want, bound = attn_ref.decode(q, kc, vc, pages, [100, 90, 40, 10], 64 ** -0.5, False)
    attn_ref.assert_within(out, want, bound)
    assert (out[2] == 0).all()
    full = torch.arange(8, dtype=torch.int32, device="cuda").reshape(4, 2) % kc.shape[0]
    cfg.maxPages = 2
    gpu.begin()
    out = decode(gpu, dgm, cfg, "f32", q, kc, vc, full, torch.tensor([32, 33, 1 << 30, -5], dtype=torch.int32,
                                                                   device="cuda"))
    with pytest.raises(dgm.DgmError) as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    want, bound = attn_ref.decode(q, kc, vc, full, [32, 32, 32, 0], 64 ** -0.5, False)
    attn_ref.assert_within(out, want, bound)


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_scores_of_minus_infinity(gpu, dgm, io, cache):
    """Keys that all score -inf leave no softmax (NaN), not the zeros of a sequence
    without keys; among others, where no operand is taken in pieces, they weigh nothing."""
    lens = [300, 300, 0, 9000]
    cfg, q, kc, vc, pages, n = cache_case(dgm, io, cache, 4, 2, 64, 16, lens)
    q.abs_().add_(0.1)
    for s, upto in ((0, 304), (1, 208), (3, 8000)):
        kc[pages[s, :upto // 16].long()] = -math.inf
    gpu.begin()
    out = decode(gpu, dgm, cfg, io, q, kc, vc, pages, n)
    gpu.end()
    assert out[0].isnan().all() and (out[2] == 0).all()
    if io == "bf16" or cache == "f32":
        for s, upto in ((1, 208), (3, 8000)):
            pos = torch.arange(upto, lens[s], device="cuda")
            ids, seen = pages[s].long()[pos // 16], torch.ones(1, len(pos), dtype=torch.bool, device="cuda")
            for h in range(4):
                k, v = (c[ids, h // 2, pos % 16].double() for c in (kc, vc))
                want, bound = attn_ref.forward(q[s, h:h + 1].double(), k, v, 0.125, seen, q.dtype, cache == "bf16")
                attn_ref.assert_within(out[s, h:h + 1], want, bound)


def write_ref(k, v, starts, lens, pages, kc, vc, page):
    kc, vc = kc.clone(), vc.clone()
    for s in range(len(starts) - 1):
        for r in range(starts[s], starts[s + 1]):
            p = lens[s] + r - starts[s]
            at = int(pages[s, p // page])
            kc[at, :, p % page], vc[at, :, p % page] = k[r].to(kc.dtype), v[r].to(vc.dtype)
    return kc, vc


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("KVH,D,page,before,new", [
    (8, 128, 16, [0, 5, 16, 31], [1, 40, 0, 2]),
    (1, 8, 1, [0], [3]),
    (2, 48, 100, [99, 0], [2, 100]),
    (3, 256, 7, [1, 2, 3, 4, 5], [0, 0, 9, 1, 0]),
])
def test_write(gpu, dgm, io, cache, KVH, D, page, before, new):
    gen = torch.Generator("cuda").manual_seed(KVH + D)
    front, back = 2, 3
    total, pages = table([b + n for b, n in zip(before, new)], page, gen)
    rows = front + sum(new) + back
    wide = torch.randn(rows, 2 * KVH, D, generator=gen, device="cuda").to(TYPES[io])
    k, v = wide[:, :KVH], wide[:, KVH:]
    wide[front, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.4e38], device="cuda").to(TYPES[io])
    kc, vc = (torch.randn(total, KVH, page, D, generator=gen, device="cuda").to(TYPES[cache]) for _ in range(2))
    starts = [front]
    for n in new:
        starts.append(starts[-1] + n)
    want = write_ref(k, v, starts, before, pages, kc, vc, page)
    cfg = dgm.CacheCfg(type=code(dgm, cache), KVH=KVH, D=D, pageSize=page, numPages=total, maxPages=pages.shape[1])
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    gpu.begin()
    gpu.cacheWrite(cfg, code(dgm, io), k, v, dev(starts), dev(before), pages, kc, vc, rows, len(new), k.stride(0),
                   v.stride(0))
    gpu.end()
    for got, ref in ((kc, want[0]), (vc, want[1])):
        bits = torch.int32 if got.dtype == torch.float32 else torch.int16
        same = (got.view(bits) == ref.view(bits)) | (got.isnan() & ref.isnan())
        assert same.all()


def test_write_one_row_each_and_fresh_sequences(gpu, dgm):
    gen = torch.Generator("cuda").manual_seed(3)
    before = [0, 15, 16, 40]
    total, pages = table([n + 1 for n in before], 16, gen)
    cfg = dgm.CacheCfg(type=dgm.DGM_TYPE_BF16, KVH=2, D=64, pageSize=16, numPages=total, maxPages=pages.shape[1])
    k, v = (torch.randn(4, 2, 64, generator=gen, device="cuda") for _ in range(2))
    kc, vc = (torch.zeros(total, 2, 16, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want = write_ref(k, v, list(range(5)), before, pages, kc, vc, 16)
    first = write_ref(k, v, list(range(5)), [0] * 4, pages, kc, vc, 16)
    gpu.begin()
    gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, None, torch.tensor(before, dtype=torch.int32, device="cuda"), pages,
                   kc, vc, 4, 4)
    gpu.end()
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    kc.zero_()
    vc.zero_()
    gpu.begin()
    gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, None, None, pages, kc, vc, 4, 4)
    gpu.end()
    assert torch.equal(kc, first[0]) and torch.equal(vc, first[1])


def test_bad_writes_are_left_out(gpu, dgm):
    """Rows of a missing page, behind the table, before position 0: not written, the others are, and it is reported."""
    cfg = dgm.CacheCfg(type=dgm.DGM_TYPE_F32, KVH=1, D=32, pageSize=4, numPages=6, maxPages=2)
    pages = torch.tensor([[0, 1], [2, 6], [-1, 3], [4, 5]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32, device="cuda")
    lens = torch.tensor([6, 3, 3, -1], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(12, 1, 32, device="cuda") for _ in range(2))
    kc, vc = (torch.zeros(6, 1, 4, 32, device="cuda") for _ in range(2))
    want = torch.zeros_like(kc)
    for r, at in ((0, (1, 2)), (1, (1, 3)), (3, (2, 3)), (7, (3, 0)), (8, (3, 1)), (10, (4, 0)), (11, (4, 1))):
        want[at[0], 0, at[1]] = k[r, 0]
    gpu.begin()
    gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, starts, lens, pages, kc, vc, 12, 4)
    with pytest.raises(dgm.DgmError) as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    assert torch.equal(kc, want)


def test_refusals(gpu, dgm):
    cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", "f32", 4, 2, 32, 16, [5, 9])
    out = torch.full((2, 4, 32), 7.0, device="cuda")
    size = gpu.attnPagedDecode_ws_bytes(cfg, 2, 4)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    k, v = (torch.randn(2, 2, 32, device="cuda") for _ in range(2))
    kept = kc.clone()

    def status(call):
        gpu.begin()
        try:
            call()
            gpu.end()
            return dgm.DGM_OK
        except dgm.DgmError as e:
            try:
                gpu.end()
            except dgm.DgmError:
                pass
            return e.code

    def changed(change):
        c = dgm.CacheCfg.from_buffer_copy(cfg)
        for name, value in change.items():
            setattr(c, name, value)
        return c

    def dec(H=4, type=0, w=ws, size=size, ldq=0, ldo=0, scale=0.2, nseq=2, queries=q, **change):
        return status(lambda: gpu.attnPagedDecode(changed(change), type, queries, kc, vc, pages, n, out, w, size, nseq,
                                                  H, ldq, ldo, scale))

    def write(rows=2, nseq=2, ldk=0, type=0, keys=k, **change):
        return status(lambda: gpu.cacheWrite(changed(change), type, keys, v, None, None, pages, kc, vc, rows, nseq,
                                             ldk, 0))

    bad = ({"KVH": 0}, {"D": 0}, {"pageSize": 0}, {"numPages": -1}, {"maxPages": -1}, {"type": 5})
    for change in bad:
        change = dict(change)
        cache_type = change.pop("type", None)
        c = {**change, **({} if cache_type is None else {})}
        if cache_type is not None:
            broken = changed({"type": cache_type})
            assert status(lambda: gpu.attnPagedDecode(broken, 0, q, kc, vc, pages, n, out, ws, size, 2, 4)) == \
                dgm.DGM_ERR_ARG
            continue
        assert dec(**c) == write(**c) == dgm.DGM_ERR_ARG
    assert dec(type=2) == dec(H=0) == dec(nseq=-1) == dec(scale=0.0) == dec(scale=math.nan) == dgm.DGM_ERR_ARG
    assert dec(size=size - 1) == dec(w=None) == dec(queries=None) == dgm.DGM_ERR_ARG
    assert dec(H=5) == dec(ldq=64) == dec(ldo=120) == dgm.DGM_ERR_SHAPE
    assert dec(D=20) == dec(D=264) == dec(ldq=132) == dec(numPages=1 << 30) == dec(nseq=65537) == \
        dec(queries=q.data_ptr() + 4) == dgm.DGM_ERR_UNSUPPORTED
    assert write(rows=3) == write(ldk=32) == dgm.DGM_ERR_SHAPE
    assert write(rows=-1, nseq=-1) == write(keys=None) == write(type=3) == dgm.DGM_ERR_ARG
    assert write(ldk=68) == write(D=12) == write(keys=k.data_ptr() + 8) == dgm.DGM_ERR_UNSUPPORTED
    assert dec(nseq=0) == write(rows=0, nseq=0) == dgm.DGM_OK
    assert (out == 7).all() and torch.equal(kc, kept)
    assert gpu.attnPagedDecode_ws_bytes(cfg, -1, 4) == gpu.attnPagedDecode_ws_bytes(cfg, 2, 3) == -1


def test_graph_replays_with_growing_lengths(dgm, torch_cuda):
    """A captured write and decode step, replayed while the device's lengths and pages change."""
    stream = torch.cuda.Stream()
    g = dgm.GPU(stream=stream)
    try:
        with torch.cuda.stream(stream):
            cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", "bf16", 8, 2, 64, 16, [200, 3, 64])
            k, v = (torch.randn(3, 2, 64, device="cuda") for _ in range(2))
            size = g.attnPagedDecode_ws_bytes(cfg, 3, 8)
            ws, before = torch.empty(size, dtype=torch.uint8, device="cuda"), n - 1
            out, eager = torch.zeros_like(q), torch.zeros_like(q)

            def step(keys, values, to):
                g.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, None, before, pages, keys, values, 3, 3)
                g.attnPagedDecode(cfg, dgm.DGM_TYPE_F32, q, keys, values, pages, n, to, ws, size, 3, 8)

            g.begin()
            step(kc, vc, out)
            kc2, vc2 = kc.clone(), vc.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(kc, vc, out)
            for lens in ([100, 1, 20], [200, 3, 64], [7, 2, 33]):
                n.copy_(torch.tensor(lens, dtype=torch.int32))
                before.copy_(n - 1)
                q.normal_()
                k.normal_()
                out.fill_(9.0)
                graph.replay()
                step(kc2, vc2, eager)
                stream.synchronize()
                assert torch.equal(out, eager) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
            g.end()
    finally:
        g.close()


def test_reports_belong_to_their_context(gpu, dgm, torch_cuda):
    """A region's end reports what its own context found, in a replayed graph as well."""
    stream = torch.cuda.Stream()
    g = dgm.GPU(stream=stream)
    try:
        cfg, q, kc, vc, pages, n = cache_case(dgm, "f32", "f32", 4, 2, 32, 16, [40, 9])
        size = g.attnPagedDecode_ws_bytes(cfg, 2, 4)
        outs, spaces = torch.zeros(2, *q.shape, device="cuda"), torch.empty(2, size, dtype=torch.uint8, device="cuda")
        broken = pages.clone()
        torch.cuda.synchronize()

        def step(x, i, table):
            x.attnPagedDecode(cfg, dgm.DGM_TYPE_F32, q, kc, vc, table, n, outs[i], spaces[i], size, 2, 4)

        g.begin()
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(g, 0, broken)
            graph.replay()
        g.end()
        good = outs[0].clone()
        broken[0, 1] = -1
        torch.cuda.synchronize()
        for _ in range(2):
            g.begin()
            gpu.begin()
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            step(gpu, 1, pages)
            gpu.end()
            assert torch.equal(outs[1], good)
            with pytest.raises(dgm.DgmError) as e:
                g.end()
            assert e.value.code == dgm.DGM_ERR_SHAPE
            g.begin()
            g.end()
    finally:
        g.close()


def test_shared_pages(gpu, dgm):
    """Sequences with a common prompt name the same pages; one names a page twice."""
    lens = [200, 170, 96, 200]
    cfg, q, kc, vc, pages, n = cache_case(dgm, "bf16", "bf16", 8, 2, 128, 16, lens)
    pages[1, :8] = pages[0, :8]
    pages[2, :6] = pages[0, 2]
    pages[3] = pages[0]
    gpu.begin()
    out = decode(gpu, dgm, cfg, "bf16", q, kc, vc, pages, n)
    gpu.end()
    want, bound = attn_ref.decode(q, kc, vc, pages, lens, 128 ** -0.5, True)
    attn_ref.assert_within(out, want, bound)


def test_cache_beyond_32_bits(gpu, dgm):
    """Pages at the end of caches of 2^33 bytes: written, and read by the next token."""
    KVH, D, page, total, lens = 8, 128, 16, 1 << 18, [500, 37]
    gen = torch.Generator("cuda").manual_seed(9)
    kc, vc = (torch.empty(total, KVH, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert kc.numel() >= 1 << 32
    pages = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    order = total - 1 - torch.randperm(60, generator=gen, device="cuda").int()
    pages[0, :32], pages[1, :3] = order[:32], order[32:35]
    cfg = dgm.CacheCfg(type=dgm.DGM_TYPE_BF16, KVH=KVH, D=D, pageSize=page, numPages=total, maxPages=40)
    rows = sum(lens)
    k, v = (torch.randn(rows, KVH, D, generator=gen, device="cuda") for _ in range(2))
    q = torch.randn(2, 16, D, generator=gen, device="cuda")
    starts = torch.tensor([0, 500, 537], dtype=torch.int32, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    gpu.begin()
    gpu.cacheWrite(cfg, dgm.DGM_TYPE_F32, k, v, starts, None, pages, kc, vc, rows, 2)
    out = decode(gpu, dgm, cfg, "f32", q, kc, vc, pages, n)
    gpu.end()
    for s in range(2):
        pos = torch.arange(lens[s], device="cuda")
        a, b = int(starts[s]), int(starts[s + 1])
        assert torch.equal(kc[pages[s].long()[pos // page], :, pos % page], k[a:b].bfloat16())
        assert torch.equal(vc[pages[s].long()[pos // page], :, pos % page], v[a:b].bfloat16())
    want, bound = attn_ref.decode(q, kc, vc, pages, lens, D ** -0.5, False)
    attn_ref.assert_within(out, want, bound)
