"""Layer norm with the residual sum, and its gradients, against 64 bits."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


def code(dgm, dtype):
    return dgm.DGM_TYPE_F32 if dtype == F32 else dgm.DGM_TYPE_BF16


def within(got, want, bound, dtype=F32):
    got, want = got.to(torch.float64), want.to(torch.float64)
    over = (got - want).abs() - bound - ref.half(dtype) * (want.abs() + bound)
    assert torch.isfinite(got).all() and (over <= 0).all(), f"over the bound by {over.max().item():.3g}"


def make(rows, cols, dtype, seed=0, offset=0):
    """offset: elements by which each buffer starts off a 16-byte boundary."""
    gen = torch.Generator("cuda").manual_seed(seed)

    def buf(*shape, of=dtype, scale=1.0):
        n = 1
        for s in shape:
            n *= s
        flat = torch.zeros(n + offset + 16, dtype=of, device="cuda")
        t = flat[offset:offset + n].view(*shape)
        t.copy_(torch.randn(*shape, generator=gen, device="cuda") * scale)
        return t
    x = buf(rows, cols)
    x.copy_(x.float() * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda")) + 3)
    return {"x": x, "res": buf(rows, cols), "w": 1 + 0.2 * buf(cols, of=F32), "b": buf(cols, of=F32, scale=0.3),
            "dy": buf(rows, cols), "dsum": buf(rows, cols), "sum": buf(rows, cols), "y": buf(rows, cols), "dx": buf(rows, cols),
            "mean": buf(rows, of=F32), "rstd": buf(rows, of=F32), "dw": buf(cols, of=F32), "db": buf(cols, of=F32)}


def backward(gpu, cfg, s, x, dsum, dx=None, dw=True, db=True):
    size = gpu.layerNormBwd_ws_bytes(cfg)
    ws = torch.full((size + 64,), 0x7F, dtype=torch.uint8, device="cuda")
    gpu.layerNormBwd(cfg, x, s["mean"], s["rstd"], s["w"], s["dy"], dsum, s["dx"] if dx is None else dx,
                     s["dw"] if dw else None, s["db"] if db else None, ws, size)
    gpu.end()
    gpu.begin()
    assert (ws[size:] == 0x7F).all()


# Around every border between kernels, and odd rows that start anywhere.
SIZES = [(1, 1), (3, 2), (5, 7), (17, 64), (33, 127), (1, 128), (40, 129), (7, 300), (9, 512), (6, 513), (5, 1000), (4, 1024),
         (4, 1025), (3, 2047), (3, 2048), (5, 2049), (2, 4096), (3, 4097), (2, 8191), (2, 8192), (2, 8193), (1, 16384),
         (2, 16383), (300, 12000), (700, 96), (1500, 130), (1030, 2056), (2100, 40),
         (2100, 500), (2101, 1000), (600, 2000), (300, 4096), (130, 8192)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes(dgm, gpu, torch_cuda, rows, cols, dtype):
    offset = (rows + cols) % 3
    s = make(rows, cols, dtype, rows * 7 + cols, offset)
    cfg = dgm.NormCfg(type=code(dgm, dtype), eps=EPS, rows=rows, cols=cols)
    residual = cols % 2 == 0
    gpu.begin()
    gpu.layerNormFwd(cfg, s["x"], s["res"] if residual else None, s["w"], s["b"], s["sum"] if residual else None, s["y"],
                     s["mean"], s["rstd"])
    h = s["x"]
    if residual:
        h = (s["x"].float() + s["res"].float()).to(dtype)
        assert torch.equal(s["sum"], h)
    y, mean, rstd, err, (emean, erstd) = ref.layer_norm(h, s["w"], s["b"], EPS)
    within(s["y"], y, err, dtype)
    within(s["mean"], mean, emean)
    within(s["rstd"], rstd, erstd)
    dsum = s["dsum"] if residual else None
    before = s["dw"].clone(), s["db"].clone()
    backward(gpu, cfg, s, h, dsum)
    dx, dw, db, edx, edw, edb = ref.layer_norm_bwd(h, s["mean"], s["rstd"], s["w"], s["dy"], dsum, rows + 140)
    within(s["dx"], dx, edx, dtype)
    within(s["dw"], before[0].double() + dw, edw)
    within(s["db"], before[1].double() + db, edb)
    gpu.end()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_the_optional(dgm, gpu, torch_cuda, dtype):
    s = make(9, 200, dtype, 5)
    cfg = dgm.NormCfg(type=code(dgm, dtype), eps=EPS, rows=9, cols=200)
    gpu.begin()
    gpu.layerNormFwd(cfg, s["x"], None, s["w"], None, None, s["y"])
    y, mean, rstd, err, _ = ref.layer_norm(s["x"], s["w"], None, EPS)
    within(s["y"], y, err, dtype)
    s["mean"].copy_(mean)
    s["rstd"].copy_(rstd)
    had = s["dw"].clone(), s["db"].clone()
    backward(gpu, cfg, s, s["x"], None, dw=False, db=False)
    assert torch.equal(s["dw"], had[0]) and torch.equal(s["db"], had[1])
    dx = s["dx"].clone()
    backward(gpu, cfg, s, s["x"], None, dw=False)
    assert torch.equal(s["dw"], had[0]) and not torch.equal(s["db"], had[1])
    backward(gpu, cfg, s, s["x"], None, db=False)
    assert not torch.equal(s["dw"], had[0]) and torch.equal(s["dx"], dx)
    gpu.end()


@pytest.mark.parametrize("cols", [96, 1024, 5000])
def test_in_place(dgm, gpu, torch_cuda, cols):
    """sum in x or in res, y where nothing is read any more, dx in dsum: the same bits."""
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=37, cols=cols)
    a, b, c = (make(37, cols, F32, 11) for _ in range(3))
    gpu.begin()
    gpu.layerNormFwd(cfg, a["x"], a["res"], a["w"], a["b"], a["sum"], a["y"], a["mean"], a["rstd"])
    gpu.layerNormFwd(cfg, b["x"], b["res"], b["w"], b["b"], b["x"], b["res"], b["mean"], b["rstd"])
    gpu.layerNormFwd(cfg, c["x"], c["res"], c["w"], c["b"], c["res"], c["x"], c["mean"], c["rstd"])
    assert torch.equal(a["sum"], b["x"]) and torch.equal(a["y"], b["res"])
    assert torch.equal(a["sum"], c["res"]) and torch.equal(a["y"], c["x"])
    backward(gpu, cfg, a, a["sum"], a["dsum"])
    backward(gpu, cfg, b, a["sum"], b["dsum"], dx=b["dsum"])
    assert torch.equal(a["dx"], b["dsum"]) and torch.equal(a["dw"], b["dw"])
    gpu.end()


def test_rows_that_are_not_finite_stay_alone(dgm, gpu, torch_cuda):
    for cols in (100, 700, 5000):
        s = make(6, cols, F32, 3)
        clean = s["x"].clone()
        s["x"][2, 17] = float("nan")
        s["x"][4, cols - 1] = float("inf")
        cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=6, cols=cols)
        gpu.begin()
        gpu.layerNormFwd(cfg, s["x"], None, s["w"], s["b"], None, s["y"])
        got = s["y"].clone()
        gpu.layerNormFwd(cfg, clean, None, s["w"], s["b"], None, s["y"])
        gpu.end()
        for r in range(6):
            assert torch.isnan(got[r]).any() if r in (2, 4) else torch.equal(got[r], s["y"][r])


def test_equal_elements_and_large_means(dgm, gpu, torch_cuda):
    """A row without variance gives the bias; a mean a thousand times the deviation keeps the deviation."""
    cols = 640
    s = make(4, cols, F32, 8)
    s["x"][0] = 0
    s["x"][1] = 2.5
    s["x"][2] = 1000 + s["x"][3]
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=4, cols=cols)
    gpu.begin()
    gpu.layerNormFwd(cfg, s["x"], None, s["w"], s["b"], None, s["y"], s["mean"], s["rstd"])
    gpu.end()
    assert torch.equal(s["y"][0], s["b"]) and torch.equal(s["y"][1], s["b"])
    y, _, _, err, _ = ref.layer_norm(s["x"], s["w"], s["b"], EPS)
    within(s["y"][2:], y[2:], err[2:])


@pytest.mark.parametrize("rows", [1, 77, 5000])
def test_rows_of_one_element(dgm, gpu, torch_cuda, rows):
    """The norm of one element is the bias, its gradient exactly 0 however the products round."""
    s = make(rows, 1, F32, rows)
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=rows, cols=1)
    gpu.begin()
    gpu.layerNormFwd(cfg, s["x"], None, s["w"], s["b"], None, s["y"], s["mean"], s["rstd"])
    backward(gpu, cfg, s, s["x"], None)
    gpu.end()
    assert (s["y"] == s["b"]).all() and (s["dx"] == 0).all()


def test_no_rows(dgm, gpu, torch_cuda):
    s = make(2, 64, F32)
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=0, cols=64)
    had = {k: t.clone() for k, t in s.items()}
    gpu.begin()
    gpu.layerNormFwd(cfg, s["x"], None, s["w"], s["b"], None, s["y"])
    assert gpu.layerNormBwd_ws_bytes(cfg) == 0
    gpu.layerNormBwd(cfg, s["x"], s["mean"], s["rstd"], s["w"], s["dy"], None, s["dx"], s["dw"], s["db"], None, 0)
    gpu.end()
    assert all(torch.equal(had[k], s[k]) for k in s)


@pytest.mark.parametrize("cols", [48, 600])
def test_gradient_against_differences(dgm, gpu, torch_cuda, cols):
    """sum of c y over all rows along a random direction of x, w and b: central differences of the kernel's forward. Of
    step h they are off by h^2 / 6 of a third derivative, and by the forward's bound over h."""
    rows, h = 3, 2.0 ** -7
    s = make(rows, cols, F32, 21)
    x = torch.randn(rows, cols, device="cuda")
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_F32, eps=EPS, rows=rows, cols=cols)
    c = s["dy"]
    dirs = [torch.randn_like(t) for t in (x, s["w"], s["b"])]

    def f(t):
        args = [a + t * d for a, d in zip((x, s["w"], s["b"]), dirs)]
        gpu.layerNormFwd(cfg, args[0], None, args[1], args[2], None, s["y"], s["mean"], s["rstd"])
        bound = (ref.layer_norm(args[0], args[1], args[2], EPS)[3] + ref.U * s["y"].abs()) * c.abs()
        # what rounding the arguments adds: half a step of each, through a map whose slopes are about rstd w
        return (s["y"].double() * c.double()).sum().item(), bound.sum().item() + 8 * ref.U * c.abs().sum().item()
    gpu.begin()
    (up, eu), (down, ed), (wide_up, _), (wide_down, _) = f(h), f(-h), f(2 * h), f(-2 * h)
    f(0.0)
    s["dw"].zero_()
    s["db"].zero_()
    backward(gpu, cfg, s, x, None)
    gpu.end()
    slope = sum((g.double() * d.double()).sum().item() for g, d in zip((s["dx"], s["dw"], s["db"]), dirs))
    diff, wide = (up - down) / (2 * h), (wide_up - wide_down) / (4 * h)
    # wide - diff = 3 h^2 / 6 f''' and more of higher order, diff - slope = h^2 / 6 f'''
    assert abs(diff - slope) <= abs(wide - diff) + (eu + ed) / (2 * h)


@pytest.mark.parametrize("cols,rows", [(16384, 131080), (200, 10737500)])
def test_offsets_beyond_32_bits(dgm, gpu, torch_cuda, cols, rows):
    """The last rows of more than 2^31 elements are those of a call on them alone, and the sums of all rows count them."""
    s = make(4, cols, BF16, 2)
    x, dy = (torch.zeros(rows, cols, dtype=BF16, device="cuda") for _ in range(2))
    x[-4:], dy[-4:] = s["x"], s["dy"]
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    cfg, few = (dgm.NormCfg(type=dgm.DGM_TYPE_BF16, eps=EPS, rows=n, cols=cols) for n in (rows, 4))
    s["dw"].zero_()
    s["db"].zero_()
    gpu.begin()
    gpu.layerNormFwd(few, s["x"], None, s["w"], s["b"], None, s["y"], s["mean"], s["rstd"])
    gpu.layerNormFwd(cfg, x, None, s["w"], s["b"], None, y, mean, rstd)
    backward(gpu, few, s, s["x"], None)
    dw, db = s["dw"].clone(), s["db"].clone()
    assert torch.equal(y[-4:], s["y"]) and torch.equal(mean[-4:], s["mean"]) and torch.equal(rstd[-4:], s["rstd"])
    whole = {**s, "mean": mean, "rstd": rstd, "dy": dy, "dx": dx}
    s["dw"].zero_()
    s["db"].zero_()
    backward(gpu, cfg, whole, x, None)
    gpu.end()
    assert torch.equal(dx[-4:], s["dx"]) and not dx[:100].any()
    _, edw, edb = ref.layer_norm_bwd(s["x"], s["mean"], s["rstd"], s["w"], s["dy"], None, 300)[3:]
    within(s["dw"], dw, 2 * edw)
    within(s["db"], db, 2 * edb)


def test_repeats_streams_and_graphs(dgm, gpu, torch_cuda):
    """The same bits on a stream of its own, and from every replay of a graph with other rows between."""
    rows, cols = 900, 768
    s = make(rows, cols, BF16, 4)
    cfg = dgm.NormCfg(type=dgm.DGM_TYPE_BF16, eps=EPS, rows=rows, cols=cols)
    size = dgm.GPU.layerNormBwd_ws_bytes(gpu, cfg)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)

    def step(g):
        s["dw"].zero_()
        s["db"].zero_()
        g.layerNormFwd(cfg, s["x"], s["res"], s["w"], s["b"], s["sum"], s["y"], s["mean"], s["rstd"])
        g.layerNormBwd(cfg, s["sum"], s["mean"], s["rstd"], s["w"], s["dy"], s["dsum"], s["dx"], s["dw"], s["db"], ws, size)
        return [s[k].clone() for k in ("sum", "y", "mean", "rstd", "dx", "dw", "db")]
    gpu.begin()
    first = step(gpu)
    gpu.end()
    torch.cuda.synchronize()
    own.begin()
    with torch.cuda.stream(side):
        second = step(own)
    own.end()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    own.begin()
    with torch.cuda.graph(graph, stream=side):
        out = step(own)
    kept = s["x"].clone()
    for i in range(4):
        s["x"].copy_(kept.float() * (1 + i % 2))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        own.end()
        own.begin()
        with torch.cuda.stream(side):
            eager = step(own)
        own.end()
        own.begin()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))
        assert all(torch.equal(a, b) for a, b in zip(replayed, first)) == (i % 2 == 0)
    own.end()
    own.close()


def test_refusals(dgm, gpu, torch_cuda):
    s = make(4, 64, F32)

    def cfg(**over):
        return dgm.NormCfg(**{**dict(type=dgm.DGM_TYPE_F32, eps=EPS, rows=4, cols=64), **over})
    addr = {k: t.data_ptr() for k, t in s.items()}

    def refused(status, c, fwd={}, bwd={}, ws=1 << 20):
        buf = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
        for direction, over in (("fwd", fwd), ("bwd", bwd)):
            if over is None:
                continue
            a = {**addr, **over}
            gpu.begin()
            with pytest.raises(dgm.DgmError) as e:
                if direction == "fwd":
                    gpu.layerNormFwd(c, a["x"], a["res"], a["w"], a["b"], a["sum"], a["y"], a["mean"], a["rstd"])
                else:
                    gpu.layerNormBwd(c, a["x"], a["mean"], a["rstd"], a["w"], a["dy"], a["dsum"], a["dx"], a["dw"], a["db"],
                                     over.get("ws", buf.data_ptr()), ws)
            assert e.value.code == status
            with pytest.raises(dgm.DgmError):
                gpu.end()
    refused(dgm.DGM_ERR_ARG, cfg(type=5))
    refused(dgm.DGM_ERR_ARG, cfg(rows=-1))
    refused(dgm.DGM_ERR_ARG, cfg(cols=0))
    refused(dgm.DGM_ERR_ARG, cfg(eps=-1.0))
    refused(dgm.DGM_ERR_ARG, cfg(eps=float("nan")))
    refused(dgm.DGM_ERR_UNSUPPORTED, cfg(cols=16385))
    refused(dgm.DGM_ERR_UNSUPPORTED, cfg(rows=1 << 31))
    for k in ("x", "w", "y", "sum", "res"):
        refused(dgm.DGM_ERR_ARG, cfg(), fwd={k: None}, bwd=None)
    for k in ("x", "w", "dy", "dx", "mean", "rstd"):
        refused(dgm.DGM_ERR_ARG, cfg(), fwd=None, bwd={k: None})
    large = cfg(rows=3000)          # whose sums go through the workspace
    refused(dgm.DGM_ERR_ARG, large, fwd=None, bwd={"ws": None})
    refused(dgm.DGM_ERR_ARG, large, fwd=None, ws=gpu.layerNormBwd_ws_bytes(large) - 1)
    for k in ("x", "w", "y", "sum", "res", "mean", "b"):
        refused(dgm.DGM_ERR_UNSUPPORTED, cfg(), fwd={k: addr[k] + 2}, bwd=None)
    for k in ("x", "dy", "dx", "dsum", "dw", "db", "mean", "rstd"):
        refused(dgm.DGM_ERR_UNSUPPORTED, cfg(), fwd=None, bwd={k: addr[k] + 2})
    for k in ("x", "dy"):
        refused(dgm.DGM_ERR_ARG, cfg(), fwd=None, bwd={"dx": addr[k]})
    refused(dgm.DGM_ERR_ARG, cfg(), fwd=None, bwd={"dw": addr["db"]})
    refused(dgm.DGM_ERR_ARG, cfg(), fwd={"sum": addr["y"]}, bwd=None)
    refused(dgm.DGM_ERR_ARG, cfg(), fwd={"mean": addr["rstd"]}, bwd=None)
    with pytest.raises(dgm.DgmError) as e:      # no open region
        gpu.layerNormFwd(cfg(), s["x"], None, s["w"], None, None, s["y"])
    assert e.value.code == dgm.DGM_ERR_NOT_BEGUN
