"""Softmax cross-entropy and its gradient against 64 bits."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref
from test_gpu_layer_norm import BF16, F32, code, within

pytestmark = pytest.mark.gpu


def make(rows, V, dtype, seed=0, ld=0, offset=0, ignored=True):
    gen = torch.Generator("cuda").manual_seed(seed)
    ld = ld or V

    def buf():
        return torch.full((rows * ld + offset + 16,), 7.0, dtype=dtype, device="cuda")
    flat, dflat = buf(), buf()
    z = flat[offset:offset + rows * ld].view(rows, ld)
    z[:, :V] = (torch.randn(rows, V, generator=gen, device="cuda") * 3 + torch.randn(rows, 1, generator=gen, device="cuda") * 20)
    targets = torch.randint(0, V, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if ignored and rows > 2:
        targets[::5] = -1
        targets[3::7] = -100
    return {"flat": flat, "z": z, "dflat": dflat, "dz": dflat[offset:offset + rows * ld].view(rows, ld), "targets": targets,
            "loss": torch.zeros(rows + 1, device="cuda"), "lse": torch.zeros(rows + 1, device="cuda"),
            "rs": torch.rand(rows, generator=gen, device="cuda") + 0.5}


def check(dgm, gpu, s, rows, V, dtype, ld=0, row_scale=False, scale=0.37):
    cfg = dgm.LossCfg(type=code(dgm, dtype), scale=scale, rows=rows, V=V, ld=ld)
    rs = s["rs"] if row_scale else None
    gpu.begin()
    gpu.crossEntropy(cfg, s["z"][:, :V], s["targets"], s["loss"], rs, s["lse"], s["dz"][:, :V] if rows % 2 else s["dz"])
    gpu.end()
    loss, lse, dz, eloss, else_, edz = ref.cross_entropy(s["z"][:, :V], s["targets"], torch.tensor(scale).item(), rs)
    within(s["loss"][:rows], loss, eloss)
    within(s["lse"][:rows], lse, else_)
    within(s["dz"][:, :V], dz, edz, dtype)
    held = s["targets"] >= 0
    assert (s["loss"][:rows][~held] == 0).all() and (s["dz"][:, :V][~held] == 0).all()
    assert s["loss"][rows] == 0 and s["lse"][rows] == 0
    if (ld or V) > V:
        assert (s["dz"][:, V:] == 7).all()
    end = s["dz"].storage_offset() + rows * (ld or V)
    assert (s["dflat"][end:] == 7).all() and (s["dflat"][:s["dz"].storage_offset()] == 7).all()


# Around every border between kernels (16, 32, 128, 256, ... 8192 pieces of 16 bytes), odd sizes, rows that start anywhere.
SIZES = [(1, 1), (7, 2), (33, 3), (100, 64), (41, 65), (19, 127), (20, 128), (6, 129), (9, 255), (9, 257), (5, 512), (5, 513),
         (7, 1000), (6, 1024), (6, 1025), (3, 2049), (3, 4095), (3, 4097), (2, 8191), (4, 8193), (3, 16383), (3, 16385),
         (2, 32767), (2, 32769), (3, 50257), (2, 65537), (2, 100003), (1, 200001), (7, 131071), (32, 40001), (33, 40001), (40, 140001), (1200, 300), (600, 2000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", SIZES)
def test_sizes(dgm, gpu, torch_cuda, rows, V, dtype):
    check(dgm, gpu, make(rows, V, dtype, V, offset=(rows + V) % 3), rows, V, dtype, row_scale=V % 2 == 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,ld", [(50, 64), (1000, 1027), (5000, 5120), (131000, 131072), (140000, 140001)])
def test_row_strides(dgm, gpu, torch_cuda, dtype, V, ld):
    check(dgm, gpu, make(5, V, dtype, V, ld=ld), 5, V, dtype, ld=ld)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [65, 3000, 40000, 150001])
def test_in_place_and_absent_results(dgm, gpu, torch_cuda, dtype, V):
    s = make(6, V, dtype, 2)
    cfg = dgm.LossCfg(type=code(dgm, dtype), scale=0.25, rows=6, V=V)
    gpu.begin()
    gpu.crossEntropy(cfg, s["z"], s["targets"], s["loss"], None, s["lse"], s["dz"])
    loss, lse = s["loss"].clone(), s["lse"].clone()
    s["loss"].zero_()
    # Without a gradient, or with one in place, the sums may go another way: both are within the bound.
    _, _, want, eloss, else_, edz = ref.cross_entropy(s["z"], s["targets"], 0.25)
    gpu.crossEntropy(cfg, s["z"], s["targets"], s["loss"])
    within(s["loss"][:6], loss[:6], 2 * eloss)
    s["lse"].zero_()
    gpu.crossEntropy(cfg, s["z"], s["targets"], None, None, s["lse"])
    within(s["lse"][:6], lse[:6], 2 * else_)
    gpu.crossEntropy(cfg, s["z"], s["targets"], None)
    gpu.crossEntropy(cfg, s["z"], s["targets"], None, None, None, s["z"])
    gpu.end()
    within(s["z"], want, edz, dtype)
    within(s["dz"], want, edz, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [70, 900, 6000, 33000, 140000])
def test_masked_logits(dgm, gpu, torch_cuda, dtype, V):
    """-inf has probability 0 wherever it lies; a row of nothing else, of a NaN, or of +inf is not a number, and rows beside it stand.
    The type's lowest value is a number like others."""
    s = make(9, V, dtype, 6, ignored=False)
    z, inf = s["z"], float("inf")
    z[0, :V // 2] = -inf
    z[1, V // 3:] = -inf
    z[2] = -inf
    z[3, 5] = float("nan")
    z[4, V - 1] = inf
    z[5] = -inf
    z[5, V - 2] = -3
    z[6, 1:] = torch.finfo(dtype).min
    z[7] = torch.finfo(dtype).min
    for r, t in ((0, V - 1), (1, 0), (2, 1), (3, 2), (4, 3), (5, V - 2), (6, 0), (7, 4), (8, 5)):
        s["targets"][r] = t
    cfg = dgm.LossCfg(type=code(dgm, dtype), scale=1.0, rows=9, V=V)
    gpu.begin()
    gpu.crossEntropy(cfg, z, s["targets"], s["loss"], None, s["lse"], s["dz"])
    gpu.end()
    good = [0, 1, 5, 6, 7, 8]
    loss, lse, dz, eloss, else_, edz = ref.cross_entropy(z[good], s["targets"][good], 1.0)
    within(s["loss"][good], loss, eloss)
    within(s["lse"][good], lse, else_)
    within(s["dz"][good], dz, edz, dtype)
    assert s["loss"][5] == 0 and (s["dz"][5] == 0).all()
    for r in (2, 3, 4):
        assert torch.isnan(s["loss"][r]) and torch.isnan(s["dz"][r]).any()
    assert s["lse"][2] == -inf and torch.isnan(s["lse"][3]) and torch.isnan(s["lse"][4])
    # A target that is masked: an infinite loss, with the gradient of the others.
    s["targets"][0] = 0
    s["targets"][2] = s["targets"][3] = s["targets"][4] = -1      # rows that do not count, whatever they hold
    gpu.begin()
    gpu.crossEntropy(cfg, z, s["targets"], s["loss"], None, None, s["dz"])
    gpu.end()
    assert s["loss"][0] == inf and torch.isfinite(s["dz"][0]).all() and s["dz"][0, 0] == -1
    assert (s["loss"][2:5] == 0).all() and (s["dz"][2:5] == 0).all()


@pytest.mark.parametrize("V", [65, 2000, 40000, 140000])
def test_targets_beyond_the_vocabulary(dgm, gpu, torch_cuda, V):
    s = make(8, V, F32, 3, ignored=False)
    cfg = dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=1.0, rows=8, V=V)
    s["targets"][2], s["targets"][5] = V, 2 ** 31 - 1
    gpu.begin()
    gpu.crossEntropy(cfg, s["z"], s["targets"], s["loss"], None, s["lse"], s["dz"])
    with pytest.raises(dgm.DgmError, match="beyond the vocabulary") as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    t = s["targets"].clone()
    t[2] = t[5] = -1
    loss, _, dz, eloss, _, edz = ref.cross_entropy(s["z"], t, 1.0)
    within(s["loss"][:8], loss, eloss)
    within(s["dz"], dz, edz)
    gpu.begin()
    gpu.crossEntropy(cfg, s["z"], t, s["loss"])
    gpu.end()      # the report is gone


def test_large_logits(dgm, gpu, torch_cuda):
    """The loss of rows at +-1e4 and +-1e30 keeps the difference; what one adds to every logit changes nothing."""
    z = torch.randn(4, 500, device="cuda") * 4
    z = torch.stack([z[0] + 1e4, z[1] - 1e4, z[2] * 1e30, z[3]])
    t = torch.tensor([3, 4, int(z[2].argmax()), 6], dtype=torch.int32, device="cuda")
    out = [torch.zeros(4, device="cuda") for _ in range(2)] + [torch.zeros_like(z)]
    gpu.begin()
    gpu.crossEntropy(dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=1.0, rows=4, V=500), z, t, out[0], None, out[1], out[2])
    gpu.end()
    loss, lse, dz, eloss, else_, edz = ref.cross_entropy(z, t, 1.0)
    within(out[0], loss, eloss)
    within(out[1], lse, else_)
    within(out[2], dz, edz)


@pytest.mark.parametrize("V", [40, 3000])
def test_gradient_against_differences(dgm, gpu, torch_cuda, V):
    """Central differences of the summed loss along a random direction, off by a sixth of h^2 f''' (from the difference between two steps) and
    the loss's own bound over h."""
    rows, h = 4, 2.0 ** -5
    s = make(rows, V, F32, 9)
    z = torch.randn(rows, V, device="cuda") * 2
    d = torch.randn(rows, V, device="cuda")
    cfg = dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=1.0, rows=rows, V=V)
    t = s["targets"]

    def f(step):
        y = z + step * d
        gpu.crossEntropy(cfg, y, t, s["loss"], None, None, s["dz"])
        noise = ref.cross_entropy(y, t, 1.0)[3] + 2 * ref.U * y.abs().max(1).values.double()
        return s["loss"][:rows].double().sum().item(), noise.sum().item()
    gpu.begin()
    (up, eu), (down, ed), (wide_up, _), (wide_down, _) = f(h), f(-h), f(2 * h), f(-2 * h)
    f(0.0)
    gpu.end()
    diff, wide = (up - down) / (2 * h), (wide_up - wide_down) / (4 * h)
    slope = (s["dz"].double() * d.double()).sum().item()
    assert abs(diff - slope) <= abs(wide - diff) + (eu + ed) / (2 * h) + 4 * ref.U * (s["dz"].double() * d.double()).abs().sum().item()


@pytest.mark.parametrize("rows,V", [(70000, 32003), (15000, 150001), (20000000, 130)])
def test_offsets_beyond_32_bits(dgm, gpu, torch_cuda, rows, V):
    """The last rows of more than 2^31 logits are those of a call on them alone."""
    s = make(5, V, BF16, 8)
    z = torch.zeros(rows, V, dtype=BF16, device="cuda")
    z[-5:] = s["z"]
    t = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    t[-5:] = s["targets"]
    dz, loss, lse = torch.ones_like(z), torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    cfg, few = (dgm.LossCfg(type=dgm.DGM_TYPE_BF16, scale=0.5, rows=n, V=V) for n in (rows, 5))
    gpu.begin()
    gpu.crossEntropy(few, s["z"], s["targets"], s["loss"], None, s["lse"], s["dz"])
    gpu.crossEntropy(cfg, z, t, loss, None, lse, dz)
    gpu.end()
    # Rows that lie at odd elements go into pieces elsewhere, and sums of them another way.
    _, _, want, eloss, else_, edz = ref.cross_entropy(s["z"], s["targets"], 0.5)
    within(loss[-5:], s["loss"][:5], 2 * eloss)
    within(lse[-5:], s["lse"][:5], 2 * else_)
    within(dz[-5:], want, edz, BF16)
    assert not dz[:100].any() and not dz[-105:-5].any()


def test_repeats_streams_and_graphs(dgm, gpu, torch_cuda):
    rows, V = 300, 5003
    s = make(rows, V, BF16, 4)
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)
    cfg = dgm.LossCfg(type=dgm.DGM_TYPE_BF16, scale=0.5, rows=rows, V=V)

    def step(g):
        g.crossEntropy(cfg, s["z"], s["targets"], s["loss"], s["rs"], s["lse"], s["dz"])
        return [s[k].clone() for k in ("loss", "lse", "dz")]
    gpu.begin()
    first = step(gpu)
    gpu.end()
    torch.cuda.synchronize()
    own.begin()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(own)
    kept = s["z"].clone()
    for i in range(3):
        s["z"].copy_(kept * (1 + i % 2))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
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
    addr = {k: s[k].data_ptr() for k in ("z", "targets", "rs", "loss", "lse", "dz")}

    def refused(status, cfg={}, **over):
        a = {**addr, **over}
        c = dgm.LossCfg(**{**dict(type=dgm.DGM_TYPE_F32, scale=1.0, rows=4, V=64, ld=0), **cfg})
        gpu.begin()
        with pytest.raises(dgm.DgmError) as e:
            gpu.crossEntropy(c, a["z"], a["targets"], a["loss"], a["rs"], a["lse"], a["dz"])
        assert e.value.code == status
        with pytest.raises(dgm.DgmError):
            gpu.end()
    refused(dgm.DGM_ERR_ARG, dict(type=-1))
    refused(dgm.DGM_ERR_ARG, dict(rows=-1))
    refused(dgm.DGM_ERR_ARG, dict(V=0))
    refused(dgm.DGM_ERR_ARG, dict(scale=float("inf")))
    refused(dgm.DGM_ERR_SHAPE, dict(ld=63))
    refused(dgm.DGM_ERR_UNSUPPORTED, dict(rows=1 << 31))
    refused(dgm.DGM_ERR_UNSUPPORTED, dict(ld=(1 << 30) + 1))
    for k in ("z", "targets"):
        refused(dgm.DGM_ERR_ARG, **{k: None})
    refused(dgm.DGM_ERR_ARG, lse=addr["loss"])
    for k in addr:
        refused(dgm.DGM_ERR_UNSUPPORTED, **{k: addr[k] + 2})
    gpu.begin()
    gpu.crossEntropy(dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=1.0, rows=0, V=64), None, None, None)
    gpu.end()
