"""AdamW over many tensors at once: in 32 bits the single calls' bits, in 8 bits numpy's with borders in 64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import step_ref as ref

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, b1=0.9, b2=0.95, eps=1e-8, wd=0.1, invBC1=1.25, invBC2=1.0625)
# One element, ends of lanes (8), blocks (256) and chunks (2048), several chunks, nothing.
SIZES = [1, 2, 7, 8, 9, 255, 256, 257, 0, 2047, 2048, 2049, 5000, 8192, 40001, 3]


def buffers(n, dtype, offset, fill):
    """A buffer of n elements that starts `offset` elements off a 16-byte boundary, with guards."""
    flat = torch.full((n + offset + 32,), fill, dtype=dtype, device="cuda")
    return flat, flat[offset:offset + n]


class Tensors:
    def __init__(self, dgm, sizes, offsets, state=32, codes=()):
        gen = torch.Generator("cuda").manual_seed(sum(sizes) + len(sizes))
        self.list, self.guards, self.state = [], [], state
        for i, n in enumerate(sizes):
            off = offsets[i % len(offsets)]
            t = {"n": n, "decay": i % 2 == 0}

            def buf(name, dtype, count, fill=9):
                flat, t[name] = buffers(count, dtype, off, fill)
                self.guards.append((flat, off, count, fill))
            for name in ("w", "g"):
                buf(name, torch.float32, n)
                t[name].copy_(torch.randn(n, generator=gen, device="cuda") * (0.1 if name == "w" else 1e-2 * 4.0 ** (i % 5)))
            if n > 600:
                t["g"][256:512] = 0
            blocks = -(-n // 256)
            if state == 32:
                buf("m", torch.float32, n)
                buf("v", torch.float32, n)
                t["m"].copy_(torch.randn(n, generator=gen, device="cuda") * 1e-2)
                t["v"].copy_(torch.rand(n, generator=gen, device="cuda") * 1e-4)
            else:
                buf("m", torch.int8, n)
                buf("v", torch.uint8, n)
                buf("ms", torch.float32, blocks)
                buf("vs", torch.float32, blocks)
                t["m"].copy_(torch.randint(-127, 128, (n,), generator=gen, device="cuda"))
                t["v"].copy_(torch.randint(0, 256, (n,), generator=gen, device="cuda"))
                t["ms"].copy_(torch.rand(blocks, generator=gen, device="cuda") * 1e-6)
                t["vs"].copy_(torch.rand(blocks, generator=gen, device="cuda") * 1e-6)
                if blocks > 2:
                    t["ms"][2] = t["vs"][2] = 0     # nothing yet
            if i < len(codes) and codes[i]:
                bits, G = codes[i]
                buf("q", torch.uint8 if bits == 4 else torch.int8, n * bits // 8)
                buf("s", torch.float32, n // G)
                t["bits"], t["G"] = bits, G
            self.list.append(t)
        self.dgm = dgm

    def tensors(self):
        return [self.dgm.adam_tensor(t["w"], t["g"], t["m"], t["v"], t.get("ms"), t.get("vs"), decay=t["decay"], q=t.get("q"),
                                     scale=t.get("s"), bits=t.get("bits", 0), qGroup=t.get("G", 0)) for t in self.list]

    def copies(self):
        return [{k: x.clone() if isinstance(x, torch.Tensor) else x for k, x in t.items()} for t in self.list]

    def check_guards(self):
        for flat, off, count, fill in self.guards:
            assert (flat[:off] == fill).all() and (flat[off + count:] == fill).all()


@pytest.mark.parametrize("offsets", [[0], [1, 0, 2, 3], [3]])
def test_32_bits_are_adam_s(dgm, gpu, torch_cuda, offsets):
    s = Tensors(dgm, SIZES, offsets)
    want = s.copies()
    plan = gpu.adamMany_plan(s.tensors())
    assert plan.tensors == len(SIZES) - 1 and plan.elements == sum(-(-n // 256) * 256 for n in SIZES)
    gpu.begin()
    for _ in range(3):
        gpu.adamMany(plan, **HYPER)
        for t in want:
            gpu.adam(t["w"], t["g"], t["m"], t["v"], t["n"], HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"],
                     HYPER["wd"] if t["decay"] else 0.0, HYPER["invBC1"], HYPER["invBC2"])
    gpu.end()
    for a, b in zip(s.list, want):
        assert all(torch.equal(a[k], b[k]) for k in ("w", "g", "m", "v"))
    s.check_guards()


@pytest.mark.parametrize("offsets", [[0], [1, 8]])
def test_codes_are_adamQuantize_s(dgm, gpu, torch_cuda, offsets):
    codes = [(8, 8), (4, 8), (8, 16), (4, 32), (8, 64), (4, 128), (8, 256), (4, 512), (8, 512), (4, 16), None, (8, 32)]
    sizes = [8 * 37, 8 * 1000, 16 * 9, 32 * 65, 64 * 100, 128 * 3, 256 * 11, 512 * 5, 512 * 17, 16 * 513, 77, 32]
    s = Tensors(dgm, sizes, offsets, codes=codes)
    want = s.copies()
    plan = gpu.adamMany_plan(s.tensors())
    gpu.begin()
    gpu.adamMany(plan, **HYPER)
    for t in want:
        args = HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], HYPER["wd"] if t["decay"] else 0.0, HYPER["invBC1"], HYPER["invBC2"]
        if "q" in t:
            gpu.adamQuantize(t["w"], t["g"], t["m"], t["v"], t["q"], t["s"], t["n"] // t["G"], t["G"], t["bits"], t["G"], *args)
        else:
            gpu.adam(t["w"], t["g"], t["m"], t["v"], t["n"], *args)
    gpu.end()
    for a, b in zip(s.list, want):
        assert all(torch.equal(a[k], b[k]) for k in ("w", "m", "v", "q", "s") if k in a)
    s.check_guards()


def pad(x):
    return np.concatenate([x, np.zeros(-len(x) % 256, x.dtype)])


def step_8(t, factor, hyper):
    """(w, codes and scales of m and v) of one tensor by numpy."""
    w, g = (pad(t[k].cpu().numpy()) for k in ("w", "g"))
    m = ref.decode_m(pad(t["m"].cpu().numpy()), t["ms"].cpu().numpy())
    v = ref.decode_v(pad(t["v"].cpu().numpy()), t["vs"].cpu().numpy())
    with np.errstate(all="ignore"):
        w, m, v = ref.adam(w, g, m, v, factor, hyper["lr"], hyper["b1"], hyper["b2"], hyper["eps"],
                           hyper["wd"] if t["decay"] else 0.0, hyper["invBC1"], hyper["invBC2"])
    m[t["n"]:] = v[t["n"]:] = 0
    return (w[:t["n"]], *ref.encode(m, False), *ref.encode(v, True))


def check_8(t, want):
    n = t["n"]
    w, cm, ms, cv, vs = want
    assert np.array_equal(t["w"].cpu().numpy(), w, equal_nan=True)
    assert np.array_equal(t["m"].cpu().numpy(), cm[:n]) and np.array_equal(t["v"].cpu().numpy(), cv[:n])
    assert np.array_equal(t["ms"].cpu().numpy(), ms, equal_nan=True) and np.array_equal(t["vs"].cpu().numpy(), vs, equal_nan=True)


@pytest.mark.parametrize("offsets", [[0], [1, 0, 8, 3]])
def test_8_bits(dgm, gpu, torch_cuda, offsets):
    s = Tensors(dgm, SIZES, offsets, state=8)
    plan = gpu.adamMany_plan(s.tensors(), 8)
    factor = torch.tensor([0.37], device="cuda")
    for turn in range(3):
        want = [step_8(t, factor.item() if turn else 1.0, HYPER) for t in s.list if t["n"]]
        gpu.begin()
        gpu.adamMany(plan, **HYPER, factor=factor if turn else None)
        gpu.end()
        for t, e in zip([t for t in s.list if t["n"]], want):
            check_8(t, e)
    s.check_guards()
    m, v = (torch.full((plan.elements,), 5.0, device="cuda") for _ in range(2))
    gpu.begin()
    gpu.adamMany_states(plan, m, v)
    gpu.end()
    at = 0
    for t in s.list:
        n = t["n"]
        if n:
            assert np.array_equal(m[at:at + n].cpu().numpy(), ref.decode_m(pad(t["m"].cpu().numpy()), t["ms"].cpu().numpy())[:n])
            assert np.array_equal(v[at:at + n].cpu().numpy(), ref.decode_v(pad(t["v"].cpu().numpy()), t["vs"].cpu().numpy())[:n])
        end = at + -(-n // 256) * 256
        assert (m[at + n:end] == 5).all() and (v[at + n:end] == 5).all()
        at = end


def test_8_bits_at_borders_and_extremes(dgm, gpu, torch_cuda):
    """Moments on the borders between codes and next to them, blocks that underflow, blocks that are not finite; b1 = b2 = 0 and g
    make them: m = g, v = g^2."""
    n = 256 * 64
    g = torch.randn(n, device="cuda").view(-1, 256)
    c = torch.arange(256, device="cuda", dtype=torch.float64)
    for k in range(20):
        top = torch.rand((), device="cuda", dtype=torch.float64) + 0.5
        g[k] = (((c.clamp(max=126) + 0.5) / 127) ** 2 * top).float()
        g[k, 200:] = -g[k, 100:156]
        g[k, 255] = top.float()
    for k in range(20, 30):
        g[k] = ((c.clamp(max=254) + 0.5) / 255).square().float()
        g[k, 255] = 1.0
    for k in range(30, 36):
        g[k] *= 2.0 ** (-100 - 6 * (k - 30))       # v far below 2^-120, m about there
    g[36] = 0
    g[37, 3], g[38, 9], g[39, 250] = float("inf"), float("nan"), -float("inf")
    g[40] = 2.0 ** -60
    g[41] = 2.0 ** -60 * (1 - 2.0 ** -24)
    g[42] = 1e25                                    # v overflows
    g[43] *= 1e-3
    g[43, 0] = 1.0
    g[44, :] = 1e-9
    g[44, 0] = 1.0                                  # codes of 0 for m, of 1 for v
    t = {"n": n, "decay": False, "w": torch.zeros(n, device="cuda"), "g": g.reshape(-1).contiguous(),
         "m": torch.zeros(n, dtype=torch.int8, device="cuda"), "v": torch.zeros(n, dtype=torch.uint8, device="cuda"),
         "ms": torch.zeros(64, device="cuda"), "vs": torch.zeros(64, device="cuda")}
    hyper = {**HYPER, "b1": 0.0, "b2": 0.0}
    want = step_8(t, 1.0, hyper)
    plan = gpu.adamMany_plan([dgm.adam_tensor(t["w"], t["g"], t["m"], t["v"], t["ms"], t["vs"], decay=False)], 8)
    gpu.begin()
    gpu.adamMany(plan, **hyper)
    gpu.end()
    check_8(t, want)
    cv = t["v"].view(-1, 256)
    assert (cv[44] >= 1).all() and (t["m"].view(-1, 256)[44, 1:] == 0).all()
    assert torch.isnan(t["ms"][37:40]).all() and torch.isnan(t["vs"][42]) and torch.isfinite(t["ms"][42])


def test_8_bit_moments_stay_near(dgm, gpu, torch_cuda):
    """Against moments of 32 bits over 50 steps of gradients that change: a code's root is within half a step, so a first
    moment of 8 bits is within (2 c + 1/2) / 127^2 ... of its block's largest each step, and errors shrink by b1 a step. Loose by
    design: 5% of a block's largest for m, 5% for the root of v."""
    n = 4096
    gen = torch.Generator("cuda").manual_seed(1)
    a = {"w": torch.zeros(n, device="cuda"), "g": torch.zeros(n, device="cuda"), "m": torch.zeros(n, dtype=torch.int8, device="cuda"),
         "v": torch.zeros(n, dtype=torch.uint8, device="cuda"), "ms": torch.zeros(16, device="cuda"), "vs": torch.zeros(16, device="cuda")}
    b = {k: torch.zeros(n, device="cuda") for k in "wmv"}
    eight = gpu.adamMany_plan([dgm.adam_tensor(a["w"], a["g"], a["m"], a["v"], a["ms"], a["vs"], decay=False)], 8)
    wide = gpu.adamMany_plan([dgm.adam_tensor(b["w"], a["g"], b["m"], b["v"], decay=False)])
    size = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for _ in range(50):
        a["g"].copy_(torch.randn(n, generator=gen, device="cuda") * size)
        gpu.begin()
        gpu.adamMany(eight, **HYPER)
        gpu.adamMany(wide, **HYPER)
        gpu.adamMany_states(eight, m, v)
        gpu.end()
    top = b["m"].abs().view(-1, 256).amax(1, keepdim=True)
    assert ((m - b["m"]).abs().view(-1, 256) <= 0.05 * top).all()
    root = b["v"].sqrt().view(-1, 256)
    assert ((v.sqrt().view(-1, 256) - root).abs() <= 0.05 * root.amax(1, keepdim=True)).all()


@pytest.mark.parametrize("state", [32, 8])
def test_norm_and_clip(dgm, gpu, torch_cuda, state):
    s = Tensors(dgm, SIZES + [700000], [0, 1], state=state)
    plan = gpu.adamMany_plan(s.tensors(), state)
    out = torch.zeros(2, device="cuda")
    norm = np.float32(np.sqrt(sum((t["g"].double() ** 2).sum().item() for t in s.list)))
    for clip, factor in ((0.5, np.float32(0.5) / (norm + np.float32(1e-6))), (1e9, 1.0), (0.0, 1.0), (-1.0, 1.0)):
        gpu.begin()
        gpu.adamMany_norm(plan, clip, out)
        gpu.end()
        got = out.cpu().numpy()
        assert abs(float(got[0]) - float(norm)) <= np.spacing(norm)
        assert abs(float(got[1]) - float(factor)) <= 2 * np.spacing(np.float32(factor)) if factor != 1 else got[1] == 1
    # The factor on the way is the factor in memory.
    other = Tensors(dgm, SIZES + [700000], [0, 1], state=state)
    gpu.begin()
    gpu.adamMany_norm(plan, 0.5, out)
    gpu.adamMany(plan, **HYPER, factor=out[1:])
    gpu.end()
    for t in other.list:
        t["g"].mul_(out[1])
    second = gpu.adamMany_plan(other.tensors(), state)
    gpu.begin()
    gpu.adamMany(second, **HYPER)
    gpu.end()
    for a, b in zip(s.list, other.list):
        assert all(torch.equal(a[k], b[k]) for k in ("w", "m", "v"))
    s.list[3]["g"][0] = float("nan")
    gpu.begin()
    gpu.adamMany_norm(plan, 0.5, out)
    gpu.end()
    assert torch.isnan(out[0]) and out[1] == 1


def test_nothing(dgm, gpu, torch_cuda):
    out = torch.full((2,), 5.0, device="cuda")
    e = torch.zeros(0, device="cuda")
    for tensors in ([], [dgm.adam_tensor(e, e, e, e, decay=True)]):
        plan = gpu.adamMany_plan(tensors)
        assert plan.chunks == 0
        gpu.begin()
        gpu.adamMany_norm(plan, 1.0, out)
        gpu.adamMany(plan, **HYPER)
        gpu.end()
        assert out.tolist() == [0.0, 1.0]


def test_many_tensors(dgm, gpu, torch_cuda):
    """A thousand tensors of a few elements to a few thousand, more chunks than the norm has workgroups."""
    sizes = [1 + (i * 7919) % 9000 for i in range(1000)]
    flat = {k: torch.randn(sum(sizes), device="cuda") for k in "wgm"}
    flat["v"] = torch.rand(sum(sizes), device="cuda")
    want = {k: x.clone() for k, x in flat.items()}
    starts = np.concatenate([[0], np.cumsum(sizes)])
    plan = gpu.adamMany_plan([dgm.adam_tensor(*(flat[k][a:a + n] for k in "wgmv"), decay=True) for a, n in zip(starts, sizes)])
    assert plan.chunks > 2048
    out = torch.zeros(2, device="cuda")
    gpu.begin()
    gpu.adamMany_norm(plan, 0.0, out)
    gpu.adamMany(plan, **HYPER)
    gpu.adam(want["w"], want["g"], want["m"], want["v"], sum(sizes), *[HYPER[k] for k in ("lr", "b1", "b2", "eps", "wd", "invBC1", "invBC2")])
    gpu.end()
    assert all(torch.equal(flat[k], want[k]) for k in "wmv")
    norm = want["g"].double().norm().item()
    assert abs(out[0].item() - norm) <= 2 * ref.U * norm


@pytest.mark.parametrize("state", [32, 8])
def test_offsets_beyond_32_bits(dgm, gpu, torch_cuda, state):
    """The last elements of a tensor of more than 2^31 are those of a small one."""
    n, few = (1 << 31) + 2048 + 77, 2048 + 77
    small = Tensors(dgm, [few], [0], state=state)
    t = small.list[0]
    big = {k: torch.zeros(n if t[k].numel() == few else -(-n // 256), dtype=t[k].dtype, device="cuda") for k in t if isinstance(t[k], torch.Tensor)}
    for k, x in big.items():
        x[-t[k].numel():] = t[k]
    plan = gpu.adamMany_plan([dgm.adam_tensor(big["w"], big["g"], big["m"], big["v"], big.get("ms"), big.get("vs"), decay=True)], state)
    one = gpu.adamMany_plan(small.tensors(), state)
    out = torch.zeros(2, 2, device="cuda")
    gpu.begin()
    for i, p in enumerate((plan, one)):
        gpu.adamMany_norm(p, 0.25, out[i])
        gpu.adamMany(p, **HYPER, factor=out[i, 1:])
    gpu.end()
    assert torch.equal(out[0], out[1])
    assert all(torch.equal(x[-t[k].numel():], t[k]) for k, x in big.items())
    assert not big["w"][:1000].any()


@pytest.mark.parametrize("state", [32, 8])
def test_graphs(dgm, gpu, torch_cuda, state):
    s, other = (Tensors(dgm, SIZES, [0, 1], state=state) for _ in range(2))
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)
    plans = [own.adamMany_plan(x.tensors(), state) for x in (s, other)]
    out = torch.zeros(2, device="cuda")
    torch.cuda.synchronize()

    def step(plan):
        own.adamMany_norm(plan, 0.1, out)
        own.adamMany(plan, **HYPER, factor=out[1:])
    own.begin()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(plans[0])
    with pytest.raises(dgm.DgmError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            try:
                own.adamMany_plan(s.tensors(), state)
            finally:
                torch.zeros(1, device="cuda").add_(1)
    assert e.value.code == dgm.DGM_ERR_UNSUPPORTED
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            step(plans[1])
        torch.cuda.synchronize()
        for a, b in zip(s.list, other.list):
            assert all(torch.equal(a[k], b[k]) for k in ("w", "m", "v"))
    with pytest.raises(dgm.DgmError):
        own.end()      # the refusal during the capture
    own.close()


def test_refusals(dgm, gpu, torch_cuda):
    base = torch.zeros(1 << 16, device="cuda")
    at = base.data_ptr()

    def tensor(**over):
        a = dict(w=at, grad=at + 4096, m=at + 8192, v=at + 12288, q=at + 16384, scale=at + 20480, n=512, decay=1, bits=0, qGroup=0)
        return dgm.AdamTensor(**{**a, **over})

    def eight(**over):
        return tensor(**{**dict(mscale=at + 24576, vscale=at + 28672), **over})

    def refused(status, tensors, state=32):
        with pytest.raises(dgm.DgmError) as e:
            gpu.adamMany_plan(tensors, state)
        assert e.value.code == status
    gpu.begin()
    for k in ("w", "grad", "m", "v"):
        refused(dgm.DGM_ERR_ARG, [tensor(**{k: None})])
        refused(dgm.DGM_ERR_UNSUPPORTED, [tensor(**{k: at + 2})])
    for k in ("mscale", "vscale"):
        refused(dgm.DGM_ERR_ARG, [eight(**{k: None})], 8)
        refused(dgm.DGM_ERR_UNSUPPORTED, [eight(**{k: at + 30001})], 8)
        refused(dgm.DGM_ERR_ARG, [tensor(**{k: at + 30000})])          # scales with moments of 32 bits
    refused(dgm.DGM_ERR_ARG, [tensor(n=-1)])
    refused(dgm.DGM_ERR_UNSUPPORTED, [tensor(n=(1 << 40) + 1)])
    refused(dgm.DGM_ERR_UNSUPPORTED, [tensor(n=1 << 40)])
    refused(dgm.DGM_ERR_BITS, [tensor()], 16)
    refused(dgm.DGM_ERR_BITS, [tensor(bits=3, qGroup=8)])
    for G in (0, 4, 24, 1024, -8):
        refused(dgm.DGM_ERR_UNSUPPORTED, [tensor(bits=8, qGroup=G)])
    refused(dgm.DGM_ERR_SHAPE, [tensor(bits=8, qGroup=8, n=500)])
    refused(dgm.DGM_ERR_ARG, [tensor(bits=8, qGroup=8, q=None)])
    refused(dgm.DGM_ERR_ARG, [tensor(bits=4, qGroup=8, scale=None)])
    refused(dgm.DGM_ERR_ARG, [tensor(), tensor()])                      # named twice
    refused(dgm.DGM_ERR_ARG, [tensor(m=at + 2044)])                     # m begins inside w
    refused(dgm.DGM_ERR_ARG, [tensor(bits=8, qGroup=8, q=at + 12288 + 2040)])
    refused(dgm.DGM_ERR_ARG, [tensor(grad=at + 2044)])                  # a gradient that a step would write to
    refused(dgm.DGM_ERR_ARG, [tensor(), tensor(w=at + 32768, grad=at + 8192 - 4, m=at + 36864, v=at + 40960)])
    gpu.adamMany_plan([tensor(m=at + 2048)])                            # next to it
    gpu.adamMany_plan([tensor(), tensor(w=at + 32768, m=at + 36864, v=at + 40960)])     # one gradient for two
    with pytest.raises(dgm.DgmError):
        gpu.end()
    plan = gpu.adamMany_plan([tensor()])
    for call in (lambda: gpu.adamMany_states(plan, base, base), lambda: gpu.adamMany_norm(plan, 1.0, None),
                 lambda: gpu.adamMany(dgm.AdamPlan(), **HYPER), lambda: gpu.adamMany(plan, **HYPER, factor=at + 2)):
        gpu.begin()
        with pytest.raises(dgm.DgmError):
            call()
        with pytest.raises(dgm.DgmError):
            gpu.end()
    gpu.begin()
    with pytest.raises(dgm.DgmError):
        gpu.adamMany_states(gpu.adamMany_plan([eight()], 8), base, base)
    with pytest.raises(dgm.DgmError):
        gpu.end()
    with pytest.raises(ValueError, match="one name"):
        dgm.AdamMany(gpu, [dgm.Param("a", 2, 8, False, True, 4, 8) for _ in range(2)])
    with pytest.raises(TypeError, match="m must be torch.float32"):
        dgm.adam_tensor(base, base, base.to(torch.int8), base, decay=True)
    with pytest.raises(ValueError, match="v holds"):
        dgm.adam_tensor(base, base, base, base[:9], decay=True)


def params(dgm, seed=0):
    out = [dgm.Param("wte", 65, 128, True, True, 4, 8), dgm.Param("ln.g", 128, 1, False, False, 4, 8),
           dgm.Param("wq", 128, 128, True, True, 8, 32), dgm.Param("odd", 30, 12, True, True, 8, 4),
           dgm.Param("fp", 77, 3, False, True, 4, 8), dgm.Param("wide", 6, 1024, True, True, 8, 1024)]
    gen = torch.Generator("cuda").manual_seed(seed)
    for p in out:
        p.w.copy_(torch.randn(p.count, generator=gen, device="cuda"))
        p.g.copy_(torch.randn(p.count, generator=gen, device="cuda"))
    return out


def test_class_against_optimizer_step(dgm, gpu, torch_cuda):
    a, b = params(dgm), params(dgm)
    many = dgm.AdamMany(gpu, a)
    for i in range(1, 4):
        dgm.optimizer_step(gpu, b, 1e-2, 0.1, 0.0, i)
        gpu.begin()
        assert many.step(1e-2, 0.1, 0.0, i) is None
        gpu.end()
        for p, q in zip(a, b):
            assert all(torch.equal(x, y) for x, y in ((p.w, q.w), (p.m, q.m), (p.v, q.v)))
            assert not p.quantized or (torch.equal(p.q, q.q) and torch.equal(p.scale, q.scale))
    # Clipped: the norms agree to fp32's sums, and what comes of them.
    norm = dgm.optimizer_step(gpu, b, 1e-2, 0.1, 0.5, 4)
    gpu.begin()
    got = many.step(1e-2, 0.1, 0.5, 4)
    gpu.end()
    assert abs(got[0].item() - norm) <= 1e-5 * norm
    for p, q in zip(a, b):
        assert torch.allclose(p.w, q.w, rtol=1e-4, atol=1e-6)


def test_class_with_8_bits(dgm, gpu, torch_cuda):
    ps = params(dgm)
    many = dgm.AdamMany(gpu, ps, 8)
    assert all(p.m is None and p.v is None for p in ps)
    before = [p.w.clone() for p in ps]
    gpu.begin()
    many.step(1e-2, 0.1, 1.0, 1)
    moments = many.moments()
    gpu.end()
    f = many.norm[1].item()
    for p, w in zip(ps, before):
        n = p.count
        want = step_8({"n": n, "decay": p.decay, "w": w[:n], "g": p.g[:n], "m": torch.zeros(n, dtype=torch.int8),
                       "v": torch.zeros(n, dtype=torch.uint8), "ms": torch.zeros(-(-n // 256)), "vs": torch.zeros(-(-n // 256))},
                      f, dict(lr=1e-2, b1=0.9, b2=0.95, eps=1e-8, wd=0.1, invBC1=dgm.bias_corrections(0.9, 0.95, 1)[0],
                              invBC2=dgm.bias_corrections(0.9, 0.95, 1)[1]))
        assert np.array_equal(p.w[:n].cpu().numpy(), want[0])
        m, v = moments[p.name]
        assert np.array_equal(m.cpu().numpy(), ref.decode_m(want[1].astype(np.int8), want[2])[:n])
        assert np.array_equal(v.cpu().numpy(), ref.decode_v(want[3].astype(np.uint8), want[4])[:n])
        if p.quantized:
            q, s = torch.zeros_like(p.q), torch.zeros_like(p.scale)
            gpu.begin()
            gpu.quantize(p.w, q, s, p.rows, p.cols, p.bits, p.qGroup)
            gpu.end()
            assert torch.equal(q, p.q) and torch.equal(s, p.scale)
