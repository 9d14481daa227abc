"""The attention wrappers refuse tensors that the kernels would read as something else. No GPU: the library is a record of
its calls, the tensors CPU ones that pass for device tensors."""
from __future__ import annotations

import pytest
import torch


class Dev:
    """A CPU tensor as if on the device."""
    is_cuda = True

    def __init__(self, t):
        self.t, self.dtype = t, t.dtype

    def data_ptr(self):
        return self.t.data_ptr()

    def is_contiguous(self):
        return self.t.is_contiguous()


class Lib:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


def calls(dgm, io, cache):
    """name -> (call, its tensors' dtypes by argument name)."""
    code = {F32: dgm.DGM_TYPE_F32, BF16: dgm.DGM_TYPE_BF16}
    a = dgm.AttnCfg(type=code[io], H=2, KVH=1, D=8, causal=1, scale=1.0, rows=4, nseq=2)
    c = dgm.CacheCfg(type=code[cache], KVH=1, D=8, pageSize=4, numPages=4, maxPages=2)
    fwd = {"q": io, "k": io, "v": io, "starts": I32, "out": io, "lse": F32}
    return {
        "attnPackedFwd": (lambda g, **t: g.attnPackedFwd(a, **t), fwd),
        "attnPackedBwd": (lambda g, **t: g.attnPackedBwd(a, ws=None, ws_bytes=0, **t),
                          {**fwd, "dout": io, "dq": io, "dk": io, "dv": io}),
        "cacheWrite": (lambda g, **t: g.cacheWrite(c, code[io], rows=4, nseq=2, **t),
                       {"k": io, "v": io, "starts": I32, "lens": I32, "pages": I32, "kcache": cache, "vcache": cache}),
        "attnPagedDecode": (lambda g, **t: g.attnPagedDecode(c, code[io], ws=None, ws_bytes=0, nseq=2, H=2, **t),
                            {"q": io, "kcache": cache, "vcache": cache, "pages": I32, "lens": I32, "out": io})}


@pytest.fixture
def g(dgm):
    x = dgm.GPU.__new__(dgm.GPU)
    x.lib, x.h = Lib(), 0
    yield x
    x.h = None


NAMES = ["attnPackedFwd", "attnPackedBwd", "cacheWrite", "attnPagedDecode"]


@pytest.mark.parametrize("io,cache", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("name", NAMES)
def test_types(g, dgm, name, io, cache):
    call, types = calls(dgm, io, cache)[name]
    right = {n: Dev(torch.zeros(16, dtype=d)) for n, d in types.items()}
    call(g, **right)
    assert [n for n, _ in g.lib.calls] == ["dgm_" + name]
    addresses = [a for a in g.lib.calls[0][1] if isinstance(a, int)]
    assert all(t.data_ptr() in addresses for t in right.values())
    for n, d in types.items():
        for other in (torch.int64, torch.int32, torch.float64, torch.float16, F32, BF16):
            if other == d:
                continue
            with pytest.raises(TypeError, match=f"^{n} must be {d}, not {other}"):
                call(g, **{**right, n: Dev(torch.zeros(16, dtype=other))})
    assert len(g.lib.calls) == 1, "a refused call reached the library"


@pytest.mark.parametrize("name", NAMES)
def test_tables_are_contiguous(g, dgm, name):
    call, types = calls(dgm, F32, F32)[name]
    right = {n: Dev(torch.zeros(16, dtype=d)) for n, d in types.items()}
    for n, d in types.items():
        if d == I32:
            with pytest.raises(ValueError, match=f"^{n} must be contiguous"):
                call(g, **{**right, n: Dev(torch.zeros(2, 16, dtype=d)[:, ::2])})
    assert not g.lib.calls


@pytest.mark.parametrize("name", NAMES)
def test_addresses_and_absent_buffers_pass(g, dgm, name):
    """Raw addresses carry no type; the library refuses what is absent, and an unknown type code."""
    call, types = calls(dgm, F32, F32)[name]
    call(g, **{n: 4096 for n in types})
    call(g, **{n: None for n in types})
    assert len(g.lib.calls) == 2
    g.attnPackedFwd(dgm.AttnCfg(type=7), *[Dev(torch.zeros(4)) for _ in range(3)], Dev(torch.zeros(4, dtype=I32)),
                    Dev(torch.zeros(4)))
    assert len(g.lib.calls) == 3


def test_host_tensors_are_refused(g, dgm):
    call, types = calls(dgm, F32, F32)["attnPagedDecode"]
    with pytest.raises(ValueError, match="device memory"):
        call(g, **{n: torch.zeros(16, dtype=d) for n, d in types.items()})
    assert not g.lib.calls
