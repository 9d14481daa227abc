"""The wrappers of a training step's operators refuse tensors that the kernels would read as something else or beyond; sizes of
workspaces and refused ones, on the host. No GPU: the library is a record of its calls, the tensors CPU ones that pass for device tensors."""
from __future__ import annotations

import pytest
import torch

from test_attn_wrappers import Lib

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


class Dev:
    """A CPU tensor as if on the device."""
    is_cuda = True

    def __init__(self, t):
        self.t, self.dtype = t, t.dtype

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def g(dgm):
    x = dgm.GPU.__new__(dgm.GPU)
    x.lib, x.h = Lib(), 0
    yield x
    x.h = None


def calls(dgm, io):
    """name -> (call, {argument: (dtype, elements)})."""
    code = {F32: dgm.DGM_TYPE_F32, BF16: dgm.DGM_TYPE_BF16}[io]
    n = dgm.NormCfg(type=code, eps=1e-5, rows=3, cols=8)
    loss = dgm.LossCfg(type=code, scale=1.0, rows=3, V=7, ld=10)
    e = dgm.RowsCfg(type=code, tableType=dgm.DGM_TYPE_BF16, scale=1.0, rows=3, C=8, V=5)
    rows, col, stat = (io, 24), (F32, 8), (F32, 3)
    plan = dgm.AdamPlan(elements=512, stateBits=8)
    return {
        "layerNormFwd": (lambda g, **t: g.layerNormFwd(n, **t),
                         {"x": rows, "res": rows, "weight": col, "bias": col, "sum": rows, "y": rows, "mean": stat, "rstd": stat}),
        "layerNormBwd": (lambda g, **t: g.layerNormBwd(n, ws=None, ws_bytes=0, **t),
                         {"x": rows, "mean": stat, "rstd": stat, "weight": col, "dy": rows, "dsum": rows, "dx": rows, "dweight": col,
                          "dbias": col}),
        "crossEntropy": (lambda g, **t: g.crossEntropy(loss, **t),
                         {"logits": (io, 27), "targets": (I32, 3), "rowScale": stat, "loss": stat, "lse": stat, "dlogits": (io, 27)}),
        "embedRows": (lambda g, **t: g.embedRows(e, **t), {"tokens": (I32, 3), "table": (BF16, 40), "y": rows}),
        "embedRowsBwd": (lambda g, **t: g.embedRowsBwd(e, ws=None, ws_bytes=0, **t), {"tokens": (I32, 3), "dy": rows, "dtable": (F32, 40)}),
        "adamMany_norm": (lambda g, **t: g.adamMany_norm(plan, 1.0, **t), {"out": (F32, 2)}),
        "adamMany": (lambda g, **t: g.adamMany(plan, 0, 0, 0, 0, 0, 0, 0, **t), {"factor": (F32, 1)}),
        "adamMany_states": (lambda g, **t: g.adamMany_states(plan, **t), {"m": (F32, 512), "v": (F32, 512)})}


NAMES = ["layerNormFwd", "layerNormBwd", "crossEntropy", "embedRows", "embedRowsBwd", "adamMany_norm", "adamMany", "adamMany_states"]


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("name", NAMES)
def test_types_and_sizes(g, dgm, name, io):
    call, args = calls(dgm, io)[name]
    right = {k: Dev(torch.zeros(n, dtype=d)) for k, (d, n) in args.items()}
    call(g, **right)
    assert [n for n, _ in g.lib.calls] == ["dgm_" + name]
    passed = [a for a in g.lib.calls[0][1] if isinstance(a, int)]
    assert all(t.data_ptr() in passed for t in right.values())
    for k, (d, n) in args.items():
        for other in (torch.int64, I32, torch.float64, torch.float16, F32, BF16):
            if other != d:
                with pytest.raises(TypeError, match=f"^{k} must be {d}, not {other}"):
                    call(g, **{**right, k: Dev(torch.zeros(n, dtype=other))})
        with pytest.raises(ValueError, match=f"^{k} holds {n - 1} elements"):
            call(g, **{**right, k: Dev(torch.zeros(n - 1, dtype=d))})
        with pytest.raises(ValueError, match=f"^{k} must be contiguous"):
            call(g, **{**right, k: Dev(torch.zeros(n + 1, 2, dtype=d)[:, 0])})
        with pytest.raises(ValueError, match="device memory"):
            call(g, **{**right, k: torch.zeros(n, dtype=d)})
    assert len(g.lib.calls) == 1, "a refused call reached the library"
    call(g, **{k: 4096 for k in args})
    assert len(g.lib.calls) == 2


def test_workspaces_hold_what_is_said(g, dgm):
    for name in ("layerNormBwd", "embedRowsBwd"):
        _, args = calls(dgm, F32)[name]
        right = {k: Dev(torch.zeros(n, dtype=d)) for k, (d, n) in args.items()}
        cfg = (dgm.NormCfg(type=0, eps=0, rows=3, cols=8) if name == "layerNormBwd" else
               dgm.RowsCfg(type=0, tableType=0, scale=1.0, rows=3, C=8, V=5))
        with pytest.raises(ValueError, match="the workspace holds 96 bytes, not 97"):
            getattr(g, name)(cfg, ws=Dev(torch.zeros(24)), ws_bytes=97, **right)
    assert not g.lib.calls


def test_adam_tensor(dgm):
    def dev(n, dtype=F32):
        return Dev(torch.zeros(n, dtype=dtype))
    t = dgm.adam_tensor(dev(300), dev(300), dev(300, torch.int8), dev(300, torch.uint8), dev(2), dev(2), decay=True, q=dev(150, torch.uint8),
                        scale=dev(37), bits=4, qGroup=8)
    assert (t.n, t.decay, t.bits, t.qGroup) == (300, 1, 4, 8)
    for bad, what in ((dict(mscale=dev(1)), "mscale holds 1"), (dict(q=dev(149, torch.uint8)), "q holds 149"), (dict(scale=dev(36)), "scale holds")):
        args = {**dict(mscale=dev(2), vscale=dev(2), q=dev(150, torch.uint8), scale=dev(37)), **bad}
        with pytest.raises(ValueError, match=what):
            dgm.adam_tensor(dev(300), dev(300), dev(300, torch.int8), dev(300, torch.uint8), decay=True, bits=4, qGroup=8, **args)
    with pytest.raises(TypeError, match="v must be torch.uint8"):
        dgm.adam_tensor(dev(300), dev(300), dev(300, torch.int8), dev(300, torch.int8), dev(2), dev(2), decay=True)


def test_sizes_that_are_refused(dgm):
    import ctypes
    lib = dgm.load_library()
    by = ctypes.byref
    norm = lambda **o: lib.dgm_layerNormBwd_ws_bytes(by(dgm.NormCfg(**{**dict(type=0, eps=1e-5, rows=9, cols=64), **o})))
    assert norm(rows=5000) > 0 and norm(rows=0) == norm() == 0       # few rows: one launch, no workspace
    assert all(norm(**o) == -1 for o in (dict(type=2), dict(rows=-1), dict(cols=0), dict(cols=16385), dict(eps=-1.0), dict(rows=1 << 31)))
    emb = lambda **o: lib.dgm_embedRowsBwd_ws_bytes(by(dgm.RowsCfg(**{**dict(type=0, tableType=1, scale=1.0, rows=9, C=64, V=65), **o})))
    assert emb(rows=5000) > 0 and emb() == 0                        # few tokens of a small vocabulary: no sort
    assert all(emb(**o) == -1 for o in (dict(type=2), dict(tableType=-1), dict(rows=-1), dict(C=0), dict(V=0), dict(V=1 << 31),
                                        dict(rows=(1 << 30) + 1), dict(C=(1 << 24) + 1), dict(scale=float("inf"))))
    assert emb(rows=1 << 30, C=1 << 24) == -1 and emb(rows=(1 << 30) - 64, C=4) > 1 << 33       # more than one launch; no overflow on the way
    assert lib.dgm_gpu_device(None) == -1
    one = dgm.AdamTensor(w=4096, grad=8192, m=12288, v=16384, n=2048, decay=1)
    plan = lambda bits, t=one, n=1: lib.dgm_adamMany_plan_bytes(by(t), n, bits)
    assert plan(32) > 0 and plan(8) == -1 and plan(16) == -1 and plan(32, n=-1) == -1
    assert lib.dgm_adamMany_plan_bytes(None, 0, 32) > 0 and lib.dgm_adamMany_plan_bytes(None, 1, 32) == -1
    assert lib.dgm_layerNormBwd_ws_bytes(None) == -1 and lib.dgm_embedRowsBwd_ws_bytes(None) == -1


def test_no_context_is_an_argument_error(dgm):
    lib = dgm.load_library()
    assert lib.dgm_layerNormFwd(None, None, *[None] * 8) == dgm.DGM_ERR_ARG
    assert lib.dgm_layerNormBwd(None, None, *[None] * 10, 0) == dgm.DGM_ERR_ARG
    assert lib.dgm_crossEntropy(None, None, *[None] * 6) == dgm.DGM_ERR_ARG
    assert lib.dgm_embedRows(None, None, None, None, None) == dgm.DGM_ERR_ARG
    assert lib.dgm_embedRowsBwd(None, None, None, None, None, 0, None, 0) == dgm.DGM_ERR_ARG
    assert lib.dgm_adamMany_plan(None, None, 0, 32, None, 0, None) == dgm.DGM_ERR_ARG
    assert lib.dgm_adamMany_norm(None, None, 1.0, None) == dgm.DGM_ERR_ARG
    assert lib.dgm_adamMany(None, None, None, *[0.0] * 7) == dgm.DGM_ERR_ARG
    assert lib.dgm_adamMany_states(None, None, None, None) == dgm.DGM_ERR_ARG


def test_8_bit_codes_by_both_ways():
    """The test's own reference: a code is the nearest root, ties up; decoding and coding again changes nothing."""
    import numpy as np

    import step_ref as ref
    rng = np.random.default_rng(0)
    for second in (False, True):
        x = rng.standard_normal(256 * 40).astype(np.float32) ** (2 if second else 1)
        c, s = ref.encode(x, second)
        most, power = (255, 4) if second else (127, 2)
        top = np.abs(x).reshape(-1, 256).max(1).astype(np.float64)[:, None]
        root = (np.abs(x).reshape(-1, 256).astype(np.float64) / top) ** (1 / power) * most
        assert (np.abs(np.abs(c.reshape(-1, 256)) - root) <= 0.5 + 1e-9).mean() > 0.999     # all but 0s that v raises to 1
        again = (ref.decode_v if second else ref.decode_m)(c, s)
        assert np.array_equal(ref.encode(again, second)[0], c)


FIRST = r"""
import sys, torch
sys.path.insert(0, "tests")
from conftest import load_package
from test_step_wrappers import Dev, calls
from test_attn_wrappers import Lib
dgm = load_package()
g = dgm.GPU.__new__(dgm.GPU)
g.lib, g.h = Lib(), 0
call, args = calls(dgm, torch.float32)[sys.argv[1]]
for k in args:
    try:
        call(g, **{n: Dev(torch.zeros(c, dtype=torch.int64 if n == k else d)) for n, (d, c) in args.items()})
    except TypeError as e:
        assert str(e).startswith(k), e
    else:
        raise SystemExit(k + " passed")
    break
g.h = None
"""


@pytest.mark.parametrize("name", ["layerNormFwd", "crossEntropy", "embedRows", "embedRowsBwd", "adamMany", "adamMany_states"])
def test_the_first_call_of_a_process_looks_at_types(name):
    import subprocess
    import sys

    from conftest import REPO
    done = subprocess.run([sys.executable, "-c", FIRST, name], cwd=REPO, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr


def test_views_of_logits(g, dgm, monkeypatch):
    """Rows of a padded vocabulary may be passed as a view; one with another stride, or too small, is refused."""
    from dgm_amd import gpu as module
    z = torch.zeros(3, 10)
    monkeypatch.setattr(module, "_elements", lambda code: torch.Tensor)
    monkeypatch.setattr(module, "_typed", lambda t, kind, what: t if t is None or isinstance(t, int) else t.data_ptr())
    cfg = dgm.LossCfg(type=dgm.DGM_TYPE_F32, scale=1.0, rows=3, V=7, ld=10)
    g.crossEntropy(cfg, z[:, :7], 4096, 8192, dlogits=z)
    assert g.lib.calls[0][1][2] == z.data_ptr()
    for bad in (z[:, :6], z[:2, :7], torch.zeros(3, 11)[:, :7], torch.zeros(10, 3).t()):
        with pytest.raises(ValueError, match="^logits"):
            g.crossEntropy(cfg, bad, 4096, 8192)
    assert len(g.lib.calls) == 1


def test_structures_are_the_header_s(dgm, tmp_path):
    import ctypes
    import os
    import subprocess

    from conftest import REPO
    lines = ["#include <stddef.h>", '#include "dgm_quant.h"']
    for name, cls in (("dgm_norm_cfg", dgm.NormCfg), ("dgm_loss_cfg", dgm.LossCfg), ("dgm_rows_cfg", dgm.RowsCfg),
                      ("dgm_adam_tensor", dgm.AdamTensor), ("dgm_adam_plan", dgm.AdamPlan)):
        lines.append(f'_Static_assert(sizeof({name}) == {ctypes.sizeof(cls)}, "{name}");')
        lines += [f'_Static_assert(offsetof({name}, {f}) == {getattr(cls, f).offset}, "{name}.{f}");' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["int main(void) { return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", os.path.join(REPO, "include"), str(src)], check=True)
