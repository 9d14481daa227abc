"""Reports of bad starts and pages: the region's end of the context that launched the kernels, and of no other."""
from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

from conftest import PKG_DIR
from test_gpu_attn_paged import cache_case

pytestmark = pytest.mark.gpu


class Step:
    """A decode of two sequences, whose table is right until spoil()."""

    def __init__(self, dgm, torch):
        self.dgm = dgm
        self.cfg, self.q, self.kc, self.vc, self.pages, self.n = cache_case(dgm, "f32", "f32", 4, 2, 32, 16, [40, 9])
        self.out = torch.zeros_like(self.q)
        self.ws = None

    def __call__(self, gpu):
        import torch
        if self.ws is None:
            self.ws = torch.empty(gpu.attnPagedDecode_ws_bytes(self.cfg, 2, 4), dtype=torch.uint8, device="cuda")
        gpu.attnPagedDecode(self.cfg, self.dgm.DGM_TYPE_F32, self.q, self.kc, self.vc, self.pages, self.n, self.out,
                            self.ws, self.ws.numel(), 2, 4)

    def spoil(self):
        self.pages[0, 1] = -1


def test_a_graph_that_outlives_its_context_blames_no_other(dgm, torch_cuda):
    torch = torch_cuda
    stream = torch.cuda.Stream()
    step = Step(dgm, torch)
    g = dgm.GPU(stream=stream)
    g.begin()
    step(g)
    g.end()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    g.begin()
    with torch.cuda.graph(graph, stream=stream):
        step(g)
    g.end()
    g.close()
    others = [dgm.GPU(stream=stream) for _ in range(4)]
    try:
        step.spoil()
        torch.cuda.synchronize()
        for x in others:
            x.begin()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        for x in others:
            x.end()
    finally:
        for x in others:
            x.close()


CAPTURE = """
import importlib.util, os, sys
import torch
PKG = sys.argv[1]
spec = importlib.util.spec_from_file_location("dgm_amd", os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
dgm = importlib.util.module_from_spec(spec)
sys.modules["dgm_amd"] = dgm
spec.loader.exec_module(dgm)
dgm.load_library()
x = torch.zeros(8, device="cuda")
x.add_(1)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
    x.add_(1)
    g = dgm.GPU()
    x.add_(1)
for want in (3, 5):
    graph.replay()
    torch.cuda.synchronize()
    assert (x == want).all(), x
g.begin()
g.zero(x, 8)
g.end()
assert (x == 0).all()
print("ok")
"""


def test_a_first_context_may_be_created_during_a_capture(torch_cuda):
    """The process's first context, whose words are allocated then, leaves the capture whole."""
    done = subprocess.run([sys.executable, "-c", CAPTURE, PKG_DIR], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stderr


def test_a_failed_region_leaves_no_report_behind(dgm, torch_cuda):
    """A HIP error at the region's end is what it returns; the next region begins without its reports."""
    torch = torch_cuda
    stream = torch.cuda.Stream()
    step = Step(dgm, torch)
    step.spoil()
    g = dgm.GPU(stream=stream)
    hip = ctypes.CDLL("libamdhip64.so.7")
    try:
        torch.cuda.synchronize()
        g.begin()
        step(g)
        stream.synchronize()
        assert hip.hipSetDevice(-1) != 0        # an error that waits to be asked for
        with pytest.raises(dgm.DgmError) as e:
            g.end()
        assert e.value.code == dgm.DGM_ERR_HIP
        g.begin()
        g.end()
    finally:
        g.close()
