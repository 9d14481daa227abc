"""Host side of the optimizer half of a training step over the C ABI.

Param mirrors the reference's parameter record (src/GPT.swift:5-36): an fp32
master w with its gradient g and Adam moments m, v, and for quantized
parameters the int8 / int4 codes q and per-group scales the forward GEMMs
read. optimizer_step() is GPT.step's update (src/GPT.swift:193-218): the
squared-gradient sums for the global-norm clip, the clip scale, AdamW on
every master and the re-quantization of the quantized ones, the last two
fused into one pass per quantized parameter (GPU.adamQuantize), which leaves
every buffer bit-identical to the reference's adam-then-quantizeAll order.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional

from .gpu import GPU, Buf, RawBuf, adam_tensor


class Param:
    """src/GPT.swift:5-36. All buffers are zero-filled device tensors."""

    def __init__(self, name: str, rows: int, cols: int, quantized: bool, decay: bool, bits: int,
                 qGroup: int, device: str = "cuda"):
        self.name, self.rows, self.cols = name, rows, cols
        self.quantized, self.decay = quantized, decay
        self.bits, self.qGroup = bits, qGroup
        n = rows * cols
        self.w, self.g, self.m, self.v = (Buf(n, device) for _ in range(4))
        self.q = self.scale = None
        if quantized:
            self.scale = Buf(rows * (cols // qGroup), device)
            self.q = RawBuf(n // 2 if bits == 4 else n, device)

    @property
    def count(self) -> int:
        return self.rows * self.cols


def bias_corrections(b1: float, b2: float, step_index: int):
    """invBC1, invBC2 of src/GPT.swift:205-206 (Float arithmetic)."""
    import numpy as np
    f = np.float32
    inv1 = f(1) / (f(1) - f(b1) ** f(step_index))
    inv2 = f(1) / (f(1) - f(b2) ** f(step_index))
    return float(inv1), float(inv2)


def zero_grads(gpu: GPU, params: Iterable[Param]) -> None:
    """src/GPT.swift:437-439 (inside an open begin()/end() region)."""
    for p in params:
        gpu.zero(p.g, p.count)


def grad_norm(gpu: GPU, params: List[Param], sumsq=None) -> float:
    """src/GPT.swift:196-204: one reduceSumsq per parameter into its slot,
    then the host sums the slots in order and takes the square root."""
    import numpy as np
    if sumsq is None:
        sumsq = Buf(len(params))
    gpu.begin()
    for i, p in enumerate(params):
        gpu.reduceSumsq(p.g, sumsq, p.count, i)
    gpu.end()
    vals = sumsq[: len(params)].cpu().numpy().astype(np.float32)
    ss = np.float32(0)
    for x in vals:
        ss = np.float32(ss + x)
    return float(np.sqrt(ss))


def optimizer_step(gpu: GPU, params: List[Param], lr: float, wd: float, clip: float, step_index: int,
                   b1: float = 0.9, b2: float = 0.95, eps: float = 1e-8, sumsq=None,
                   fused: bool = True) -> float:
    """The update of GPT.step (src/GPT.swift:193-218) after the backward has
    filled every p.g. Returns the pre-clip gradient norm. With fused=False the
    reference's dispatch order is kept literally (adam for all, then quantize
    for all quantized parameters); the results are the same bits."""
    import numpy as np
    norm = grad_norm(gpu, params, sumsq)
    inv1, inv2 = bias_corrections(b1, b2, step_index)
    gpu.begin()
    if clip > 0 and norm > clip:
        s = float(np.float32(clip) / (np.float32(norm) + np.float32(1e-6)))
        for p in params:
            gpu.scale(p.g, p.count, s)
    for p in params:
        decay = wd if p.decay else 0.0
        if fused and p.quantized and p.bits != 32:
            gpu.adamQuantize(p.w, p.g, p.m, p.v, p.q, p.scale, p.rows, p.cols, p.bits, p.qGroup, lr, b1, b2,
                             eps, decay, inv1, inv2)
        else:
            gpu.adam(p.w, p.g, p.m, p.v, p.count, lr, b1, b2, eps, decay, inv1, inv2)
    if not fused:
        for p in params:
            if p.quantized and p.bits != 32:
                gpu.quantize(p.w, p.q, p.scale, p.rows, p.cols, p.bits, p.qGroup)
    gpu.end()
    return norm


class AdamMany:
    """AdamW over all parameters in one launch (GPU.adamMany), the re-quantization of the
    quantized ones in it, the norm of all gradients and the clip's factor on the device: a
    step never waits for the host. No counterpart in the reference, which dispatches
    once a parameter; with 32-bit moments and without a clip the buffers end up the same bits as optimizer_step's.

    state_bits 8 keeps the moments as codes in self.codes, about a quarter of the memory; they start at
    zero, and the parameters' own m and v are given up (None). Its own buffers are made on the
    context's stream. Make it again if a parameter's buffers are replaced: it holds their addresses (2.5 ms for 388
    parameters), so gradients should keep theirs from step to step."""

    def __init__(self, gpu: GPU, params: Iterable[Param], state_bits: int = 32):
        import torch
        self.gpu, self.params, self.state_bits = gpu, list(params), state_bits
        self.codes, self.rest, tensors = {}, [], []
        if len({p.name for p in self.params}) < len(self.params):
            raise ValueError("two parameters have one name")
        with gpu.torch_stream():
            self.norm = Buf(2)
            for p in self.params:
                n, moments = p.count, (p.m, p.v)
                if state_bits == 8:
                    blocks = -(-n // 256)
                    moments = self.codes[p.name] = [
                        torch.zeros(max(count, 1), dtype=dtype, device=p.w.device)
                        for count, dtype in ((n, torch.int8), (n, torch.uint8), (blocks, torch.float32), (blocks, torch.float32))]
                codes, G = {}, p.qGroup
                if p.quantized and p.bits != 32:
                    if p.cols % G == 0 and 8 <= G <= 512 and G & (G - 1) == 0:
                        codes = {"q": p.q, "scale": p.scale, "bits": p.bits, "qGroup": G}
                    else:
                        self.rest.append(p)
                tensors.append(adam_tensor(p.w[:n], p.g[:n], moments[0][:n], moments[1][:n], *moments[2:], decay=p.decay, **codes))
        self.plan = gpu.adamMany_plan(tensors, state_bits)
        if state_bits == 8:
            for p in self.params:
                p.m = p.v = None

    def step(self, lr: float, wd: float, clip: float, step_index: int, b1: float = 0.9, b2: float = 0.95,
             eps: float = 1e-8):
        """One update (inside an open begin()/end() region). With clip > 0 returns the device
        tensor [norm, factor] that the next step overwrites; the gradients are scaled on the way, not in memory. The numbers
        go into the launch by value: a captured step repeats its learning rate, decay and corrections, so capture what comes before it
        and call step() between the replays."""
        inv1, inv2 = bias_corrections(b1, b2, step_index)
        factor = None
        if clip > 0:
            self.gpu.adamMany_norm(self.plan, clip, self.norm)
            factor = self.norm[1:]
        self.gpu.adamMany(self.plan, lr, b1, b2, eps, wd, inv1, inv2, factor=factor)
        for p in self.rest:
            self.gpu.quantize(p.w, p.q, p.scale, p.rows, p.cols, p.bits, p.qGroup)
        return self.norm if clip > 0 else None

    def moments(self):
        """{name: (m, v)} as fp32 tensors, for a checkpoint (inside an open region; with 8 bits what the codes stand for)."""
        if self.state_bits == 32:
            return {p.name: (p.m, p.v) for p in self.params}
        with self.gpu.torch_stream():
            m, v = Buf(self.plan.elements), Buf(self.plan.elements)
        self.gpu.adamMany_states(self.plan, m, v)
        out, at = {}, 0
        for p in self.params:
            out[p.name] = (m[at:at + p.count], v[at:at + p.count])
            at += -(-p.count // 256) * 256
        return out


__all__ = ["Param", "AdamMany", "bias_corrections", "zero_grads", "grad_norm", "optimizer_step"]
