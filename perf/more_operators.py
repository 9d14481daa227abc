"""What the operators of a training step around its linears are measured on.

The lookup of token embeddings and its gradient, layer norm with the residual
sum before it and its gradients, softmax cross-entropy with its gradient, and
AdamW over many tensors at once, with moments in 32 or 8 bits. Sizes run from the character
GPT's (16 x 64 tokens, width 128, 65 characters) to a large decoder's.

`run` computes each in its plain form, in 32 bits with elementary torch
operations, or, where `own` is set, calls the framework's operators.
listed() names the cases; draw() gives others of the same ranges.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusion-gpt-metal_amd")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
BLOCK = 256                     # elements of a tensor that share the scales of 8-bit moments
LEAST = 2.0 ** -120             # a block's largest moment below this counts as zero


def _f(x):
    """x as the fp32 number that an operator takes."""
    return float(np.float32(x))


LR, B1, B2, EPS, WD, CLIP, STEP = _f(3e-3), _f(0.9), _f(0.95), _f(1e-8), _f(0.1), 1.0, 100
REST1, REST2 = float(np.float32(1) - np.float32(B1)), float(np.float32(1) - np.float32(B2))
INV1 = float(np.float32(1) / (np.float32(1) - np.float32(B1) ** np.float32(STEP)))
INV2 = float(np.float32(1) / (np.float32(1) - np.float32(B2) ** np.float32(STEP)))
NORM_EPS = _f(1e-5)


# ---- the cases --------------------------------------------------------------


def _embed(kind, type_, table, rows, V, C, scale=1.0, add=False):
    return {"kind": kind, "type": type_, "table": table, "rows": rows, "V": V, "C": C, "scale": _f(scale), "add": add}


def _norm(kind, type_, rows, cols, residual):
    return {"kind": kind, "type": type_, "rows": rows, "cols": cols, "residual": residual}


def _loss(kind, type_, rows, V):
    return {"kind": kind, "type": type_, "rows": rows, "V": V}


def _adam(bits, sizes, clip):
    return {"kind": "adam", "bits": bits, "sizes": ",".join(str(n) for n in sizes), "clip": clip}


def _sizes(case):
    return [int(n) for n in case["sizes"].split(",")]


def _gpt(V, block, layers, C):
    """Elements of a GPT's parameters: two embeddings, per layer two norms, four attention linears and two of the MLP
    with biases, the last norm."""
    layer = [C, C] + [C * C, C] * 4 + [C, C, 4 * C * C, 4 * C, 4 * C * C, C]
    return [V * C, block * C] + layer * layers + [C, C]


def listed():
    cases = {
        # Prompts of a serving batch, 8162 tokens, into a large decoder that scales its embeddings by sqrt(width).
        "lookup_prompts_bf16": _embed("lookup", "bf16", "bf16", 8162, 50257, 4096, scale=64.0),
        # The character GPT's step: 16 x 64 characters of 65.
        "embed_gpt_f32": _embed("embed", "f32", "f32", 1024, 65, 128),
        # A training batch of a larger decoder whose head shares the table: the gradient is added to the head's.
        "embed_train_bf16": _embed("embed", "bf16", "f32", 32768, 50257, 2048, add=True),
        # One new token each of 48 sequences, fp32 rows from the linears, with the residual sum.
        "norm_step_f32": _norm("norm", "f32", 48, 4096, True),
        # The character GPT's norm in one training step.
        "norm_train_gpt_f32": _norm("norm_train", "f32", 1024, 128, False),
        # A training batch of a large decoder, with the residual sum and the gradient that comes past the norm.
        "norm_train_bf16": _norm("norm_train", "bf16", 16384, 4096, True),
        # The character GPT's loss: 65 characters.
        "loss_gpt_f32": _loss("loss", "f32", 1024, 65),
        # Texts scored in fp32, what the framework's linears produce: no gradient.
        "score_f32": _loss("score", "f32", 517, 32000),
        # The loss of a training batch over a vocabulary of odd size.
        "loss_train_bf16": _loss("loss", "bf16", 8192, 50257),
        # The character GPT's update: 68 tensors, most of them a few KB.
        "adam_gpt": _adam(32, _gpt(65, 64, 4, 128), False),
        # The update of a decoder of 24 layers of 1024, clipped, moments in 32 bits.
        "adam_decoder": _adam(32, _gpt(50257, 1024, 24, 1024), True),
        # The same with moments in 8 bits, which the caller takes as values too (a checkpoint's step).
        "adam_decoder_8bit": _adam(8, _gpt(50257, 1024, 24, 1024), True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "embed", "embed", "norm", "norm_train", "norm_train", "loss", "loss", "score", "adam",
                       "adam"])
    type_ = rng.choice(["f32", "bf16"])
    if kind in ("lookup", "embed"):
        C = rng.choice([33, 64, 100, 128, 192, 256, 512, 768, 1000, 1024, 2048, 4096, 8192])
        rows = _log(rng, 1, min(32768, (1 << 26) // C))
        V = _log(rng, 2, min(200000, (1 << 27) // C))
        return _embed(kind, type_, rng.choice(["f32", "bf16"]), rows, V, C, rng.choice([1.0, 0.5, math.sqrt(C)]),
                      rng.random() < 0.5)
    if kind in ("norm", "norm_train"):
        cols = rng.choice([_log(rng, 1, 16384), 8 * _log(rng, 1, 1024), 64 * _log(rng, 1, 128)])
        return _norm(kind, type_, _log(rng, 1, min(32768, (1 << 26) // cols)), cols, rng.random() < 0.6)
    if kind in ("loss", "score"):
        V = rng.choice([_log(rng, 2, 200000), 64 * _log(rng, 1, 2048)])
        return _loss(kind, type_, _log(rng, 1, min(16384, (1 << 28) // V)), V)
    sizes = [_log(rng, 1, 1 << 22) for _ in range(_log(rng, 1, 150))]
    return _adam(rng.choice([8, 32]), sizes, rng.random() < 0.6)


def _distinct(rows, V):
    """Different ids among `rows` of _text's, on average: the k-th has a share of log((k + 1) / k) / log(V + 1)."""
    k = np.arange(1, V + 1, dtype=np.float64)
    return int(-np.expm1(rows * np.log1p(-np.log1p(1 / k) / math.log(V + 1))).sum())


def work(case):
    kind = case["kind"]
    if kind in ("lookup", "embed"):
        rows, C, e = case["rows"], case["C"], SIZE[case["type"]]
        met = _distinct(rows, case["V"])
        n = rows * C
        size = met * C * SIZE[case["table"]] + n * e + rows * 4
        if kind == "embed":
            size += n * e + rows * 4 + (2 * met if case["add"] else case["V"]) * C * 4
        return {"bytes": size, "flops": n * (1 if kind == "lookup" else 2)}
    if kind in ("norm", "norm_train"):
        n, cols, e = case["rows"] * case["cols"], case["cols"], SIZE[case["type"]]
        size = n * e * (4 if case["residual"] else 2) + 8 * cols
        if kind == "norm_train":      # x, dy (and what came past the norm) read, dx written; the sums added to
            size += n * e * (4 if case["residual"] else 3) + 16 * cols
        return {"bytes": size, "flops": n * (8 if kind == "norm" else 22)}
    if kind in ("loss", "score"):
        n = case["rows"] * case["V"]
        return {"bytes": n * SIZE[case["type"]] * (2 if kind == "loss" else 1) + 12 * case["rows"],
                "flops": n * (8 if kind == "loss" else 4)}
    n = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 15 * n}
    return {"bytes": (12 + 2 + 2 + 8) * n + 16 * (n // BLOCK), "flops": 40 * n}


# ---- inputs -----------------------------------------------------------------


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _text(gen, rows, V):
    """Ids as a text has them: the k-th most frequent about 1 / k as often as the first, frequent ones anywhere in the
    vocabulary; the last thirtieth of the rows are padding (-1)."""
    rank = ((torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64) * math.log(V + 1)).exp() - 1).long()
    order = torch.randperm(V, generator=gen, device="cuda")
    ids = order[rank.clamp(max=V - 1)].to(torch.int32)
    if rows >= 30:
        ids[rows - rows // 30:] = -1
    return ids


def _round_up(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    if kind in ("lookup", "embed"):
        rows, V, C = case["rows"], case["V"], case["C"]
        dtype = TYPES[case["type"]]
        s["tokens"] = _text(gen, rows, V)
        s["table"] = (_randn(gen, V, C) * 0.02).to(TYPES[case["table"]])
        s["y"] = torch.zeros(rows, C, dtype=dtype, device="cuda")
        if kind == "embed":
            s["dy"] = (_randn(gen, rows, C) * 1e-3).to(dtype)
            s["dtable"] = _randn(gen, V, C) * 1e-3      # the head's gradient, or what an earlier step left
        return s
    if kind in ("norm", "norm_train"):
        rows, cols = case["rows"], case["cols"]
        dtype = TYPES[case["type"]]
        # Rows differ in size, columns in their mean, as a decoder's residual stream has them.
        x = _randn(gen, rows, cols) * torch.exp(_randn(gen, rows, 1)) + 2 * _randn(gen, cols)
        s["x"] = x.to(dtype)
        s["res"] = _randn(gen, rows, cols).to(dtype) if case["residual"] else None
        s["weight"], s["bias"] = 1 + 0.1 * _randn(gen, cols), 0.1 * _randn(gen, cols)
        s["y"] = torch.zeros_like(s["x"])
        s["sum"] = torch.zeros_like(s["x"]) if case["residual"] else None
        if kind == "norm_train":
            s["mean"], s["rstd"] = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
            s["dy"] = (_randn(gen, rows, cols) * 1e-3).to(dtype)
            s["dsum"] = (_randn(gen, rows, cols) * 1e-3).to(dtype) if case["residual"] else None
            s["dx"] = torch.zeros_like(s["x"])
            s["dweight"], s["dbias"] = torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
        return s
    if kind in ("loss", "score"):
        rows, V = case["rows"], case["V"]
        s["targets"] = _text(gen, rows, V)
        logits = _randn(gen, rows, V) * 2
        logits[torch.arange(rows, device="cuda"), s["targets"].long().clamp(min=0)] += 4    # what has been learnt
        s["logits"] = logits.to(TYPES[case["type"]])
        s["loss"], s["lse"] = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        s["scale"] = _f(1.0 / max(1, rows - rows // 30 if rows >= 30 else rows))
        s["dlogits"] = torch.zeros_like(s["logits"]) if kind == "loss" else None
        return s
    # Parameters of one store, each at a multiple of BLOCK; between them are zeros.
    sizes = _sizes(case)
    starts = np.concatenate([[0], np.cumsum([_round_up(n) for n in sizes])])
    total = int(starts[-1])
    s["sizes"], s["starts"] = sizes, starts.tolist()
    count = torch.tensor([_round_up(n) for n in sizes], device="cuda")
    at = torch.arange(total, device="cuda")
    which = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), count, output_size=total)
    used = at - torch.tensor(s["starts"][:-1], device="cuda")[which] < torch.tensor(sizes, device="cuda")[which]
    del at
    # Linears decay, norms and biases (few elements) do not; gradients differ in size from tensor to tensor.
    decay = torch.tensor([n >= 4096 for n in sizes], device="cuda")
    s["decay"] = decay.tolist()
    s["wd"] = torch.where(decay, torch.tensor(WD, device="cuda"), torch.zeros((), device="cuda"))[which]
    size = torch.exp(0.7 * _randn(gen, len(sizes)) - 8)[which] * used
    del which, used
    s["w"] = _randn(gen, total) * 0.02 * (size > 0)
    s["g"] = _randn(gen, total) * size
    # Rows of an embedding that the batch did not meet have no gradient.
    s["g"].view(-1, BLOCK)[torch.rand(total // BLOCK, generator=gen, device="cuda") < 0.05] = 0
    m, v = _randn(gen, total) * size * 0.3, (_randn(gen, total).square() * 0.5 + 0.5) * size.square()
    if case["bits"] == 8:
        s["m"], s["mscale"] = _codes_m(m)
        s["v"], s["vscale"] = _codes_v(v)
        s["mvalue"], s["vvalue"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    else:
        s["m"], s["v"] = m, v
    s["norm"] = torch.zeros(2, device="cuda")
    return s


# ---- moments in 8 bits --------------------------------------------------------
# Blocks of 256 share a scale. A first moment is c |c| times max|m| / 127^2, c = -127 .. 127; a second one the square
# of c^2 times sqrt(max v) / 255^2, c = 0 .. 255, and never 0 for what is not. Small values keep what a linear code loses.
# The code is the nearest to the fp32 moment, ties up; roots are taken in 64 bits, for those next to a border.


def _scale(most, value):
    return torch.where(most >= LEAST, value, torch.zeros_like(most)).view(-1)


def _codes_m(m):
    m = m.view(-1, BLOCK)
    most = m.abs().amax(1, keepdim=True)
    c = torch.floor(torch.sqrt(m.abs().double() / most.double()) * 127 + 0.5).float()
    c = torch.where(most >= LEAST, torch.where(m < 0, -c, c), torch.zeros((), device="cuda"))
    return c.to(torch.int8).view(-1), _scale(most, most / 16129)


def _codes_v(v):
    v = v.view(-1, BLOCK)
    most = v.amax(1, keepdim=True)
    c = torch.floor(torch.sqrt(torch.sqrt(v.double() / most.double())) * 255 + 0.5).float()
    c = torch.where(v > 0, c.clamp(min=1), c)
    c = torch.where(most >= LEAST, c, torch.zeros((), device="cuda"))
    return c.to(torch.uint8).view(-1), _scale(most, torch.sqrt(most) / 65025)


def _values_m(c, scale):
    c = c.view(-1, BLOCK).float()
    return (c * c.abs() * scale[:, None]).view(-1)


def _values_v(c, scale):
    c = c.view(-1, BLOCK).float()
    return (c * c * scale[:, None]).square().view(-1)


# ---- one pass ---------------------------------------------------------------


def _plain_embed(s):
    c = s["case"]
    ids = s["tokens"].long()
    held = (ids >= 0)[:, None]
    y = torch.where(held, s["table"][ids.clamp(min=0)].float() * c["scale"], torch.zeros((), device="cuda"))
    y = y.to(s["y"].dtype)
    if c["kind"] == "lookup":
        return y
    dy = torch.where(held, s["dy"].float(), torch.zeros((), device="cuda"))
    sums = torch.zeros_like(s["dtable"]).index_add_(0, ids.clamp(min=0), dy) * c["scale"]
    s["dtable"].copy_(s["dtable"] + sums if c["add"] else sums)
    return {"y": y, "dtable": s["dtable"]}


def _plain_norm(s):
    dtype = s["x"].dtype
    h = s["x"]
    if s["res"] is not None:
        h = (h.float() + s["res"].float()).to(dtype)
    x = h.float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt(d.square().mean(1, keepdim=True) + NORM_EPS)
    xhat = d * rstd
    y = (xhat * s["weight"] + s["bias"]).to(dtype)
    out = {"y": y} if s["res"] is None else {"y": y, "sum": h}
    if s["case"]["kind"] == "norm":
        return out
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    s["dweight"] += (dy * xhat).sum(0)
    s["dbias"] += dy.sum(0)
    return {**out, "mean": mean.view(-1), "rstd": rstd.view(-1), "dx": dx.to(dtype), "dweight": s["dweight"],
            "dbias": s["dbias"]}


def _plain_loss(s):
    z = s["logits"].float()
    ids = s["targets"].long()
    held = ids >= 0
    row = torch.arange(z.shape[0], device="cuda")
    most = z.amax(1, keepdim=True)
    p = torch.exp(z - most)
    total = p.sum(1, keepdim=True)
    lse = (torch.log(total) + most).view(-1)
    zero = torch.zeros((), device="cuda")
    loss = torch.where(held, lse - z[row, ids.clamp(min=0)], zero)
    if s["case"]["kind"] == "score":
        return {"loss": loss, "lse": lse}
    p = p / total
    p[row, ids.clamp(min=0)] -= 1.0
    p = torch.where(held[:, None], p * s["scale"], zero)
    return {"loss": loss, "lse": lse, "dlogits": p.to(s["logits"].dtype)}


def _plain_adam(s):
    c = s["case"]
    g, eight = s["g"], c["bits"] == 8
    if c["clip"]:
        norm = torch.sqrt(g.double().square().sum()).float()
        factor = torch.where(norm > CLIP, CLIP / (norm + _f(1e-6)), torch.ones((), device="cuda"))
        g = g * factor
    m = _values_m(s["m"], s["mscale"]) if eight else s["m"]
    v = _values_v(s["v"], s["vscale"]) if eight else s["v"]
    m = B1 * m + REST1 * g
    v = B2 * v + REST2 * g * g
    s["w"].sub_(LR * ((m * INV1) / (torch.sqrt(v * INV2) + EPS) + s["wd"] * s["w"]))
    if eight:
        s["m"], s["mscale"] = _codes_m(m)
        s["v"], s["vscale"] = _codes_v(v)
        m, v = _values_m(s["m"], s["mscale"]), _values_v(s["v"], s["vscale"])
    else:
        s["m"], s["v"] = m, v
    return {"w": s["w"], "m": m, "v": v, "norm": torch.stack([norm, factor])} if c["clip"] else {"w": s["w"], "m": m, "v": v}


_CONTEXT = {}


def _context():
    """The framework's package and a context on torch's stream, with its region open."""
    if not _CONTEXT:
        if "dgm_amd" not in sys.modules:
            spec = importlib.util.spec_from_file_location(
                "dgm_amd", os.path.join(PKG_DIR, "__init__.py"), submodule_search_locations=[PKG_DIR])
            mod = importlib.util.module_from_spec(spec)
            sys.modules["dgm_amd"] = mod
            spec.loader.exec_module(mod)
        _CONTEXT["dgm"] = sys.modules["dgm_amd"]
        _CONTEXT["gpu"] = _CONTEXT["dgm"].GPU(stream=torch.cuda.current_stream())
        _CONTEXT["gpu"].begin()
    return _CONTEXT["dgm"], _CONTEXT["gpu"]


def _workspace(s, size):
    if "ws" not in s:
        s["ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return s["ws"]


def _own_embed(s, dgm, gpu, code):
    c = s["case"]
    if "cfg" not in s:
        s["cfg"] = dgm.RowsCfg(type=code[c["type"]], tableType=code[c["table"]], scale=c["scale"], rows=c["rows"],
                               C=c["C"], V=c["V"])
    gpu.embedRows(s["cfg"], s["tokens"], s["table"], s["y"])
    if c["kind"] == "lookup":
        return s["y"]
    ws = s.get("ws")
    if ws is None:
        ws = _workspace(s, gpu.embedRowsBwd_ws_bytes(s["cfg"]))
    gpu.embedRowsBwd(s["cfg"], s["tokens"], s["dy"], s["dtable"], ws, ws.numel(), accumulate=c["add"])
    return {"y": s["y"], "dtable": s["dtable"]}


def _own_norm(s, dgm, gpu, code):
    c = s["case"]
    if "cfg" not in s:
        s["cfg"] = dgm.NormCfg(type=code[c["type"]], eps=NORM_EPS, rows=c["rows"], cols=c["cols"])
    gpu.layerNormFwd(s["cfg"], s["x"], s["res"], s["weight"], s["bias"], s["sum"], s["y"], s.get("mean"), s.get("rstd"))
    out = {"y": s["y"]} if s["res"] is None else {"y": s["y"], "sum": s["sum"]}
    if c["kind"] == "norm":
        return out
    ws = s.get("ws")
    if ws is None:
        ws = _workspace(s, gpu.layerNormBwd_ws_bytes(s["cfg"]))
    gpu.layerNormBwd(s["cfg"], s["x"] if s["res"] is None else s["sum"], s["mean"], s["rstd"], s["weight"], s["dy"],
                     s["dsum"], s["dx"], s["dweight"], s["dbias"], ws, ws.numel())
    return {**out, "mean": s["mean"], "rstd": s["rstd"], "dx": s["dx"], "dweight": s["dweight"], "dbias": s["dbias"]}


def _own_loss(s, dgm, gpu, code):
    c = s["case"]
    if "cfg" not in s:
        s["cfg"] = dgm.LossCfg(type=code[c["type"]], scale=s["scale"], rows=c["rows"], V=c["V"])
    gpu.crossEntropy(s["cfg"], s["logits"], s["targets"], s["loss"], lse=s["lse"], dlogits=s["dlogits"])
    if c["kind"] == "score":
        return {"loss": s["loss"], "lse": s["lse"]}
    return {"loss": s["loss"], "lse": s["lse"], "dlogits": s["dlogits"]}


def _own_adam(s, dgm, gpu):
    c = s["case"]
    eight = c["bits"] == 8
    if "plan" not in s:
        def tensor(i):
            at, n = s["starts"][i], s["sizes"][i]
            part = [s[x][at:at + n] for x in "wgmv"]
            if eight:
                part += [s[x][at // BLOCK:at // BLOCK + _round_up(n) // BLOCK] for x in ("mscale", "vscale")]
            return dgm.adam_tensor(*part, decay=s["decay"][i])
        s["plan"] = gpu.adamMany_plan([tensor(i) for i in range(len(s["sizes"]))], c["bits"])
    if c["clip"]:
        gpu.adamMany_norm(s["plan"], CLIP, s["norm"])
    gpu.adamMany(s["plan"], LR, B1, B2, EPS, WD, INV1, INV2, factor=s["norm"][1:] if c["clip"] else None)
    out = {"w": s["w"], "m": s["m"], "v": s["v"]}
    if eight:
        gpu.adamMany_states(s["plan"], s["mvalue"], s["vvalue"])
        out["m"], out["v"] = s["mvalue"], s["vvalue"]
    return {**out, "norm": s["norm"]} if c["clip"] else out


def run(state):
    kind = state["case"]["kind"]
    if own:
        dgm, gpu = _context()
        if kind == "adam":
            return _own_adam(state, dgm, gpu)
        code = {"f32": dgm.DGM_TYPE_F32, "bf16": dgm.DGM_TYPE_BF16}
        return {"lookup": _own_embed, "embed": _own_embed, "norm": _own_norm, "norm_train": _own_norm,
                "loss": _own_loss, "score": _own_loss}[kind](state, dgm, gpu, code)
    return {"lookup": _plain_embed, "embed": _plain_embed, "norm": _plain_norm, "norm_train": _plain_norm,
            "loss": _plain_loss, "score": _plain_loss, "adam": _plain_adam}[kind](state)


# ---- the definition in 64 bits ------------------------------------------------


def _exact_embed(case, s):
    f64 = torch.float64
    ids = s["tokens"].long()
    y = torch.zeros(case["rows"], case["C"], dtype=f64, device="cuda")
    met = (ids >= 0).nonzero().view(-1)
    y[met] = s["table"][ids[met]].to(f64) * case["scale"]
    if case["kind"] == "lookup":
        return y
    # Each token's rows lie together once sorted: its sum is a difference of running sums.
    dtable = s["dtable"].to(f64) if case["add"] else torch.zeros(case["V"], case["C"], dtype=f64, device="cuda")
    order = met[torch.argsort(ids[met], stable=True)]
    tokens, counts = torch.unique_consecutive(ids[order], return_counts=True)
    ends = counts.cumsum(0)
    for c0 in range(0, case["C"], 512):
        cols = slice(c0, min(c0 + 512, case["C"]))
        running = torch.nn.functional.pad(s["dy"][order, cols].to(f64).cumsum(0), (0, 0, 1, 0))
        dtable[tokens, cols] += (running[ends] - running[ends - counts]) * case["scale"]
    return {"y": y, "dtable": dtable}


def _exact_norm(case, s):
    f64 = torch.float64
    out = {}
    h = s["x"]
    if case["residual"]:
        h = (s["x"].to(f64) + s["res"].to(f64)).to(h.dtype)   # held in the rows' type, as the next layer reads it
        out["sum"] = h.to(f64)
    x = h.to(f64)
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    rstd = (var + NORM_EPS).rsqrt()
    xhat = (x - mean).mul_(rstd)
    del x
    w = s["weight"].to(f64)
    out["y"] = torch.addcmul(s["bias"].to(f64), xhat, w)
    if case["kind"] == "norm":
        return out
    dy = s["dy"].to(f64)
    n = case["cols"]
    # The Jacobian of one row: rstd (I - 1 1^T / n - xhat xhat^T / n) diag(w).
    a = dy @ w / n
    b = torch.einsum("rc,rc,c->r", dy, xhat, w) / n
    dx = rstd * (dy * w - a[:, None] - xhat * b[:, None])
    if case["residual"]:
        dx += s["dsum"].to(f64)
    return {**out, "mean": mean.view(-1), "rstd": rstd.view(-1), "dx": dx, "dweight": torch.einsum("rc,rc->c", dy, xhat),
            "dbias": torch.einsum("rc->c", dy)}


def _exact_loss(case, s):
    f64 = torch.float64
    rows, V = case["rows"], case["V"]
    loss, lse = torch.zeros(rows, dtype=f64, device="cuda"), torch.zeros(rows, dtype=f64, device="cuda")
    train = case["kind"] == "loss"
    dlogits = torch.zeros(rows, V, dtype=f64, device="cuda") if train else None
    for r0 in range(0, rows, 1024):
        r = slice(r0, min(r0 + 1024, rows))
        ids = s["targets"][r].long()
        z = s["logits"][r].to(f64)
        lse[r] = torch.logsumexp(z, 1)
        met = (ids >= 0).nonzero().view(-1)
        loss[r0 + met] = lse[r][met] - z[met, ids[met]]
        if train:
            p = torch.softmax(z, 1)
            p[met, ids[met]] -= 1
            dlogits[r0 + met] = p[met] * s["scale"]
    return {"loss": loss, "lse": lse, "dlogits": dlogits} if train else {"loss": loss, "lse": lse}


def _exact_adam(case, s):
    f64 = torch.float64
    out, g = {}, s["g"].to(f64)
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        factor = torch.clamp(CLIP / (norm + _f(1e-6)), max=1.0) if norm > CLIP else torch.ones((), dtype=f64, device="cuda")
        out["norm"] = torch.stack([norm, factor])
        g *= factor
    eight = case["bits"] == 8
    if eight:
        c = s["m"].to(f64).view(-1, BLOCK)
        m = (c.sign() * c * c * s["mscale"].to(f64)[:, None]).view(-1)
        c = s["v"].to(f64).view(-1, BLOCK)
        v = (c ** 4 * s["vscale"].to(f64).square()[:, None]).view(-1)
        del c
    else:
        m, v = s["m"].to(f64), s["v"].to(f64)
    m.mul_(B1).add_(g, alpha=REST1)
    v.mul_(B2).addcmul_(g, g, value=REST2)
    w = s["w"].to(f64)
    out["w"] = w - LR * (m * INV1 / ((v * INV2).sqrt() + EPS) + s["wd"].to(f64) * w)
    del w
    if not eight:
        return {**out, "m": m, "v": v}
    del m, v, g
    # What is coded are fp32 moments, each operation rounded, as AdamW has them in 32 bits; their codes are the largest c
    # whose border, half a code below it, they reach.
    g = s["g"] * out["norm"][1].float() if case["clip"] else s["g"]
    code = s["m"].float().view(-1, BLOCK)
    m = B1 * (code * code.abs() * s["mscale"][:, None]) + REST1 * g.view(-1, BLOCK)
    code = s["v"].float().view(-1, BLOCK)
    v = B2 * (code * code * s["vscale"][:, None]).square() + REST2 * g.view(-1, BLOCK) * g.view(-1, BLOCK)
    del code, g
    for name, x, codes, power in (("m", m, 127, 2), ("v", v, 255, 4)):
        value = torch.zeros_like(x, dtype=f64)
        for r0 in range(0, x.shape[0], 1 << 17):
            y = x[r0:r0 + (1 << 17)]
            top = y.abs().amax(1, keepdim=True).to(f64)
            share = y.abs().to(f64) / top.clamp(min=LEAST)
            border = ((torch.arange(codes, device="cuda", dtype=f64) + 0.5) / codes) ** power
            c = torch.bucketize(share, border, right=True)
            if name == "v":
                c = torch.where(y > 0, c.clamp(min=1), c)
            value[r0:r0 + (1 << 17)] = y.sign() * (c.to(f64) / codes) ** power * top * (top >= LEAST)
        out[name] = value.view(-1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("lookup", "embed"):
        return _exact_embed(case, s)
    if kind in ("norm", "norm_train"):
        return _exact_norm(case, s)
    return _exact_adam(case, s) if kind == "adam" else _exact_loss(case, s)
