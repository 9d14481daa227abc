"""What the attention operators are measured on.

Attention over packed sequences (forward, and a training pass with its
gradient), the write of keys and values into a paged cache, and the attention
of one new token per sequence over that cache. Sizes run from the character
GPT's (16 x 64 tokens, 4 heads of 32) to a large decoder's (32 query and 8 key
heads of 128, prompts of 8192 tokens, 48 sequences in decoding).

`run` computes each in its plain form, in 32 bits with elementary torch
operations, or, where `own` is set, calls the framework's operators.
listed() names the cases; draw() gives others of the same ranges.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

own = False

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusion-gpt-metal_amd")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases --------------------------------------------------------------


def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(case):
    return [int(t) for t in case["lens"].split(",")]


def _packed(kind, type_, H, KVH, D, lens, causal=True, fused=False):
    return {"kind": kind, "type": type_, "H": H, "KVH": KVH, "D": D, "lens": _text(lens), "causal": causal,
            "fused": fused}


def _cached(kind, type_, cache, H, KVH, D, page, lens):
    return {"kind": kind, "type": type_, "cache": cache, "H": H, "KVH": KVH, "D": D, "page": page,
            "lens": _text(lens)}


def listed():
    ragged = [1900, 1, 77, 640, 1023, 350, 64, 1280, 15, 512, 201, 900, 33, 1500, 128, 411, 760, 5, 290, 1111]
    serving = [(977 * i * i + 131 * i) % 8192 + 1 for i in range(48)]
    cases = {
        # The character GPT's batch of 16 blocks of 64 characters, scored.
        "prompt_gpt_f32": _packed("prompt", "f32", 4, 4, 32, [64] * 16),
        # Twenty prompts of a serving batch, back to back, as one fused
        # projection of q, k and v leaves them.
        "prompt_ragged_bf16": _packed("prompt", "bf16", 32, 8, 128, ragged, fused=True),
        # One long prompt of a large decoder.
        "prompt_8192_bf16": _packed("prompt", "bf16", 32, 8, 128, [8192]),
        # Documents scored in fp32, what the framework's linears produce.
        "prompt_f32": _packed("prompt", "f32", 16, 4, 64, [2048, 1000, 1531, 640], fused=True),
        # The character GPT's attention in one training step.
        "train_gpt_f32": _packed("train", "f32", 4, 4, 32, [64] * 16),
        # Four full blocks of a larger decoder in training.
        "train_8192_bf16": _packed("train", "bf16", 16, 8, 128, [2048] * 4),
        # Stories of different lengths packed into one fp32 training batch.
        "train_ragged_f32": _packed("train", "f32", 12, 4, 64, [700, 33, 1024, 1, 511, 256, 900], fused=True),
        # One sequence, one new token, after 8000.
        "decode_one_bf16": _cached("decode", "bf16", "bf16", 32, 8, 128, 16, [8000]),
        # A serving batch: 48 sequences between a few and 8192 tokens, fp32
        # queries from the linears, a bf16 cache.
        "decode_48": _cached("decode", "f32", "bf16", 32, 8, 128, 16, serving),
        # The character GPT generating 16 texts, everything in fp32.
        "decode_gpt_f32": _cached("decode", "f32", "f32", 4, 4, 32, 16, [3 + 17 * i for i in range(16)]),
        # The new tokens' keys and values of that serving batch.
        "write_step": _cached("write", "f32", "bf16", 32, 8, 128, 16, [1] * 48),
        # The keys and values of prompts, 8000 tokens and more in all.
        "write_prompts": _cached("write", "f32", "bf16", 32, 8, 128, 16, ragged[:10] + [2300]),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "write"])
    KVH = rng.choice([1, 2, 4, 8])
    H = KVH * rng.choice([1, 1, 2, 3, 4, 6, 8])
    D = rng.choice([32, 48, 64, 64, 80, 96, 128, 128] + ([] if kind == "train" else [256]))
    if kind in ("prompt", "train"):
        lens = [_log(rng, 1, 4096) for _ in range(_log(rng, 1, 24))]
        while len(lens) * H * D * max(lens) ** 2 > (1 << 34):   # the plain form pads its scores
            lens.remove(max(lens)) if len(lens) > 1 else lens.__setitem__(0, lens[0] // 2)
        return _packed(kind, rng.choice(["f32", "bf16"]), H, KVH, D, lens, rng.random() < 0.75, rng.random() < 0.5)
    page = rng.choice([8, 16, 16, 32, 64, 100])
    if kind == "write":
        lens = [1] * _log(rng, 1, 64) if rng.random() < 0.5 else [_log(rng, 1, 4096) for _ in range(_log(rng, 1, 8))]
        return _cached(kind, rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16", "bf16"]), H, KVH, D, page, lens)
    lens = [_log(rng, 1, 8192) for _ in range(_log(rng, 1, 48))]
    while len(lens) * max(lens) * KVH * D > 48 * 8192 * 8 * 128:   # and its keys
        lens.remove(max(lens)) if len(lens) > 1 else lens.__setitem__(0, lens[0] // 2)
    return _cached(kind, rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16", "bf16"]), H, KVH, D, page, lens)


def work(case):
    lens, H, KVH, D = _lens(case), case["H"], case["KVH"], case["D"]
    rows, size = sum(lens), {"f32": 4, "bf16": 2}
    if case["kind"] in ("prompt", "train"):
        e = size[case["type"]]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        qo, kv = rows * H * D * e, rows * KVH * D * e
        if case["kind"] == "prompt":
            return {"bytes": 2 * qo + 2 * kv, "flops": 4 * D * H * pairs}
        # q, k, v, dout read; out, dq, dk, dv written; two products forward, five backward.
        return {"bytes": 4 * qo + 4 * kv, "flops": 14 * D * H * pairs}
    e, c = size[case["type"]], size[case["cache"]]
    if case["kind"] == "write":
        return {"bytes": 2 * rows * KVH * D * (e + c), "flops": 0}
    return {"bytes": 2 * rows * KVH * D * c + 2 * len(lens) * H * D * e, "flops": 4 * D * H * rows}


# ---- inputs -----------------------------------------------------------------


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    lens, H, KVH, D = _lens(case), case["H"], case["KVH"], case["D"]
    rows, dtype = sum(lens), TYPES[case["type"]]
    # Heads attend more or less sharply: their queries differ in length.
    sharp = torch.linspace(0.5, 2.0, H, device="cuda")[:, None]
    s = {"case": case, "scale": D ** -0.5}
    if case["kind"] in ("prompt", "train"):
        qkv = _randn(gen, rows, H + 2 * KVH, D)
        qkv[:, :H] *= sharp
        qkv = qkv.to(dtype)
        parts = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
        s["q"], s["k"], s["v"] = parts if case["fused"] else (t.contiguous() for t in parts)
        s["starts"] = _starts(lens)
        s["maxlen"] = max(lens)
        s["out"] = torch.zeros(rows, H, D, dtype=dtype, device="cuda")
        if case["kind"] == "train":
            s["dout"] = (_randn(gen, rows, H, D) * 1e-3).to(dtype)
            s["lse"] = torch.zeros(H, rows, device="cuda")
            dqkv = torch.zeros(rows, H + 2 * KVH, D, dtype=dtype, device="cuda")
            parts = dqkv[:, :H], dqkv[:, H:H + KVH], dqkv[:, H + KVH:]
            s["dq"], s["dk"], s["dv"] = parts if case["fused"] else (t.contiguous() for t in parts)
        return s
    # The cache of a running server: pages in no order, some of them not in use.
    page, kind = case["page"], case["kind"]
    before = [(37 * i * i + 11 * i) % 500 if kind == "write" else 0 for i in range(len(lens))]
    need = [-(-(b + n) // page) for b, n in zip(before, lens)]
    total = sum(need) + 1 + sum(need) // 16
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["pages"] = table
    cache = TYPES[case["cache"]]
    if kind == "write":
        s["kcache"], s["vcache"] = (torch.zeros(total, KVH, page, D, dtype=cache, device="cuda") for _ in range(2))
        s["k"], s["v"] = (_randn(gen, rows, KVH, D).to(dtype) for _ in range(2))
        s["starts"] = _starts(lens)
        s["lens"] = torch.tensor(before, dtype=torch.int32, device="cuda")
    else:
        s["kcache"], s["vcache"] = (_randn(gen, total, KVH, page, D).to(cache) for _ in range(2))
        s["q"] = (_randn(gen, len(lens), H, D) * sharp).to(dtype)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros(len(lens), H, D, dtype=dtype, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------


def _pad(x, rows, heads, G):
    """[rows, heads, D] -> fp32 [nseq, heads / G, G * maxlen, D] by the row numbers [nseq, maxlen]."""
    n, T = rows.shape
    return x.float()[rows].view(n, T, heads // G, G, -1).permute(0, 2, 3, 1, 4).reshape(n, heads // G, G * T, -1)


def _unpad(x, inside, G):
    """The inverse, the sequences' rows alone: [nseq, KVH, G * maxlen, D] -> [rows, heads, D]."""
    n, T = inside.shape
    return x.view(n, x.shape[1], G, T, -1).permute(0, 3, 1, 2, 4).reshape(n, T, -1, x.shape[-1])[inside]


def _plain_packed(s):
    c = s["case"]
    H, KVH, T = c["H"], c["KVH"], s["maxlen"]
    G, dtype = H // KVH, s["q"].dtype
    at = torch.arange(T, device="cuda")
    starts = s["starts"].long()
    inside = at < (starts[1:] - starts[:-1])[:, None]
    rows = (starts[:-1, None] + at).clamp(max=s["q"].shape[0] - 1)
    hidden = ~inside[:, None, None, None, :]
    if c["causal"]:
        hidden = hidden | (at > at[:, None])
    q, k, v = _pad(s["q"], rows, H, G), _pad(s["k"], rows, KVH, 1), _pad(s["v"], rows, KVH, 1)
    n = q.shape[0]
    p = (q @ k.transpose(-1, -2)) * s["scale"]
    p.view(n, KVH, G, T, T).masked_fill_(hidden, float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = _unpad(p @ v, inside, G).to(dtype)
    if c["kind"] == "prompt":
        return out
    do = _pad(s["dout"], rows, H, G) * inside[:, None, None, :, None].expand(n, 1, G, T, 1).reshape(n, 1, G * T, 1)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
    dk = ds.transpose(-1, -2) @ q
    return {"out": out, "dq": _unpad(ds @ k, inside, G).to(dtype), "dk": _unpad(dk, inside, 1).to(dtype),
            "dv": _unpad(dv, inside, 1).to(dtype)}


def _plain_write(s):
    page = s["case"]["page"]
    starts = s["starts"].long()
    row = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    pos = s["lens"].long()[seq] + row - starts[seq]
    where = s["pages"].long()[seq, pos // page]
    s["kcache"][where, :, pos % page] = s["k"].to(s["kcache"].dtype)
    s["vcache"][where, :, pos % page] = s["v"].to(s["vcache"].dtype)
    return {"kcache": s["kcache"], "vcache": s["vcache"]}


def _plain_decode(s):
    c = s["case"]
    KVH, D = c["KVH"], c["D"]
    n, most = s["pages"].shape
    pages = s["pages"].long().clamp(min=0)
    k, v = (s[x][pages].float().transpose(1, 2).reshape(n, KVH, most * c["page"], D) for x in ("kcache", "vcache"))
    hidden = (torch.arange(most * c["page"], device="cuda") >= s["lens"][:, None])[:, None, None, :]
    q = s["q"].float().view(n, KVH, -1, D)
    p = ((q @ k.transpose(-1, -2)) * s["scale"]).masked_fill(hidden, float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    return ((p @ v) / p.sum(-1, keepdim=True)).view(n, -1, D).to(s["q"].dtype)


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


def _own(s):
    dgm, gpu = _context()
    c = s["case"]
    code = {"f32": dgm.DGM_TYPE_F32, "bf16": dgm.DGM_TYPE_BF16}
    if c["kind"] in ("prompt", "train"):
        if "cfg" not in s:
            s["cfg"] = dgm.AttnCfg(type=code[c["type"]], H=c["H"], KVH=c["KVH"], D=c["D"], causal=int(c["causal"]),
                                   scale=s["scale"], rows=s["q"].shape[0], nseq=s["starts"].numel() - 1,
                                   ldq=s["q"].stride(0), ldk=s["k"].stride(0), ldv=s["v"].stride(0),
                                   ldo=s["out"].stride(0))
        cfg = s["cfg"]
        gpu.attnPackedFwd(cfg, s["q"], s["k"], s["v"], s["starts"], s["out"], s.get("lse"))
        if c["kind"] == "prompt":
            return s["out"]
        if "ws" not in s:
            s["ws"] = torch.empty(gpu.attnPackedBwd_ws_bytes(cfg), dtype=torch.uint8, device="cuda")
        gpu.attnPackedBwd(cfg, s["q"], s["k"], s["v"], s["starts"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"],
                          s["dv"], s["ws"], s["ws"].numel())
        return {"out": s["out"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    if "cfg" not in s:
        s["cfg"] = dgm.CacheCfg(type=code[c["cache"]], KVH=c["KVH"], D=c["D"], pageSize=c["page"],
                                numPages=s["kcache"].shape[0], maxPages=s["pages"].shape[1])
    cfg = s["cfg"]
    if c["kind"] == "write":
        gpu.cacheWrite(cfg, code[c["type"]], s["k"], s["v"], s["starts"], s["lens"], s["pages"], s["kcache"],
                       s["vcache"], s["k"].shape[0], s["lens"].numel(), s["k"].stride(0), s["v"].stride(0))
        return {"kcache": s["kcache"], "vcache": s["vcache"]}
    n = s["lens"].numel()
    if "ws" not in s:
        s["ws"] = torch.empty(gpu.attnPagedDecode_ws_bytes(cfg, n, c["H"]), dtype=torch.uint8, device="cuda")
    gpu.attnPagedDecode(cfg, code[c["type"]], s["q"], s["kcache"], s["vcache"], s["pages"], s["lens"], s["out"],
                        s["ws"], s["ws"].numel(), n, c["H"], s["q"].stride(0), s["out"].stride(0), s["scale"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_packed, "train": _plain_packed, "write": _plain_write,
            "decode": _plain_decode}[state["case"]["kind"]](state)


# ---- the definition in 64 bits ------------------------------------------------


def exact(case, seed):
    """Sequence by sequence and key head by key head, from the formulas."""
    s = prepare(case, seed)
    lens, H, KVH, D = _lens(case), case["H"], case["KVH"], case["D"]
    G, f64 = H // KVH, torch.float64
    if case["kind"] == "write":
        at, base, page = 0, s["lens"].tolist(), case["page"]
        kc, vc = s["kcache"].to(f64), s["vcache"].to(f64)
        for i, n in enumerate(lens):
            pos = base[i] + torch.arange(n, device="cuda")
            where = s["pages"][i].long()[pos.div(page, rounding_mode="floor")]
            kc[where, :, pos.remainder(page)] = s["k"][at:at + n].to(f64)
            vc[where, :, pos.remainder(page)] = s["v"][at:at + n].to(f64)
            at += n
        return {"kcache": kc, "vcache": vc}
    if case["kind"] == "decode":
        out = torch.zeros(len(lens), H, D, dtype=f64, device="cuda")
        for i, n in enumerate(lens):
            used = s["pages"][i, :-(-n // case["page"])].long()
            keys, values = (s[x][used].to(f64).permute(1, 0, 2, 3).reshape(KVH, -1, D)[:, :n]
                            for x in ("kcache", "vcache"))
            for h in range(H):
                w = torch.softmax((keys[h // G] @ s["q"][i, h].to(f64)) * s["scale"], 0)
                out[i, h] = w @ values[h // G]
        return out
    q, k, v = (s[x].to(f64) for x in "qkv")
    out, train = torch.zeros_like(q), case["kind"] == "train"
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = 0
    for n in lens:
        r = slice(at, at + n)
        later = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else None
        for h in range(H):
            qh, kh, vh = q[r, h], k[r, h // G], v[r, h // G]
            w = torch.einsum("id,jd->ij", qh, kh).mul_(s["scale"])
            if later is not None:
                w[later] = -math.inf
            w = torch.softmax(w, 1)
            out[r, h] = torch.einsum("ij,jd->id", w, vh)
            if not train:
                continue
            g = s["dout"][r, h].to(f64)
            dv[r, h // G] += torch.einsum("ij,id->jd", w, g)
            slope = torch.einsum("id,jd->ij", g, vh)
            slope = (slope - torch.einsum("id,id->i", g, out[r, h])[:, None]).mul_(w).mul_(s["scale"])
            dq[r, h] = torch.einsum("ij,jd->id", slope, kh)
            dk[r, h // G] += torch.einsum("ij,id->jd", slope, qh)
        at += n
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else out
