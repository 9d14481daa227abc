"""Attention over packed sequences, forward and backward, against 64 bits
(attn_ref.py derives the element-wise bounds)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


class Case:
    """Inputs of packed sequences with `front` rows before the first and `back` behind the last one."""

    def __init__(self, dgm, type_, H, KVH, D, lens, causal=True, fused=False, front=0, back=0, seed=0, scale=None):
        gen = torch.Generator("cuda").manual_seed(seed + 7 * D + len(lens))
        dt, self.rows = TYPES[type_], front + sum(lens) + back
        self.lens, self.causal, self.scale = lens, causal, D ** -0.5 if scale is None else scale
        starts = [front]
        for n in lens:
            starts.append(starts[-1] + n)
        self.starts_list = starts
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        wide = torch.randn(self.rows, H + 2 * KVH, D, generator=gen, device="cuda").to(dt)
        grad = torch.full((self.rows, H + 2 * KVH, D), 7.0, device="cuda").to(dt)
        cut = lambda t: (t[:, :H], t[:, H:H + KVH], t[:, H + KVH:])  # noqa: E731
        whole = (lambda t: t) if fused else (lambda t: t.contiguous())
        self.q, self.k, self.v = (whole(t) for t in cut(wide))
        self.dq, self.dk, self.dv = (whole(t) for t in cut(grad))
        self.dout = torch.randn(self.rows, H, D, generator=gen, device="cuda").to(dt)
        self.out = torch.full((self.rows, H, D), 7.0, device="cuda").to(dt)
        self.lse = torch.full((H, self.rows), 7.0, device="cuda")
        code = dgm.DGM_TYPE_F32 if type_ == "f32" else dgm.DGM_TYPE_BF16
        self.cfg = dgm.AttnCfg(type=code, H=H, KVH=KVH, D=D, causal=int(causal), scale=self.scale, rows=self.rows,
                               nseq=len(lens), ldq=self.q.stride(0) if fused else 0, ldk=self.k.stride(0),
                               ldv=self.v.stride(0), ldo=0)

    def forward(self, gpu):
        gpu.attnPackedFwd(self.cfg, self.q, self.k, self.v, self.starts, self.out, self.lse)

    def backward(self, gpu):
        n = gpu.attnPackedBwd_ws_bytes(self.cfg)
        self.ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        gpu.attnPackedBwd(self.cfg, self.q, self.k, self.v, self.starts, self.out, self.lse, self.dout, self.dq,
                          self.dk, self.dv, self.ws, n)

    def check(self, backward):
        val, bnd = attn_ref.packed(self.q, self.k, self.v, self.starts_list, self.scale, self.causal,
                                   self.dout if backward else None)
        a, b = self.starts_list[0], self.starts_list[-1]
        for name, want in val.items():
            got = getattr(self, name)
            attn_ref.assert_within(got[a:b], want[a:b], bnd[name][a:b], name)
            assert (got[:a] == 7).all() and (got[b:] == 7).all(), f"{name}: rows of no sequence were written"


# One token up to several tiles, lengths around them, empty sequences first, last and in a row.
FORWARD = [
    ("f32", 4, 4, 32, [64] * 3, True, False, 0, 0),
    ("bf16", 4, 4, 32, [64] * 3, True, False, 0, 0),
    ("f32", 1, 1, 8, [1], True, False, 0, 0),
    ("bf16", 1, 1, 8, [1], False, False, 0, 0),
    ("f32", 4, 1, 48, [64, 64], False, False, 0, 0),
    ("f32", 6, 2, 64, [0, 5, 0, 0, 33, 1, 0], True, True, 3, 5),
    ("bf16", 6, 2, 64, [0, 5, 0, 0, 33, 1, 0], False, True, 3, 5),
    ("bf16", 8, 2, 128, [127, 129, 1, 65, 300], True, True, 0, 9),
    ("f32", 8, 2, 128, [127, 129, 1, 65, 300], True, True, 130, 0),
    ("f32", 3, 1, 80, [31, 32, 33, 257], False, False, 1, 1),
    ("bf16", 3, 1, 96, [255, 256, 257], False, False, 0, 0),
    ("bf16", 12, 1, 24, [513], True, False, 0, 0),
    ("f32", 2, 2, 128, [1000], True, False, 0, 0),
    ("bf16", 4, 2, 64, [700, 150, 65, 449], True, True, 2, 3),
    ("f32", 4, 2, 64, [700, 150, 65, 449], True, True, 2, 3),
    ("f32", 2, 1, 32, [385, 129, 1], False, False, 0, 4),
    ("bf16", 2, 1, 128, [385, 129, 1], False, False, 0, 4),
    ("bf16", 72, 8, 64, [300, 1, 640], True, False, 0, 0),      # over two workgroups to a CU
    ("f32", 72, 8, 64, [300, 1, 640], True, False, 0, 0),
]


@pytest.mark.parametrize("type_,H,KVH,D,lens,causal,fused,front,back", FORWARD + [
    ("f32", 2, 1, 256, [70, 1, 200], True, False, 0, 2),
    ("bf16", 2, 1, 256, [70, 1, 200], True, True, 0, 0),
    ("bf16", 4, 2, 136, [33, 150], False, True, 0, 0),
    ("f32", 4, 2, 200, [33, 150], False, True, 0, 0),
    ("bf16", 2, 1, 64, [1] * 300, True, False, 0, 0),
])
def test_forward(gpu, dgm, type_, H, KVH, D, lens, causal, fused, front, back):
    c = Case(dgm, type_, H, KVH, D, lens, causal, fused, front, back)
    gpu.begin()
    c.forward(gpu)
    gpu.end()
    c.check(False)
    lse = torch.full_like(c.lse, 7.0)
    a, b = c.starts_list[0], c.starts_list[-1]
    assert (c.lse[:, :a] == lse[:, :a]).all() and (c.lse[:, b:] == lse[:, b:]).all()


@pytest.mark.parametrize("type_,H,KVH,D,lens,causal,fused,front,back", FORWARD)
def test_backward(gpu, dgm, type_, H, KVH, D, lens, causal, fused, front, back):
    c = Case(dgm, type_, H, KVH, D, lens, causal, fused, front, back)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    c.check(True)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_many_short_sequences(gpu, dgm, type_):
    """Over 64 sequences, more than one round of the search for a tile's rows."""
    lens = [(i * 37) % 11 for i in range(5000)]
    c = Case(dgm, type_, 2, 1, 32, lens, True, False, 2, 2)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    one = Case(dgm, type_, 2, 1, 32, lens, True, False, 2, 2)
    a, b = c.starts_list[4000], c.starts_list[4100]
    val, bnd = attn_ref.packed(one.q, one.k, one.v, c.starts_list[4000:4101], c.scale, True, one.dout)
    for name in val:
        attn_ref.assert_within(getattr(c, name)[a:b], val[name][a:b], bnd[name][a:b], name)


def test_sharp_scores(gpu, dgm):
    """Scores of hundreds: weights of 0 and 1, statistics far from 0."""
    c = Case(dgm, "f32", 2, 2, 64, [200, 64], True, scale=20.0)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    c.check(True)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("mid", [131, 331])     # one wave for a block of queries, and two
def test_masked_values_take_no_part(gpu, dgm, type_, bad, mid):
    """Infinite and NaN k, v of a token leave earlier tokens and other sequences as they are; a bad q or dout leaves later keys."""
    lens, end = [50, mid, 40], 50 + mid
    for what, at in (("v", 90), ("k", 90), ("v", end - 1), ("q", 90), ("dout", 90), ("v", 50 + mid // 2)):
        c = Case(dgm, type_, 4, 2, 64, lens, True)
        clean = Case(dgm, type_, 4, 2, 64, lens, True)
        getattr(c, what)[at] = bad
        gpu.begin()
        for x in (c, clean):
            x.forward(gpu)
            x.backward(gpu)
        gpu.end()
        others = torch.ones(c.rows, dtype=torch.bool, device="cuda")
        others[50:end] = False
        early, late = others.clone(), others.clone()
        early[50:at] = True                  # rows before the token
        late[at + 1:end] = True              # and behind it
        rest = torch.ones_like(others)
        rest[at] = False
        clean_rows = {"v": {"out": early, "dq": early, "dk": others, "dv": others},
                      "k": {"out": early, "dq": early, "dk": others, "dv": others},
                      "q": {"out": rest, "dq": rest, "dk": late, "dv": late},
                      "dout": {"out": rest | True, "dq": rest, "dk": late, "dv": late}}[what]
        for name, rows in clean_rows.items():
            assert torch.equal(getattr(c, name)[rows], getattr(clean, name)[rows]), (what, at, name)
        if what == "v":                      # seen by the token itself and what follows it
            o = c.out[at:end].float()
            assert (o.isnan() if math.isnan(bad) else o == bad).all()
            assert not c.dq[at].float().isfinite().any()
        if what == "k":
            assert not c.dk[60].float().isfinite().all() or not math.isnan(bad)


def test_gradient_against_differences(gpu, dgm):
    """The loss's difference along a direction, by the kernel's own forward, is the gradient along it up to
    the difference's truncation (taken from the 64-bit loss) and the forward's bound."""
    c = Case(dgm, "f32", 4, 2, 48, [70, 20], True)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    base = {n: getattr(c, n).clone() for n in "qkv"}
    gen = torch.Generator("cuda").manual_seed(5)
    h = 2.0 ** -6
    for name in "qkv":
        step = (torch.randint(0, 2, base[name].shape, generator=gen, device="cuda") * 2 - 1).float() * h
        got, want, noise = 0.0, 0.0, 0.0
        for sign in (1, -1):
            moved = base[name] + sign * step
            getattr(c, name).copy_(moved)
            gpu.begin()
            c.forward(gpu)
            gpu.end()
            val, bnd = attn_ref.packed(c.q, c.k, c.v, c.starts_list, c.scale, True)
            got += sign * float((c.out.double() * c.dout.double()).sum())
            want += sign * float((val["out"] * c.dout.double()).sum())
            noise += float((bnd["out"] * c.dout.double().abs()).sum())
            getattr(c, name).copy_(base[name])
        taken = (base[name] + step).double() - (base[name] - step).double()   # the step that was made
        val, bnd = attn_ref.packed(c.q, c.k, c.v, c.starts_list, c.scale, True, c.dout)
        along = float((getattr(c, "d" + name).double() * taken).sum())
        exact = float((val["d" + name] * taken).sum())
        slack = float((bnd["d" + name] * taken.abs()).sum())
        assert abs(got - along) <= abs(want - exact) + noise + slack, name
        assert abs(got - along) <= 0.05 * abs(along) + noise + slack, name


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_same_bits_on_another_stream_and_in_a_graph(dgm, torch_cuda, type_):
    """Captured forward and backward, replayed with other lengths, between eager calls."""
    lens = [100, 1, 64, 91]
    stream = torch.cuda.Stream()
    g = dgm.GPU(stream=stream)
    try:
        with torch.cuda.stream(stream):
            c = Case(dgm, type_, 4, 2, 64, lens)
            eager = Case(dgm, type_, 4, 2, 64, lens)
            ws = torch.empty(g.attnPackedBwd_ws_bytes(c.cfg), dtype=torch.uint8, device="cuda")

            def both(x):
                g.attnPackedFwd(x.cfg, x.q, x.k, x.v, x.starts, x.out, x.lse)
                g.attnPackedBwd(x.cfg, x.q, x.k, x.v, x.starts, x.out, x.lse, x.dout, x.dq, x.dk, x.dv, ws, ws.numel())

            g.begin()
            both(c)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                both(c)
            for other in ([100, 1, 64, 91], [0, 200, 56, 0], [64, 64, 64, 64]):
                starts = [0]
                for n in other:
                    starts.append(starts[-1] + n)
                for x in (c, eager):
                    x.starts.copy_(torch.tensor(starts, dtype=torch.int32))
                    for t in (x.out, x.dq, x.dk, x.dv):
                        t.fill_(7.0)
                both(eager)
                graph.replay()
                stream.synchronize()
                for name in ("out", "lse", "dq", "dk", "dv"):
                    assert torch.equal(getattr(c, name), getattr(eager, name)), (other, name)
            g.end()
    finally:
        g.close()


@pytest.mark.parametrize("starts", [[0, 300], [-1, 64], [0, 64, 32, 96]])
def test_bad_starts_are_reported(gpu, dgm, starts):
    """Starts beyond the rows or out of order: nothing outside the buffers, and an error at the region's end, once."""
    c = Case(dgm, "f32", 2, 1, 32, [32] * (len(starts) - 1), back=96)
    c.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    gpu.begin()
    c.forward(gpu)
    with pytest.raises(dgm.DgmError) as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    ok = Case(dgm, "f32", 2, 1, 32, [32])
    gpu.begin()
    ok.forward(gpu)
    gpu.end()


def test_refusals(gpu, dgm):
    c = Case(dgm, "f32", 4, 2, 32, [40])

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

    def fwd(**change):
        cfg = dgm.AttnCfg.from_buffer_copy(c.cfg)
        for name, value in change.items():
            setattr(cfg, name, value)
        return status(lambda: gpu.attnPackedFwd(cfg, c.q, c.k, c.v, c.starts, c.out, c.lse))

    before = c.out.clone()
    assert fwd(type=2) == fwd(rows=-1) == fwd(nseq=-1) == fwd(H=0) == fwd(KVH=0) == fwd(D=0) == dgm.DGM_ERR_ARG
    assert fwd(scale=0.0) == fwd(scale=-1.0) == fwd(scale=math.nan) == fwd(scale=math.inf) == dgm.DGM_ERR_ARG
    assert fwd(KVH=3) == fwd(ldq=64) == fwd(ldk=32) == fwd(ldo=8) == dgm.DGM_ERR_SHAPE
    assert fwd(D=12) == fwd(D=264) == fwd(ldq=132) == fwd(rows=(1 << 30) + 1) == dgm.DGM_ERR_UNSUPPORTED
    assert status(lambda: gpu.attnPackedFwd(c.cfg, None, c.k, c.v, c.starts, c.out, c.lse)) == dgm.DGM_ERR_ARG
    assert status(lambda: gpu.attnPackedFwd(c.cfg, c.q, c.k, c.v, None, c.out, c.lse)) == dgm.DGM_ERR_ARG
    assert status(lambda: gpu.attnPackedFwd(c.cfg, c.q.data_ptr() + 4, c.k, c.v, c.starts, c.out, None)) == \
        dgm.DGM_ERR_UNSUPPORTED
    n = gpu.attnPackedBwd_ws_bytes(c.cfg)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    bwd = lambda cfg, w, size: status(lambda: gpu.attnPackedBwd(  # noqa: E731
        cfg, c.q, c.k, c.v, c.starts, c.out, c.lse, c.dout, c.dq, c.dk, c.dv, w, size))
    assert bwd(c.cfg, ws, n - 1) == bwd(c.cfg, None, n) == dgm.DGM_ERR_ARG
    wide = dgm.AttnCfg.from_buffer_copy(c.cfg)
    wide.D = 136
    assert bwd(wide, ws, n) == dgm.DGM_ERR_UNSUPPORTED
    assert torch.equal(c.out, before) and (c.dq == 7).all()
    with pytest.raises(dgm.DgmError) as e:      # outside a region
        gpu.attnPackedFwd(c.cfg, c.q, c.k, c.v, c.starts, c.out, c.lse)
    assert e.value.code == dgm.DGM_ERR_NOT_BEGUN
    for rows, nseq in ((0, 1), (40, 0)):        # nothing to do
        assert fwd(rows=rows, nseq=nseq) == dgm.DGM_OK
    assert torch.equal(c.out, before)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("nseq", [63, 64, 65, 129])
def test_sequence_counts_about_a_wave(gpu, dgm, type_, nseq):
    """Up to 64 sequences are ranked by a wave's lanes, more are searched in rounds."""
    lens = [(i * 53) % 200 * (i % 7 != 3) for i in range(nseq)]
    c = Case(dgm, type_, 2, 1, 32, lens, True, False, 1, 1)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    c.check(True)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("nseq", [4, 64, 100])
def test_backward_with_bad_starts(gpu, dgm, type_, nseq):
    """Wild starts write to the buffers' rows only, and are reported."""
    c = Case(dgm, type_, 4, 2, 64, [12] * nseq)
    wild = [0, 2 ** 31 - 1, -2 ** 31, 12 * nseq, 0, 5, 12 * nseq + 1, -1] * 16
    c.starts.copy_(torch.tensor(wild[:nseq + 1], dtype=torch.int32))
    behind = {}
    for name in ("out", "dq", "dk", "dv"):
        t = getattr(c, name)
        behind[name] = torch.full((2 * t.shape[0], *t.shape[1:]), 7.0, device="cuda").to(t.dtype)
        setattr(c, name, behind[name][c.rows // 2:c.rows // 2 + c.rows])
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    with pytest.raises(dgm.DgmError) as e:
        gpu.end()
    assert e.value.code == dgm.DGM_ERR_SHAPE
    for t in behind.values():
        assert (t[:c.rows // 2] == 7).all() and (t[c.rows // 2 + c.rows:] == 7).all()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_masked_huge_values_take_no_part(gpu, dgm, type_):
    """Values near the type's largest and lowest, whose products overflow, at masked positions."""
    lens, at = [50, 300, 40], 200
    for what in ("k", "v", "q", "dout"):
        c, clean = (Case(dgm, type_, 4, 2, 64, lens, True) for _ in range(2))
        getattr(c, what)[at, :, ::2] = torch.finfo(TYPES[type_]).max
        getattr(c, what)[at, :, 1::2] = torch.finfo(TYPES[type_]).min
        gpu.begin()
        for x in (c, clean):
            x.forward(gpu)
            x.backward(gpu)
        gpu.end()
        for name in ("out", "dq") if what in "kv" else ("dk", "dv"):
            rows = torch.ones(c.rows, dtype=torch.bool, device="cuda")
            if what in "kv":
                rows[at:350] = False         # what sees the token
            else:
                rows[50:at + 1] = False      # what the token sees
            assert torch.equal(getattr(c, name)[rows], getattr(clean, name)[rows]), (what, name)


def test_rows_beyond_32_bits(gpu, dgm):
    """Sequences at the end of buffers of over 2^31 elements."""
    H, KVH, D, rows, lens = 4, 2, 128, (1 << 21) + 300, [200, 100]
    wide, grad = (torch.empty(rows, H + 2 * KVH, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out, dout = (torch.empty(rows, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lse = torch.empty(H, rows, device="cuda")
    small = Case(dgm, "bf16", H, KVH, D, lens, True, True)
    last = slice(rows - 300, rows)
    wide[last, :H], wide[last, H:H + KVH], wide[last, H + KVH:], dout[last] = small.q, small.k, small.v, small.dout
    starts = torch.tensor([rows - 300, rows - 100, rows], dtype=torch.int32, device="cuda")
    cfg = dgm.AttnCfg.from_buffer_copy(small.cfg)
    cfg.rows, ld = rows, (H + 2 * KVH) * D
    cfg.ldq = cfg.ldk = cfg.ldv = ld
    assert (rows - 300) * ld >= 1 << 31
    n = gpu.attnPackedBwd_ws_bytes(cfg)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    cut = lambda t: (t[:, :H], t[:, H:H + KVH], t[:, H + KVH:])  # noqa: E731
    q, k, v = cut(wide)
    dq, dk, dv = cut(grad)
    gpu.begin()
    gpu.attnPackedFwd(cfg, q, k, v, starts, out, lse)
    gpu.attnPackedBwd(cfg, q, k, v, starts, out, lse, dout, dq, dk, dv, ws, n)
    gpu.end()
    small.out, small.lse, small.dq, small.dk, small.dv = out[last], lse[:, last], dq[last], dk[last], dv[last]
    small.check(True)


def test_two_contexts_at_once(dgm, torch_cuda):
    """Two streams with a context and a workspace each give what each gives alone."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    gpus = [dgm.GPU(stream=s) for s in streams]
    try:
        lens = [[900, 400, 1], [128] * 12]
        cases = [Case(dgm, t, 8, 2, 64, n) for t, n in zip(("f32", "bf16"), lens)]
        alone = [Case(dgm, t, 8, 2, 64, n) for t, n in zip(("f32", "bf16"), lens)]
        for x in cases + alone:
            x.space = torch.empty(gpus[0].attnPackedBwd_ws_bytes(x.cfg), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

        def step(g, x):
            g.attnPackedFwd(x.cfg, x.q, x.k, x.v, x.starts, x.out, x.lse)
            g.attnPackedBwd(x.cfg, x.q, x.k, x.v, x.starts, x.out, x.lse, x.dout, x.dq, x.dk, x.dv, x.space,
                            x.space.numel())

        for g, x in zip(gpus, alone):
            g.begin()
            step(g, x)
            g.end()
        for g in gpus:
            g.begin()
        for _ in range(4):
            for g, x in zip(gpus, cases):
                step(g, x)
        for g in gpus:
            g.end()
        for x, y in zip(cases, alone):
            for name in ("out", "lse", "dq", "dk", "dv"):
                assert torch.equal(getattr(x, name), getattr(y, name)), name
    finally:
        for g in gpus:
            g.close()


# Grids for each way of laying a block of queries over waves: few workgroups, some, many, short sequences.
LAYOUTS = [(4, 2, [300, 1, 640]), (24, 8, [300, 1, 640]), (72, 8, [300, 1, 640]), (8, 4, [100] * 9)]


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("D", [16, 64, 72, 96, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,KVH,lens", LAYOUTS)
def test_layouts(gpu, dgm, type_, D, causal, H, KVH, lens):
    c = Case(dgm, type_, H, KVH, D, lens, causal, True, 2, 3)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    c.check(True)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("H,KVH,lens", LAYOUTS)
def test_masked_values_in_every_layout(gpu, dgm, type_, D, H, KVH, lens):
    """A NaN token leaves what its mask hides it from as it is."""
    first = sum(lens[:-1])
    for what, at in (("k", first + 70), ("v", first + 33), ("q", first + 70), ("dout", first + 33)):
        c, clean = (Case(dgm, type_, H, KVH, D, lens) for _ in range(2))
        getattr(c, what)[at] = math.nan
        gpu.begin()
        for x in (c, clean):
            x.forward(gpu)
            x.backward(gpu)
        gpu.end()
        rows = torch.ones(c.rows, dtype=torch.bool, device="cuda")
        if what in "kv":
            rows[at:] = False
        else:
            rows[first:at + 1] = False
        for name in ("out", "dq") if what in "kv" else ("dk", "dv"):
            assert torch.equal(getattr(c, name)[rows], getattr(clean, name)[rows]), (what, name)
        if what in "kv":
            assert c.out[at:].isnan().any(2).all()


@pytest.mark.parametrize("lens", [[2], [1, 3, 7, 64], [33, 40, 17]])
@pytest.mark.parametrize("KVH,D", [(8, 32), (2, 32), (8, 64), (2, 64), (8, 80), (2, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_keys_keep_the_precision_of_bf16(gpu, dgm, lens, KVH, D, causal):
    """Over a tile of keys or less dq and dk are rounded where they are written, not where out was: delta is as exact as
    the products, and dS is taken in two pieces, off by 2^-8 of what one is."""
    c = Case(dgm, "bf16", 8, KVH, D, lens, causal)
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    q, k, v, dout = (t.double() for t in (c.q, c.k, c.v, c.dout))
    want, off = ([torch.zeros_like(q), torch.zeros_like(k)] for _ in range(2))
    for a, b in zip(c.starts_list[:-1], c.starts_list[1:]):
        n = b - a
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda")
        seen = seen.tril() if causal else seen
        for h in range(8):
            g = h * KVH // 8
            args = [t.contiguous() for t in (q[a:b, h], k[a:b, g], v[a:b, g])]
            S, W, eW = attn_ref.scores(args[0], args[1], c.scale, seen)
            lse = torch.logsumexp(S, 1, keepdim=True)
            eP = 2 * eW + (n + 4) * attn_ref.U + 4 * attn_ref.U * lse.abs()
            near = (W * (eP + (D + n + 4) * attn_ref.U)) @ args[2].abs()    # the sum of P dP, as an error of out
            (dq, dk, _), e0 = attn_ref.backward(*args, c.scale, seen, near, dout[a:b, h].contiguous(), False)
            _, e1 = attn_ref.backward(*args, c.scale, seen, near, dout[a:b, h].contiguous(), True)
            for i, (x, at) in enumerate(((dq, h), (dk, g))):
                want[i][a:b, at] += x
                off[i][a:b, at] += e0[i] + 2.0 ** -8 * (e1[i] - e0[i]) + 4 * n * attn_ref.U * x.abs()
    for i, name in enumerate(("dq", "dk")):
        bound = off[i] + attn_ref.rounding(torch.bfloat16) * (want[i].abs() + off[i]) + 1e-30
        attn_ref.assert_within(getattr(c, name), want[i], bound, name)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("KVH,D", [(8, 32), (2, 64), (8, 96), (2, 128)])
def test_one_key_has_no_slope(gpu, dgm, type_, KVH, D):
    """A softmax over one key is 1 whatever the score: dq and dk are 0, not what rounding leaves."""
    c = Case(dgm, type_, 8, KVH, D, [1, 1, 1])
    gpu.begin()
    c.forward(gpu)
    c.backward(gpu)
    gpu.end()
    assert not c.dq.any() and not c.dk.any()
    c.check(True)
