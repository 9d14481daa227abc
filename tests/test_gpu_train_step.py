"""The operators of a training step together, as a language model's step runs them: embeddings with a scale, a layer of packed
attention between norms, the quantized head, the loss, back through all of them, and AdamW over all tensors."""
from __future__ import annotations

import pytest
import torch

import step_ref as ref

pytestmark = pytest.mark.gpu

V, C, H, D = 96, 64, 4, 16
LENS = [7, 1, 30, 26]
ROWS = sum(LENS)


class Model:
    """embed -> norm 1 -> attention of (q = k = v = the rows' heads) -> + residual, norm 2 -> head in int8 codes."""

    def __init__(self, dgm, gpu, seed=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.dgm, self.gpu = dgm, gpu
        self.params = [dgm.Param("wte", V, C, False, True, 8, 32), dgm.Param("head", V, C, True, True, 8, 32)]
        self.params += [dgm.Param(f"ln{i}.{k}", C, 1, False, False, 8, 32) for i in (1, 2) for k in "gb"]
        self.p = {p.name: p for p in self.params}
        for name in ("wte", "head"):
            self.p[name].w.copy_(torch.randn(V * C, generator=gen, device="cuda") * 0.3)
        for i in (1, 2):
            self.p[f"ln{i}.g"].w.copy_(1 + 0.1 * torch.randn(C, generator=gen, device="cuda"))
            self.p[f"ln{i}.b"].w.copy_(0.1 * torch.randn(C, generator=gen, device="cuda"))
        self.tokens = torch.randint(0, V, (ROWS,), generator=gen, device="cuda", dtype=torch.int32)
        self.targets = torch.randint(0, V, (ROWS,), generator=gen, device="cuda", dtype=torch.int32)
        at = 0
        for n in LENS:      # a sequence's last row has nothing to predict
            self.targets[at + n - 1] = -1
            at += n
        self.starts = torch.tensor([sum(LENS[:i]) for i in range(len(LENS) + 1)], dtype=torch.int32, device="cuda")
        f = dgm.DGM_TYPE_F32
        self.rows = dgm.RowsCfg(type=f, tableType=f, scale=C ** 0.5, rows=ROWS, C=C, V=V)
        self.norm = dgm.NormCfg(type=f, eps=1e-5, rows=ROWS, cols=C)
        self.loss_cfg = dgm.LossCfg(type=f, scale=1.0 / (ROWS - len(LENS)), rows=ROWS, V=V)
        self.attn = dgm.AttnCfg(type=f, H=H, KVH=H, D=D, causal=1, scale=D ** -0.5, rows=ROWS, nseq=len(LENS))
        z = lambda *s: torch.zeros(*s, device="cuda")
        self.x, self.y1, self.a, self.h, self.y2 = (z(ROWS, C) for _ in range(5))
        self.dy1, self.dy2, self.dh, self.dq, self.dk, self.dv, self.dx = (z(ROWS, C) for _ in range(7))
        self.stats = [z(ROWS) for _ in range(4)]
        self.lse, self.logits, self.loss = z(H, ROWS), z(ROWS, V), z(ROWS)
        sizes = (gpu.layerNormBwd_ws_bytes(self.norm), gpu.attnPackedBwd_ws_bytes(self.attn), gpu.embedRowsBwd_ws_bytes(self.rows))
        self.ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes]

    def quantize(self):
        p = self.p["head"]
        self.gpu.quantize(p.w, p.q, p.scale, V, C, 8, 32)

    def forward(self):
        g, p, w = self.gpu, self.p, {n: t.w for n, t in self.p.items()}
        m1, r1, m2, r2 = self.stats
        g.embedRows(self.rows, self.tokens, w["wte"], self.x)
        g.layerNormFwd(self.norm, self.x, None, w["ln1.g"], w["ln1.b"], None, self.y1, m1, r1)
        g.attnPackedFwd(self.attn, self.y1, self.y1, self.y1, self.starts, self.a, self.lse)
        g.layerNormFwd(self.norm, self.a, self.x, w["ln2.g"], w["ln2.b"], self.h, self.y2, m2, r2)
        g.gemmNT(8, None, p["head"].q, p["head"].scale, self.y2, None, self.logits, ROWS, V, C, 32)

    def backward(self):
        g, p = self.gpu, self.p
        m1, r1, m2, r2 = self.stats
        G = {n: t.g for n, t in p.items()}
        self.dgm.zero_grads(g, self.params)
        g.crossEntropy(self.loss_cfg, self.logits, self.targets, self.loss, dlogits=self.logits)
        g.gemmBwd(8, None, p["head"].q, p["head"].scale, self.logits, self.y2, self.dy2, G["head"], ROWS, V, C, 32)
        g.layerNormBwd(self.norm, self.h, m2, r2, p["ln2.g"].w, self.dy2, None, self.dh, G["ln2.g"], G["ln2.b"], self.ws[0],
                       self.ws[0].numel())
        g.attnPackedBwd(self.attn, self.y1, self.y1, self.y1, self.starts, self.a, self.lse, self.dh, self.dq, self.dk, self.dv,
                        self.ws[1], self.ws[1].numel())
        g.add(self.dq, self.dk, self.dy1, ROWS * C)
        g.add(self.dy1, self.dv, self.dy1, ROWS * C)
        g.layerNormBwd(self.norm, self.x, m1, r1, p["ln1.g"].w, self.dy1, self.dh, self.dx, G["ln1.g"], G["ln1.b"], self.ws[0],
                       self.ws[0].numel())
        g.embedRowsBwd(self.rows, self.tokens, self.dx, G["wte"], self.ws[2], self.ws[2].numel(), accumulate=True)

    def exact(self, over=None):
        """(mean loss, gradients) in 64 bits on the CPU, the head's codes as they are (gradient straight through)."""
        with torch.enable_grad():
            w = {n: t.w[:t.count].double().cpu().requires_grad_() for n, t in self.p.items()}
            p = self.p["head"]
            codes = (p.q[:V * C].view(torch.int8).double().cpu().view(V, C // 32, 32) * p.scale.double().cpu().view(V, C // 32, 1)).view(V, C)
            head = codes + (w["head"].view(V, C) - w["head"].view(V, C).detach())
            x = w["wte"].view(V, C)[self.tokens.long().cpu()] * torch.tensor(C ** 0.5).item()
            ln = lambda t, i: torch.nn.functional.layer_norm(t, (C,), w[f"ln{i}.g"], w[f"ln{i}.b"], self.norm.eps)
            y1, out, at = ln(x, 1), [], 0
            for n in LENS:
                t = y1[at:at + n].view(n, H, D).transpose(0, 1)
                s = (t @ t.transpose(1, 2)) * D ** -0.5
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
                out.append((torch.softmax(s, -1) @ t).transpose(0, 1).reshape(n, C))
                at += n
            z = ln(x + torch.cat(out), 2) @ head.t()
            loss = torch.nn.functional.cross_entropy(z, self.targets.long().cpu(), ignore_index=-1)
            loss.backward()
        return loss.item(), {n: t.grad for n, t in w.items()}


def test_gradients(dgm, gpu, torch_cuda):
    """A chain of fp32 operators: each adds a few u relative to its rows' size, the products 1e-5 (their bar); 1e-4 of a
    gradient's norm holds them all."""
    m = Model(dgm, gpu)
    gpu.begin()
    m.quantize()
    m.forward()
    m.backward()
    gpu.end()
    loss, grads = m.exact()
    assert abs(m.loss.double().sum().item() / (ROWS - len(LENS)) - loss) <= 1e-5 * loss
    for n, want in grads.items():
        got = m.p[n].g[:m.p[n].count].double().cpu()
        assert (got - want.view(-1)).norm() <= 1e-4 * want.norm(), n


@pytest.mark.parametrize("state", [32, 8])
def test_steps_as_a_graph(dgm, torch_cuda, state):
    """Three whole steps eagerly, and the same from one captured graph (the learning rate and the corrections
    stay those of the capture): the same bits."""
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)
    models = [Model(dgm, own, 3) for _ in range(2)]
    opts = [dgm.AdamMany(own, m.params, state) for m in models]
    torch.cuda.synchronize()

    def step(i):
        models[i].forward()
        models[i].backward()
        return opts[i].step(1e-2, 0.1, 0.5, 1)
    own.begin()
    for m in models:
        m.quantize()
    own.end()
    own.begin()
    graph = torch.cuda.CUDAGraph()
    step(1)     # the products' workspace is there before a capture
    own.end()
    for p, q in zip(models[0].params, models[1].params):
        q.w.copy_(p.w)
        if state == 32:
            q.m.zero_()
            q.v.zero_()
    for codes in opts[1].codes.values():
        for t in codes:
            t.zero_()
    torch.cuda.synchronize()
    own.begin()
    models[1].quantize()
    own.end()
    own.begin()
    with torch.cuda.graph(graph, stream=side):
        step(1)
    losses = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        step(0)
        own.end()
        own.begin()
        losses.append(models[0].loss.sum().item())
        for p, q in zip(models[0].params, models[1].params):
            assert torch.equal(p.w, q.w) and (not p.quantized or torch.equal(p.q, q.q)), p.name
        assert torch.equal(models[0].loss, models[1].loss)
    own.end()
    own.close()
    assert losses[2] != losses[0]


def test_two_steps_at_once(dgm, torch_cuda):
    """Two models on two contexts and streams, their steps in flight together: each the bits that it has alone."""
    def run(together):
        sides = [torch.cuda.Stream() for _ in range(2)]
        owns = [dgm.GPU(stream=s) for s in sides]
        models = [Model(dgm, g, 10 + i) for i, g in enumerate(owns)]
        opts = [dgm.AdamMany(g, m.params, 8 if i else 32) for i, (g, m) in enumerate(zip(owns, models))]
        torch.cuda.synchronize()
        for g, m in zip(owns, models):
            g.begin()
            m.quantize()
        for _ in range(4):
            for g, m, o in zip(owns, models, opts):
                m.forward()
                m.backward()
                o.step(1e-2, 0.1, 0.5, 1)
                if not together:
                    g.end()
                    g.begin()
        for g in owns:
            g.end()
        out = [[t.clone() for p in m.params for t in (p.w, p.g)] + [m.loss.clone(), m.dx.clone()] for m in models]
        torch.cuda.synchronize()
        for g in owns:
            g.close()
        return out
    alone, both = run(False), run(True)
    assert all(torch.equal(a, b) for x, y in zip(alone, both) for a, b in zip(x, y))


def test_replays_report_tokens_and_targets(dgm, torch_cuda):
    """A captured step that meets a token or target beyond the vocabulary tells the next end() of its context, and once."""
    side = torch.cuda.Stream()
    own = dgm.GPU(stream=side)
    m = Model(dgm, own, 5)
    torch.cuda.synchronize()
    own.begin()
    m.quantize()
    m.forward()
    own.end()
    own.begin()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        own.embedRows(m.rows, m.tokens, m.p["wte"].w, m.x)
        own.crossEntropy(m.loss_cfg, m.logits, m.targets, m.loss)
    tokens, targets = m.tokens.clone(), m.targets.clone()
    for where, what in ((None, None), (m.tokens, V), (None, None), (m.targets, V + 7), (m.tokens, -2), (None, None)):
        m.tokens.copy_(tokens)
        m.targets.copy_(targets)
        if where is not None:
            where[3] = what
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        if where is None:
            own.end()
        else:
            with pytest.raises(dgm.DgmError, match="beyond the vocabulary") as e:
                own.end()
            assert e.value.code == dgm.DGM_ERR_SHAPE
            assert (m.x[3] == 0).all() if where is m.tokens else m.loss[3] == 0
        own.begin()
    own.end()
    own.close()
