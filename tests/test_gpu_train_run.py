"""GPU: the operators together as a program that trains all weights of a small model on packed
sequences uses them: embedding, packed attention, log-probabilities of the targets, their backwards
by hand, and AdamW over the list of weights with 16-bit working copies.  The loss and every weight's
gradient against torch autograd in float64 (the framework's bounds: loss within 1e-3, gradients
within 1e-2 relative L2), the update against its formula, and the whole step captured into a graph
against eager steps."""
import math

import pytest
import torch

import llmt

pytestmark = pytest.mark.gpu

V, W, NQ, NKV, D, LAYERS = 97, 192, 4, 2, 64, 2
LENGTHS = [40, 1, 71, 23]
SCALE = W ** 0.5          # of the embedding: rows of variance 1, logits of order 1 from the tied head
LOSS_SCALE = 256.0


class Model:
    def __init__(self, dev, dtype, bits, lengths=LENGTHS):
        g = torch.Generator().manual_seed(4)
        rnd = lambda *s: torch.randn(*s, generator=g)
        shapes = [(V, W)] + [((NQ + 2 * NKV) * D, W), (W, NQ * D)] * LAYERS
        self.p = [(rnd(*s) * s[1] ** -0.5).to(dev) for s in shapes]
        self.w = [p.to(dtype) for p in self.p]
        for p, w in zip(self.p, self.w):
            p.copy_(w)                       # the oracle sees what the kernels see
        self.g = [torch.zeros_like(p) for p in self.p]
        self.state = [llmt.adamw_state(p, bits) for p in self.p]
        self.list = llmt.AdamTensors(self.p, self.g, self.state, self.w)
        T = sum(lengths)
        self.off = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(dev)
        self.tok = torch.randint(0, V, (T,), generator=g).to(torch.int32).to(dev)
        target = self.tok.roll(-1)
        target[(self.off[1:] - 1).long()] = -1   # a sequence's last token has none
        self.target = target
        self.count = int((target >= 0).sum())
        self.dlogp = torch.full((T,), -LOSS_SCALE / self.count, device=dev)
        self.factor = torch.full((1,), 1 / LOSS_SCALE, device=dev)
        self.hp = llmt.hparams(lr=1e-3)

    def heads(self, qkv):
        T = qkv.shape[0]
        a, b = NQ * D, (NQ + NKV) * D
        return qkv[:, :a].view(T, NQ, D), qkv[:, a:b].view(T, NKV, D), qkv[:, b:].view(T, NKV, D)

    def forward_backward(self):
        """logp of the targets; gradients times the loss scale into self.g."""
        E = self.w[0]
        x = llmt.embedding(self.tok, E, scale=SCALE)
        kept = []
        for i in range(LAYERS):
            wqkv, wo = self.w[1 + 2 * i:3 + 2 * i]
            qkv = x @ wqkv.t()
            o, lse = llmt.packed_attention(*self.heads(qkv), self.off)
            kept.append((x, qkv, o, lse))
            x = x + o.view(len(x), -1) @ wo.t()
        logits = x @ E.t()
        logp, stats, _ = llmt.token_logprobs(logits, self.target)
        d = llmt.token_logprobs_bwd(logits, self.target, stats, self.dlogp)
        self.g[0].copy_(d.float().t() @ x.float())       # the tied head's part
        dx = d @ E
        for i in reversed(range(LAYERS)):
            wqkv, wo = self.w[1 + 2 * i:3 + 2 * i]
            xin, qkv, o, lse = kept[i]
            self.g[2 + 2 * i].copy_(dx.float().t() @ o.view(len(x), -1).float())
            do = (dx @ wo).view(o.shape)
            dqkv = torch.empty_like(qkv)
            llmt.packed_attention_bwd(*self.heads(qkv), o, lse, do, self.off, out=self.heads(dqkv))
            self.g[1 + 2 * i].copy_(dqkv.float().t() @ xin.float())
            dx = dx + dqkv @ wqkv
        llmt.embedding_bwd(self.tok, dx, self.g[0], scale=SCALE, accumulate=True)
        return logp

    def step(self, t):
        logp = self.forward_backward()
        llmt.adamw_update(self.list, self.hp, t, grad_scale=self.factor, seed=2)
        return logp

    def oracle(self):
        """(loss, gradients) in float64 by autograd."""
        p = [x.double().cpu().requires_grad_() for x in self.p]
        tok, target, off = self.tok.cpu().long(), self.target.cpu().long(), self.off.tolist()
        x = p[0][tok] * SCALE
        for i in range(LAYERS):
            q, k, v = self.heads(x @ p[1 + 2 * i].t())
            parts = []
            for a, b in zip(off, off[1:]):
                see = torch.ones(b - a, b - a, dtype=torch.bool).tril()
                hs = []
                for h in range(NQ):
                    s = q[a:b, h] @ k[a:b, h * NKV // NQ].t() / math.sqrt(D)
                    hs.append(torch.softmax(s.masked_fill(~see, -math.inf), 1) @ v[a:b, h * NKV // NQ])
                parts.append(torch.cat(hs, 1))
            x = x + torch.cat(parts) @ p[2 + 2 * i].t()
        lp = torch.log_softmax(x @ p[0].t(), 1)
        ok = target >= 0
        loss = -lp[ok, target[ok]].mean()
        return loss.item(), torch.autograd.grad(loss, p)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_loss_and_gradients(dev, dtype):
    m = Model(dev, dtype, 32)
    logp = m.forward_backward()
    loss, grads = m.oracle()
    # bf16 weights times bf16 activations, rounded at every step: 8 times fp16's
    room = 1.0 if dtype == torch.float16 else 8.0
    assert abs(-logp.double().sum().item() / m.count - loss) < 1e-3 * room
    for i, (a, b) in enumerate(zip(m.g, grads)):
        a = a.double().cpu() / LOSS_SCALE
        rel = float((a - b).norm() / b.norm())
        assert rel < 1e-2 * (1.0 if dtype == torch.float16 else 3.0), (i, rel)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_update_is_the_formulas(dev, bits):
    m = Model(dev, torch.float16, bits)
    before = [p.clone() for p in m.p]
    m.step(1)
    for p0, p, w, g in zip(before, m.p, m.w, m.g):
        g = g.double() / LOSS_SCALE
        lr, wd = 1e-3, 0.01
        want = p0.double() * (1 - lr * wd) - lr * g / (g.abs() + 1e-8)   # the first step's m and v
        # moments in fp32: 2^-22 of the update; at gradients near eps the quotient bends
        assert ((p.double() - want).abs() <= 1e-6 * lr + 2 ** -22 * (p0.double().abs() + lr)).all()
        assert torch.equal(w, p.half())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_the_eager_ones(dev, bits):
    """Replays with eager work of the same weights between them; a captured step keeps its number."""
    a, b = Model(dev, torch.float16, bits), Model(dev, torch.float16, bits)
    a.step(1)
    b.step(1)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.forward_backward()                      # library products set up outside the capture
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = b.step(2)
    for _ in range(3):
        want = a.step(2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        for x, y in zip(a.p + a.w + a.g, b.p + b.w + b.g):
            assert torch.equal(x, y)
        for x, y in zip(a.state, b.state):
            assert all(torch.equal(s, t) for s, t in zip(x, y) if s is not None)
        llmt.embedding(b.tok, b.w[0])
        torch.cuda.synchronize()
