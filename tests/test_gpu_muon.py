"""GPU: Newton-Schulz orthogonalisation and the Muon update against float64 on the CPU.

The library computes in fp64 from the fp32 inputs and rounds once: half a step of the
result (U = 2^-24 of it).  What its polynomial of the Gram matrix and the reference's
products round differently is 2^-53 of the largest square, times at most (3.4445^2)^steps
for the smallest singular values: 1e-7 at 8 steps and below 1e-9 at 5."""
import ctypes as C
import math

import pytest
import torch

import llmt
from helpers import SMALL, small_problem, upload_model

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
A_, B_, C_ = 3.4445, -4.7750, 2.0315


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def ns64(x, steps=5, eps=1e-7):
    """By the definition, on the matrix itself, in float64."""
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    x = x / (x.pow(2).sum((-1, -2), keepdim=True).sqrt() + f32(eps))
    for _ in range(steps):
        g = x @ x.transpose(-1, -2)
        x = A_ * x + (B_ * g + C_ * (g @ g)) @ x
    return x.transpose(-1, -2) if tall else x


def spectrum(g, count, rows, cols, low=1e-3):
    """Matrices with singular values from 1 down to `low`."""
    k = min(rows, cols)
    q1 = torch.linalg.qr(torch.randn(count, rows, k, generator=g, dtype=torch.double))[0]
    q2 = torch.linalg.qr(torch.randn(count, cols, k, generator=g, dtype=torch.double))[0]
    s = torch.logspace(0, math.log10(low), k, dtype=torch.double)
    return ((q1 * s) @ q2.transpose(1, 2)).float()


SHAPES = [(1, 1, 1), (1, 1, 7), (2, 5, 1), (3, 4, 4), (1, 16, 16), (1, 16, 2048), (2, 2048, 16),
          (5, 8, 100), (3, 16, 65), (4, 129, 16), (2, 17, 300), (1, 300, 31), (3, 32, 1000),
          (2, 33, 33), (1, 40, 4099), (2, 1024, 48), (1, 64, 64), (2, 64, 5000), (1, 12288, 64),
          (300, 16, 130), (1, 16, 40001), (70, 1024, 16), (1, 61, 61), (260, 16, 2048),
          (3, 5000, 16), (9, 16, 2432), (2, 2433, 15)]


@pytest.mark.parametrize("count,rows,cols", SHAPES)
def test_orthogonalize(dev, count, rows, cols):
    g = torch.Generator().manual_seed(count + rows * 7 + cols)
    for steps, x in ((5, torch.randn(count, rows, cols, generator=g) * 1e-4),
                     (5, spectrum(g, count, rows, cols)), (1, torch.randn(count, rows, cols, generator=g)),
                     (8, spectrum(g, count, rows, cols, 0.05))):
        want = ns64(x, steps)
        got = llmt.orthogonalize(x.to(dev), steps=steps).cpu().double()
        assert ((got - want).abs() <= U * want.abs() + (1e-7 if steps > 5 else 1e-9)).all(), \
            (steps, float((got - want).abs().max()))


def test_orthogonal_rows(dev):
    """Five steps bring every singular value from [0.1, 1] of the norm into [0.65, 1.2]."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(16, 2048, generator=g)
    s = torch.linalg.svdvals(llmt.orthogonalize(x.to(dev)).cpu().double())
    assert 0.65 <= s.min() and s.max() <= 1.2


def test_rank_deficient_zero_and_bad_matrices(dev):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 16, 500, generator=g)
    x[0] = torch.outer(torch.randn(16, generator=g), torch.randn(500, generator=g))
    x[1] = 0
    x[2, 3, 77] = math.nan
    x[3, 0, 0] = math.inf
    x[4] *= 1e30
    got = llmt.orthogonalize(x.to(dev)).cpu().double()
    assert (got[1] == 0).all() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    for i in (0, 4, 5):
        want = ns64(x[i])
        # x[0]: its rounding to fp32 has other directions, amplified alike on both sides
        assert ((got[i] - want).abs() <= U * want.abs() + 1e-8).all(), i


@pytest.mark.parametrize("count,rows,cols", [(3, 16, 129), (2, 200, 16), (2, 33, 70), (40, 16, 1024)])
def test_strides_in_place_and_what_lies_between(dev, count, rows, cols):
    g = torch.Generator().manual_seed(3)
    buf = torch.full((count, rows + 2, cols + 5), 7.0)
    buf[:, :rows, 1:cols + 1] = torch.randn(count, rows, cols, generator=g)
    d = buf.to(dev)
    view = d[:, :rows, 1:cols + 1]
    want = llmt.orthogonalize(view.contiguous())
    out = torch.full((count, rows, cols + 3), -3.0, device=dev)
    llmt.orthogonalize(view, out=out[:, :, :cols])
    assert torch.equal(out[:, :, :cols], want) and (out[:, :, cols:] == -3).all()
    llmt.orthogonalize(view, out=view)
    assert torch.equal(view, want)
    assert (d[:, rows:] == 7).all() and (d[:, :, 0] == 7).all() and (d[:, :, cols + 1:] == 7).all()
    one = llmt.orthogonalize(buf[0, :rows, 1:cols + 1].to(dev))
    assert one.shape == (rows, cols) and torch.equal(one, want[0])


def test_no_matrices(dev):
    assert llmt.orthogonalize(torch.empty(0, 4, 8, device=dev)).shape == (0, 4, 8)


def muon64(p, g, m, shapes, hp):
    """The update in float64, with the momentum and the update rounded as documented: fp32."""
    mu, lr, wd = hp.momentum, hp.lr, hp.wd
    m = (mu * m.double() + g.double()).float()
    u = (mu * m.double() + g.double()).float() if hp.nesterov else m
    per = sum(r * c for r, c in shapes)
    new, size = p.double() * (1 - lr * wd), p.double().abs()
    for l in range(len(p) // per):
        at = l * per
        for r, c in shapes:
            sl = slice(at, at + r * c)
            s = 0.2 * math.sqrt(max(r, c)) if hp.scale == 0 else math.sqrt(max(1.0, r / c))
            o = lr * s * ns64(u[sl].view(r, c), hp.steps, hp.eps).reshape(-1)
            new[sl] -= o
            size[sl] += o.abs()
            at += r * c
    return new, m, size


ARENAS = [(3, [(16, 256), (256, 16), (16, 128), (512, 16)]), (1, [(16, 2048)]),
          (28, [(16, 2048), (2048, 16), (16, 2048), (1024, 16), (16, 2048), (1024, 16), (16, 2048),
                (2048, 16)]),
          (2, [(8, 100), (33, 70), (1, 9), (64, 64), (1000, 40), (7, 7)]), (5, [(4, 5000), (3, 11)])]


@pytest.mark.parametrize("nesterov,scale", [(True, "rms"), (False, "shape")])
@pytest.mark.parametrize("layers,shapes", ARENAS)
def test_muon_update(dev, layers, shapes, nesterov, scale):
    n = layers * sum(r * c for r, c in shapes)
    g = torch.Generator().manual_seed(n)
    p, gr, m = (torch.randn(n, generator=g) * s for s in (0.02, 1e-3, 5e-3))
    hp = llmt.muon_hparams(lr=0.02, momentum=0.9, wd=0.1, nesterov=nesterov, scale=scale)
    pd, gd, md = p.to(dev), gr.to(dev), m.to(dev)
    for _ in range(2):
        want, wm, size = muon64(p, gr, m, shapes, hp)
        llmt.muon_update(pd, gd, md, shapes, hp)
        assert torch.equal(md.cpu(), wm)
        # the orthogonal matrix, the decayed parameter, the step's factor and the sum
        # round once each
        assert ((pd.cpu().double() - want).abs() <= 4 * U * size + 1e-9).all()
        p, m = pd.cpu(), md.cpu()
    assert torch.equal(gd.cpu(), gr)


def test_muon_moves_against_the_gradient(dev):
    """The direction is a descent direction: <update, gradient> = sum of singular values > 0."""
    g = torch.Generator().manual_seed(6)
    p, gr = torch.zeros(16 * 300), torch.randn(16 * 300, generator=g)
    pd, md = p.to(dev), torch.zeros(16 * 300, device=dev)
    llmt.muon_update(pd, gr.to(dev), md, [(16, 300)], llmt.muon_hparams(wd=0.0))
    assert float((pd.cpu() * gr).sum()) < 0


def test_same_bits_on_a_side_stream_and_in_a_graph(dev):
    layers, shapes = 3, [(16, 2048), (2048, 16), (20, 300)]
    n = layers * sum(r * c for r, c in shapes)
    g = torch.Generator().manual_seed(4)
    p, gr, m = (torch.randn(n, generator=g).to(dev) for _ in range(3))
    hp = llmt.muon_hparams()
    p1, m1 = p.clone(), m.clone()
    llmt.muon_update(p1, gr, m1, shapes, hp)
    side = torch.cuda.Stream()
    p2, m2 = p.clone(), m.clone()
    side.wait_stream(torch.cuda.current_stream())
    llmt.muon_update(p2, gr, m2, shapes, hp, stream=side)
    side.synchronize()
    assert torch.equal(p1, p2) and torch.equal(m1, m2)
    x = p[:16 * 2048].view(16, 2048)
    want = llmt.orthogonalize(x)
    graph = torch.cuda.CUDAGraph()
    p3, m3 = p.clone(), m.clone()
    with torch.cuda.graph(graph):
        llmt.muon_update(p3, gr, m3, shapes, hp)
        o = llmt.orthogonalize(x)
    for _ in range(3):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, llmt.orthogonalize(x))   # x as the graph read it
        llmt.muon_update(p, gr, m, shapes, hp)
        torch.cuda.synchronize()
        assert torch.equal(p, p3) and torch.equal(m, m3)
    assert not torch.equal(o, want)


def test_context_muon_updates_adapters_and_their_operand_copies(dev):
    W, ad, tok, tgt = small_problem()
    dims = llmt.make_dims(SMALL)
    ctx = llmt.Context(dims, max_batch=2, seq_len=64)
    try:
        upload_model(ctx, W, dev)
        ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
        ctx.forward_backward(tok.to(dev), tgt.to(dev))
        p, g, m = (ctx.lora_get(k) for k in ("param", "grad", "m"))
        r, h, q, kv = 16, SMALL.hidden, SMALL.q_dim, SMALL.kv_dim
        shapes = [(r, h), (q, r), (r, h), (kv, r), (r, h), (kv, r), (r, q), (h, r)]
        hp = llmt.muon_hparams(lr=0.01)
        for _ in range(2):
            ctx.muon(hp)
            llmt.muon_update(p, g, m, shapes, hp)
            assert torch.equal(ctx.lora_get("param"), p) and torch.equal(ctx.lora_get("m"), m)
        loss = ctx.forward_backward(tok.to(dev), tgt.to(dev))
        ctx.lora_set("param", p)                       # rewrites the operand copies
        assert ctx.forward_backward(tok.to(dev), tgt.to(dev)) == loss
    finally:
        ctx.close()


def test_the_binding_refuses_wrong_arguments(dev):
    x, v = torch.zeros(4, 8, device=dev), torch.zeros(64, device=dev)
    hp = llmt.muon_hparams()
    for call in (lambda: llmt.orthogonalize(x.half()), lambda: llmt.orthogonalize(x[0]),
                 lambda: llmt.orthogonalize(x.t()), lambda: llmt.orthogonalize(x, out=x[:3]),
                 lambda: llmt.orthogonalize(x, steps=0), lambda: llmt.orthogonalize(x, eps=0.0),
                 lambda: llmt.orthogonalize(torch.zeros(65, 65, device=dev)),
                 lambda: llmt.orthogonalize(x.expand(3, 4, 8)),
                 lambda: llmt.muon_update(v, v.clone(), v.clone(), [(5, 5)], hp),
                 lambda: llmt.muon_update(v, v, v.clone(), [(8, 8)], hp),
                 lambda: llmt.muon_update(v, v.clone(), v[:32], [(8, 8)], hp),
                 lambda: llmt.muon_update(v, v.clone(), v.clone(), [], hp)):
        with pytest.raises(llmt.LlmtError):
            call()
