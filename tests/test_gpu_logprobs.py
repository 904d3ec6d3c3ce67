"""GPU: token log-probabilities and their gradient against float64 on the CPU.

Tolerances, with u = 2^-24 (half a step of fp32, relative):
 - exp(x - m): the difference, its product with log2 e and exp2 are each off by
   at most 2 u of themselves, so a term is off by (|z| + 2) 4 u; weighted by
   the terms themselves |z| averages to at most ln V.  A sum of n positive
   terms in turn adds n u, n at most V / 64 terms a thread plus 16 merges.
 - the gradient takes its stats as given: p is off by (|z| + 2) 4 u.
 - a result in type t is rounded once: finfo(t).eps / 2 of itself, or half its
   smallest subnormal.
"""
import math

import pytest
import torch

import llmt

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SUBNORMAL = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def problem(rows, V, dtype, seed=0, skip=0.2, scale=3.0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + V)
    x = (torch.randn(rows, V, generator=g) * scale).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32)
    drop = torch.rand(rows, generator=g) < skip
    t[drop] = torch.tensor([-1, V, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)[
        torch.randint(0, 4, (int(drop.sum()),), generator=g)]
    return g, x, t


def forward64(x, t, temperature=1.0):
    """logp, ln p of every logit, entropy in float64; rows without a target are 0."""
    V = x.shape[1]
    ok = (t >= 0) & (t < V)
    x = x.double() * float(torch.tensor(1.0 / temperature, dtype=torch.float32))
    lg = torch.log_softmax(x, 1)
    lp = lg.gather(1, t.long().clamp(0, V - 1)[:, None])[:, 0]
    ent = -(lg.exp() * torch.where(lg == -math.inf, torch.zeros_like(lg), lg)).sum(1)
    return torch.where(ok, lp, torch.zeros_like(lp)), lg, torch.where(ok, ent, torch.zeros_like(ent)), ok


def sum_tol(V):
    return (V / 64 + 16) * U + (math.log(V) + 2) * 4 * U


def check_forward(x, t, got, temperature=1.0):
    logp, stats, ent = (None if v is None else v.cpu().double() for v in got)
    want, lg, want_ent, ok = forward64(x, t, temperature)
    tol = sum_tol(x.shape[1])
    assert ((logp - want).abs() <= tol + 4 * U * want.abs()).all(), (logp - want).abs().max()
    m = (x.double() * float(torch.tensor(1.0 / temperature, dtype=torch.float32))).amax(1)
    lse = torch.where(ok, stats.sum(1), torch.zeros_like(m))
    true = torch.where(ok, (m - lg.amax(1)), torch.zeros_like(m))
    assert ((lse - true).abs() <= tol + 4 * U * (true.abs() + stats.abs().sum(1))).all()
    assert (stats[~ok] == 0).all() and (logp[~ok] == 0).all()
    if ent is not None:  # its two sums are each off by tol of themselves and at most ln V
        assert ((ent - want_ent).abs() <= tol * (2 + math.log(x.shape[1])) * 2).all(), \
            (ent - want_ent).abs().max()
        assert (ent[~ok] == 0).all()


def backward64(x, t, stats, dlogp, ent, dent, temperature):
    """The documented formula in float64 from the given stats, and the size of its terms."""
    it = float(torch.tensor(1.0 / temperature, dtype=torch.float32))
    V = x.shape[1]
    ok = (t >= 0) & (t < V)
    z = x.double() * it - stats.double()[:, :1] - stats.double()[:, 1:]
    p = z.exp()
    hot = torch.nn.functional.one_hot(t.long().clamp(0, V - 1), V).double()
    d = dlogp.double()[:, None] * (hot - p)
    size = dlogp.double().abs()[:, None] * torch.where(hot > 0, (hot - p).abs(), p)
    if dent is not None:
        zf = torch.where(z == -math.inf, torch.zeros_like(z), z)
        e = dent.double()[:, None] * p * (zf + ent.double()[:, None])
        d, size = d - e, size + dent.double().abs()[:, None] * p * (zf.abs() + ent.double()[:, None])
    z0 = torch.where(z == -math.inf, torch.zeros_like(z), z)
    return d * it * ok[:, None], size * it * ok[:, None] * (z0.abs() + 4) * 4 * U


def check_backward(x, t, stats, dlogp, ent, dent, got, temperature=1.0):
    want, tol = backward64(x, t, stats, dlogp, ent, dent, temperature)
    err = (got.double() - want).abs()
    lim = tol + (want.abs() + tol) * torch.finfo(x.dtype).eps / 2 + SUBNORMAL[x.dtype]
    assert (err <= lim).all(), float((err - lim).max())


SIZES = [(1, 1), (3, 2), (5, 7), (4, 63), (9, 64), (7, 1000), (33, 2048), (130, 257), (2, 8192),
         (6, 50257), (1, 151936), (64, 151936), (3, 262147), (2100, 300)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,V", SIZES)
def test_forward_and_backward(dev, rows, V, dtype):
    g, x, t = problem(rows, V, dtype)
    xd, td = x.to(dev), t.to(dev)
    for temperature, want_ent in ((1.0, False), (0.7, True)):
        got = llmt.token_logprobs(xd, td, temperature=temperature, want_entropy=want_ent)
        check_forward(x, t, got, temperature)
        dlogp = torch.randn(rows, generator=g)
        dent = torch.randn(rows, generator=g) if want_ent else None
        d = llmt.token_logprobs_bwd(xd, td, got[1], dlogp.to(dev), entropy=got[2],
                                    dentropy=None if dent is None else dent.to(dev),
                                    temperature=temperature)
        assert d.dtype == dtype
        check_backward(x, t, got[1].cpu(), dlogp, None if dent is None else got[2].cpu(), dent,
                       d.cpu(), temperature)


@pytest.mark.parametrize("V", [50, 3001, 40000])
def test_gradient_against_autograd_and_differences(dev, V):
    """dlogits of sum(a logp + b H): float64 autograd, and central differences of the
    forward along a direction (fp32 logits: each value of the sum is off by about rows x
    1e-5, so a difference over 2 x 0.01 is off by 1e-3 of a derivative of size 1)."""
    rows = 6
    g, x, t = problem(rows, V, torch.float32, seed=3, skip=0.0)
    a, b = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    x64 = x.double().requires_grad_()
    lg = torch.log_softmax(x64 / 0.5, 1)
    f = (a.double() * lg.gather(1, t.long()[:, None])[:, 0]).sum() - \
        (b.double() * (lg.exp() * lg).sum(1)).sum()
    f.backward()
    xd, td = x.to(dev), t.to(dev)
    lp, st, ent = llmt.token_logprobs(xd, td, temperature=0.5, want_entropy=True)
    d = llmt.token_logprobs_bwd(xd, td, st, a.to(dev), ent, b.to(dev), temperature=0.5)
    scale = x64.grad.abs().max()
    assert (d.cpu().double() - x64.grad).abs().max() <= 1e-5 * scale
    v = torch.sign(d) * (torch.rand(rows, V, generator=g).to(dev) > 0.5)
    value = lambda y: float((a.to(dev).double() * llmt.token_logprobs(y, td, 0.5, True)[0] +
                             b.to(dev).double() * llmt.token_logprobs(y, td, 0.5, True)[2]).sum())
    h = 0.01
    diff = (value(xd + h * v) - value(xd - h * v)) / (2 * h)
    slope = float((d.double() * v).sum())
    assert abs(diff - slope) <= 2e-3 * (1 + abs(slope)), (diff, slope)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strided_rows_and_offset_views(dev, dtype):
    """Rows farther apart than V, starting off any alignment; what lies between them stays."""
    g, x, t = problem(7, 1001, dtype, seed=1)
    buf = torch.full((7, 1100), 9.0, dtype=dtype, device=dev)
    view = buf[:, 3:1004]
    view.copy_(x)
    lp, st, ent = llmt.token_logprobs(view, t.to(dev), want_entropy=True)
    check_forward(x, t, (lp, st, ent))
    dlogp = torch.randn(7, generator=g)
    out = torch.full((7, 1203), 5.0, dtype=dtype, device=dev)
    d = llmt.token_logprobs_bwd(view, t.to(dev), st, dlogp.to(dev), out=out[:, 5:1006])
    check_backward(x, t, st.cpu(), dlogp, None, None, d.cpu())
    assert (out[:, :5] == 5).all() and (out[:, 1006:] == 5).all()
    llmt.token_logprobs_bwd(view, t.to(dev), st, dlogp.to(dev), out=view)  # in place
    assert torch.equal(view, d)
    assert (buf[:, :3] == 9).all() and (buf[:, 1004:] == 9).all()


@pytest.mark.parametrize("V", [100, 9000, 151936, 230000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_masked_logits(dev, dtype, V):
    """Logits of -inf and of the type's lowest value: probability 0, gradient 0; a row of
    nothing but -inf; a target that is masked."""
    g, x, t = problem(5, V, dtype, seed=2, skip=0.0)
    keep = torch.rand(5, V, generator=g) < 0.3
    keep[torch.arange(5), t.long()] = True
    x[~keep] = -math.inf
    x[1][~keep[1]] = torch.finfo(dtype).min
    x[2] = -math.inf
    x[3, t[3]] = -math.inf
    lp, st, ent = (v.cpu() for v in llmt.token_logprobs(x.to(dev), t.to(dev), want_entropy=True))
    ok = [0, 1, 4]
    check_forward(x[ok], t[ok], (lp[ok], st[ok], ent[ok]))
    assert lp[2] == -math.inf and st[2].tolist() == [-math.inf, 0.0] and ent[2] == 0
    assert lp[3] == -math.inf and math.isfinite(st[3].sum()) and math.isfinite(ent[3])
    dlogp, dent = torch.randn(5, generator=g), torch.randn(5, generator=g)
    for e in (None, dent):
        d = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), st.to(dev), dlogp.to(dev),
                                    ent.to(dev), None if e is None else e.to(dev)).cpu()
        assert (d[2] == 0).all()
        rows = [0, 1, 3, 4]
        check_backward(x[rows], t[rows], st[rows], dlogp[rows], ent[rows],
                       None if e is None else e[rows], d[rows])
        masked = ~keep
        masked[2] = False
        assert (d[masked] == 0).all()


@pytest.mark.parametrize("mask", [-1e4, -2e8, -1e9, -1e10, -3e12, -1e20, -1e30, -3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,V", [(4, 1500), (4, 30000), (4, 230000), (300, 4001)])
def test_finite_masks(dev, rows, V, dtype, mask):
    """Masks of large finite values: whole stretches of a row, all of a row but one logit, and
    all of a row, which leaves its logits equal and every probability 1 / V; logits that are
    large and positive.  (Sizes where the product with the inverse temperature is off by more
    than the logits of a softmax differ.)"""
    g, x, t = problem(rows, V, dtype, seed=11, skip=0.0)
    x[0, V // 3:] = mask
    x[1] = mask
    x[1, V // 2] = 1.0
    x[2] = mask
    x[3, :] = -mask
    x[3, V // 4:] = mask
    t[0], t[1], t[2], t[3] = 5, V // 2, V - 1, 0
    dlogp, dent = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    for temperature in (1.0, 0.9, 1.7):
        if abs(mask) > 2e38 and temperature < 1:
            continue                      # the scaled logits leave fp32
        got = llmt.token_logprobs(x.to(dev), t.to(dev), temperature, want_entropy=True)
        check_forward(x, t, got, temperature)
        want, lg, ent, _ = forward64(x, t, temperature)
        assert abs(float(got[0][2]) + math.log(V)) <= 1e-5 and abs(float(got[2][2]) - math.log(V)) <= 1e-4
        # the gradient by the formula, from probabilities in float64
        it = float(torch.tensor(1.0 / temperature, dtype=torch.float32))
        p = lg.exp()
        lz = torch.where(p > 0, lg, torch.zeros_like(lg))
        hot = torch.nn.functional.one_hot(t.long(), V).double()
        for e in (None, dent):
            d = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), got[1], dlogp.to(dev), got[2],
                                        None if e is None else e.to(dev), temperature).cpu().double()
            a = dlogp.double()[:, None] * it
            ref, size = a * (hot - p), a.abs() * torch.where(hot > 0, (hot - p).abs() + p, p)
            if e is not None:
                b = e.double()[:, None] * it
                ref, size = ref - b * p * (lz + ent[:, None]), size + b.abs() * p * (lz.abs() + ent[:, None])
            # p and the entropy are off as in the forward; one rounding
            tol = size * (sum_tol(V) * 4 * (2 + math.log(V)) + (lz.abs() + 4) * 8 * U)
            tol = tol + (ref.abs() + tol) * torch.finfo(dtype).eps / 2 + SUBNORMAL[dtype]
            if e is not None:             # H where it all but vanishes: its absolute error
                tol = tol + b.abs() * p * sum_tol(V) * 2 * (2 + math.log(V))
            assert ((d - ref).abs() <= tol).all(), float(((d - ref).abs() - tol).max())


@pytest.mark.parametrize("V", [100, 9000, 230000])
def test_scaled_logits_that_leave_fp32(dev, V):
    """Masks that the inverse temperature takes to -inf are -inf."""
    g, x, t = problem(3, V, torch.float32, seed=12, skip=0.0)
    x[0, 50:] = torch.finfo(torch.float32).min
    t[0] = 3
    x[1] = torch.finfo(torch.float32).min
    lp, st, ent = (v.cpu() for v in llmt.token_logprobs(x.to(dev), t.to(dev), 0.5, want_entropy=True))
    check_forward(x[[0, 2]], t[[0, 2]], tuple(v[[0, 2]] for v in (lp, st, ent)), 0.5)
    assert lp[1] == -math.inf and st[1].tolist() == [-math.inf, 0.0] and ent[1] == 0
    one = torch.ones(3, device=dev)
    d = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), st.to(dev), one, ent.to(dev), one, 0.5).cpu()
    assert (d[1] == 0).all() and torch.isfinite(d).all() and (d[0, 50:] == 0).all()


def test_a_bad_logit_stays_in_its_row(dev):
    g, x, t = problem(6, 20000, torch.float32, seed=4, skip=0.0)
    x[1, 777], x[3, 19999], x[4] = math.nan, math.inf, math.nan
    lp, st, ent = llmt.token_logprobs(x.to(dev), t.to(dev), want_entropy=True)
    one = torch.ones(6, device=dev)
    d = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), st, one, ent, one)
    for i in (1, 3, 4):
        assert torch.isnan(lp[i]) and torch.isnan(st[i].sum()) and torch.isnan(ent[i])
        assert torch.isnan(d[i]).all()
    good = [0, 2, 5]
    check_forward(x[good], t[good], tuple(v.cpu()[good] for v in (lp, st, ent)))
    assert torch.isfinite(d[good]).all()


def test_rows_without_a_part_are_not_read(dev):
    """Rows without a target, and in the backward rows with no gradient: NaN there stays
    there; their outputs are zeros."""
    g, x, t = problem(8, 5000, torch.float16, seed=5, skip=0.0)
    t[2], t[6] = -1, 5000
    x[2] = math.nan
    lp, st, ent = llmt.token_logprobs(x.to(dev), t.to(dev), want_entropy=True)
    assert lp[2] == 0 and (st[2] == 0).all() and ent[2] == 0
    dlogp = torch.randn(8, generator=g)
    dlogp[4] = 0.0
    x[4] = math.nan
    d = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), st, dlogp.to(dev))
    assert (d[[2, 4, 6]] == 0).all() and torch.isfinite(d).all()


def test_no_rows(dev):
    x = torch.empty(0, 100, device=dev)
    lp, st, ent = llmt.token_logprobs(x, torch.empty(0, dtype=torch.int32, device=dev))
    assert lp.shape == (0,) and st.shape == (0, 2)
    assert llmt.token_logprobs_bwd(x, torch.empty(0, dtype=torch.int32, device=dev), st, lp).shape == (0, 100)


def test_offsets_past_32_bits(dev):
    """Two rows 2^31 + 64 elements apart."""
    V, ld = 70001, 2 ** 31 + 64
    g, x, t = problem(2, V, torch.float16, seed=6, skip=0.0)
    buf = torch.empty(ld + V, dtype=torch.float16, device=dev)
    view = buf.as_strided((2, V), (ld, 1))
    view.copy_(x)
    lp, st, ent = llmt.token_logprobs(view, t.to(dev), want_entropy=True)
    check_forward(x, t, (lp, st, ent))
    dlogp = torch.randn(2, generator=g)
    want = llmt.token_logprobs_bwd(x.to(dev), t.to(dev), st, dlogp.to(dev))
    llmt.token_logprobs_bwd(view, t.to(dev), st, dlogp.to(dev), out=view)
    assert torch.equal(view, want)


@pytest.mark.parametrize("rows,V", [(3, 151936), (300, 5000), (40, 500), (5, 230001)])
def test_same_bits_on_a_side_stream_and_in_a_graph(dev, rows, V):
    g, x, t = problem(rows, V, torch.float32, seed=8)
    xd, td, dl = x.to(dev), t.to(dev), torch.randn(rows, generator=g).to(dev)

    def both():
        lp, st, ent = llmt.token_logprobs(xd, td, want_entropy=True)
        return lp, st, ent, llmt.token_logprobs_bwd(xd, td, st, dl, ent, dl)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lp, st, ent = llmt.token_logprobs(xd, td, want_entropy=True, stream=side)
    d = llmt.token_logprobs_bwd(xd, td, st, dl, ent, dl, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (lp, st, ent, d)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(3):
        xd.mul_(0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))
