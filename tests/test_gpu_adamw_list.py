"""GPU: llmt.adamw_update over lists of tensors against float64 (the parameters) and, for the
moments, against the same fp32 operations one at a time; 8-bit codes bit for bit against
adam_ref.py.

p: the update's factors carry a few fp32 roundings and two hardware approximations of one ulp (8
steps of 2^-24 of the update cover them), and p' one rounding each of the product and the sum."""
import math

import numpy as np
import pytest
import torch

import adam_ref as ref
import llmt

pytestmark = pytest.mark.gpu
F, H, B = torch.float32, torch.float16, torch.bfloat16
HP = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, wd=0.1)
f32 = lambda x: np.float32(x)


def numpy_step(p, g, m, v, step, hp=HP, scale=None):
    """(p' float64, update's size, m', v' fp32 as defined)."""
    b1, b2, lr, eps, wd = (f32(hp[x]) for x in ("beta1", "beta2", "lr", "eps", "wd"))
    g = g.astype(np.float32)
    if scale is not None:
        g = g * f32(scale)
    with np.errstate(all="ignore"):
        m = b1 * m + (f32(1) - b1) * g
        v = b2 * v + ((f32(1) - b2) * g) * g
        b1, b2, lr, eps, wd = map(float, (b1, b2, lr, eps, wd))
        up = lr * (m.astype(np.float64) / (1 - b1 ** step)) / (
            np.sqrt(v.astype(np.float64) / (1 - b2 ** step)) + eps)
    return p.astype(np.float64) * (1 - lr * wd) - up, np.abs(up), m, v


def problem(sizes, gt=F, seed=0, dev="cpu"):
    g = torch.Generator().manual_seed(seed + len(sizes))
    ps = [torch.randn(n, generator=g) for n in sizes]
    gs = [(torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(gt) for n in sizes]
    return [p.to(dev) for p in ps], [x.to(dev) for x in gs]


def check_p(got, want, up):
    got = got.cpu().numpy().astype(np.float64)
    bound = 2 ** -23 * np.abs(want) + 8 * 2 ** -24 * up + 2 ** -23 * up
    assert (np.abs(got - want) <= bound + 1e-300).all(), np.max(np.abs(got - want) / (bound + 1e-300))


SIZES = [[1], [3, 0, 5], [255, 256, 257], [4095, 4096, 4097, 1], [70000, 2], [7] * 100 + [9000]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("gt,ct", [(F, None), (B, B), (H, H), (F, B)])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(dev, sizes, gt, ct, bits):
    ps, gs = problem(sizes, gt, dev=dev)
    states = [llmt.adamw_state(p, bits) for p in ps]
    copies = None if ct is None else [torch.zeros(p.shape, dtype=ct, device=dev) for p in ps]
    if copies and len(copies) > 2:
        copies[1] = None
    lst = llmt.AdamTensors(ps, gs, states, copies)
    factor = torch.full((1,), 0.75, device=dev)
    hp = llmt.hparams(**HP)
    m = [np.zeros(n, np.float32) for n in sizes]
    v = [np.zeros(n, np.float32) for n in sizes]
    for step in (1, 2, 3):
        before = [p.cpu().numpy() for p in ps]
        llmt.adamw_update(lst, hp, step, grad_scale=factor, seed=11)
        for i, n in enumerate(sizes):
            if n == 0:
                continue
            want, up, m[i], v[i] = numpy_step(before[i], gs[i].float().cpu().numpy(), m[i], v[i],
                                              step, scale=0.75)
            check_p(ps[i], want, up)
            if copies and copies[i] is not None:
                assert torch.equal(copies[i], ps[i].to(ct))
            s = states[i]
            if bits == 32:
                assert np.array_equal(s.m.cpu().numpy(), m[i])
                assert np.array_equal(s.v.cpu().numpy(), v[i])
                continue
            dm, dv = ref.draws(n, 11, step, i)
            for code, ex, x, top, d in ((s.m, s.m_exp, m[i], 15, dm), (s.v, s.v_exp, v[i], 31, dv)):
                want_e = ref.block_exps(x)
                assert np.array_equal(ex.cpu().numpy(), want_e)
                want_c = ref.codes_of(x, want_e, top, d)
                assert np.array_equal(code.cpu().numpy(), want_c)
            got_m, got_v = (x.cpu().numpy() for x in llmt.adamw_moments(s))
            m[i] = ref.values(s.m.cpu().numpy(), s.m_exp.cpu().numpy(), 15).astype(np.float32)
            v[i] = ref.values(s.v.cpu().numpy(), s.v_exp.cpu().numpy(), 31).astype(np.float32)
            assert np.array_equal(got_m, m[i]) and np.array_equal(got_v, v[i])


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views_give_the_same(dev, bits):
    """Tensors that begin anywhere in larger ones; what lies around them stays."""
    n = 5003
    ps, gs = problem([n], B, dev=dev)
    s = llmt.adamw_state(ps[0], bits)
    c = torch.zeros(n, dtype=B, device=dev)
    hp = llmt.hparams(**HP)
    p0 = ps[0].clone()
    llmt.adamw_update(llmt.AdamTensors(ps, gs, [s], [c]), hp, 1, seed=5)

    def inside(t, shift):
        big = torch.full((n + 16,), 3, dtype=t.dtype, device=dev)
        big[shift:shift + n] = t
        return big, big[shift:shift + n]
    for shift in (1, 2, 3):
        bp, p = inside(p0, shift)
        bg, g = inside(gs[0], shift)
        z = llmt.adamw_state(p, bits)
        bm, m = inside(z.m, shift)
        bv, v = inside(z.v, shift)
        bc, k = inside(torch.zeros_like(c), shift)
        llmt.adamw_update(llmt.AdamTensors([p], [g], [(m, v, z.m_exp, z.v_exp)], [k]), hp, 1, seed=5)
        assert torch.equal(p, ps[0]) and torch.equal(k, c) and torch.equal(m, s.m) and torch.equal(v, s.v)
        if bits == 8:
            assert torch.equal(z.m_exp, s.m_exp) and torch.equal(z.v_exp, s.v_exp)
        for b in (bp, bg, bm, bv, bc):
            assert (b[:shift] == 3).all() and (b[shift + n:] == 3).all()


def test_the_rounding_of_moments_is_unbiased(dev):
    """b2 = 0.999 with a constant gradient: v grows by 0.1% of its end a step, less than half of
    a code's step from the first few steps on, and still ends where the average does.  With r the
    relative step of a code (2^-3 at most) a rounding has a variance of at most (r / 2)^2 of its value
    and the average keeps 0.999 of it a step: the deviation of a mean over N elements is at most r / 2
    / sqrt(N) sqrt(sum of 0.999^2k) < 1.4 / sqrt(N).  Six of those."""
    n, steps = 1 << 16, 400
    p = torch.zeros(n, device=dev)
    g = torch.ones(n, device=dev)
    g[::256] = 1.8                                   # the blocks' scale is not the rest's
    s = llmt.adamw_state(p, 8)
    lst = llmt.AdamTensors([p], [g], [s])
    hp = llmt.hparams(lr=0.0, beta1=0.99, beta2=0.999)
    for t in range(1, steps + 1):
        llmt.adamw_update(lst, hp, t, seed=3)
    m, v = llmt.adamw_moments(s)
    rest = torch.ones(n, dtype=torch.bool, device=dev)
    rest[::256] = False
    room = 6 * 1.4 / math.sqrt(n)
    for x, b in ((m, 0.99), (v, 0.999)):
        assert abs(float(x[rest].double().mean()) / (1 - float(f32(b)) ** steps) - 1) < room


def test_small_moments_beside_large_ones(dev):
    """One block with 12 decades of gradients: a v above 0 stays above 0, and no step is larger
    than the formula allows."""
    n = 256
    g = (10.0 ** torch.linspace(-12, 0, n)).to(dev)
    p = torch.zeros(n, device=dev)
    s = llmt.adamw_state(p, 8)
    lst = llmt.AdamTensors([p], [g], [s])
    hp = llmt.hparams(lr=1e-3, eps=1e-30, wd=0.0)
    for t in range(1, 30):
        before = p.clone()
        llmt.adamw_update(lst, hp, t, seed=1)
        # |m'| / sqrt(v') <= (1 - b1) / sqrt(1 - b2) for fresh moments, and kept ones only shrink it
        assert ((p - before).abs() <= 1e-3 * 40).all()
        m, v = llmt.adamw_moments(s)
        assert (v > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_smallest_gradients(dev, bits):
    """Squares that are subnormal numbers, under an eps below them: the moments bit for bit, the
    update as for any other size."""
    n = 768
    g = (10.0 ** torch.linspace(-20, -17, n)).to(dev)
    hp = dict(HP, eps=1e-30)
    p = torch.zeros(n, device=dev)
    s = llmt.adamw_state(p, bits)
    z = np.zeros(n, np.float32)
    llmt.adamw_update(llmt.AdamTensors([p], [g], [s]), llmt.hparams(**hp), 1, seed=2)
    want, up, m, v = numpy_step(z, g.cpu().numpy(), z, z, 1, hp=hp)
    assert (v > 0).all() and v.min() < 2.0 ** -126 and up.min() > 0.9 * HP["lr"]
    check_p(p, want, up)
    if bits == 32:
        assert np.array_equal(s.m.cpu().numpy(), m) and np.array_equal(s.v.cpu().numpy(), v)


def test_a_list_keeps_its_memory(dev):
    """A parameter that is given other memory afterwards: the list's own is updated, not freed."""
    ps, gs = problem([4000], dev=dev)
    first = ps[0]
    old = first.detach()
    lst = llmt.AdamTensors(ps, gs, [llmt.adamw_state(first)])
    want = old.clone()
    llmt.adamw_update(llmt.AdamTensors([want], gs, [llmt.adamw_state(want)]), llmt.hparams(**HP), 1)
    other = torch.full_like(old, 5.0)
    first.data = other
    llmt.adamw_update(lst, llmt.hparams(**HP), 1)
    assert torch.equal(old, want) and (other == 5).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
def test_values_beyond_range(dev, bad):
    ps, gs = problem([700], dev=dev)
    g = gs[0]
    g[300] = bad
    for bits in (32, 8):
        p = ps[0].clone()
        s = llmt.adamw_state(p, bits)
        llmt.adamw_update(llmt.AdamTensors([p], [g], [s]), llmt.hparams(**HP), 1)
        ok = torch.ones(700, dtype=torch.bool, device=dev)
        ok[300] = False
        assert p[ok].isfinite().all()
        m, v = llmt.adamw_moments(s)
        if bits == 8:
            assert v[256:512].isnan().all() and v[:256].isfinite().all() and v[512:].isfinite().all()
        else:
            assert v[ok].isfinite().all() and not v[300].isfinite()


def test_zero_gradients_leave_zero_moments(dev):
    p = torch.ones(1000, device=dev)
    for bits in (32, 8):
        s = llmt.adamw_state(p, bits)
        q = p.clone()
        llmt.adamw_update(llmt.AdamTensors([q], [torch.zeros_like(p)], [s]), llmt.hparams(**HP), 1)
        m, v = llmt.adamw_moments(s)
        assert not m.any() and not v.any()
        assert torch.equal(q, p * float(f32(1 - float(f32(HP["lr"])) * float(f32(HP["wd"])))))


def test_captured_replayed_and_on_another_stream(dev):
    ps, gs = problem([3000, 17, 5000], B, dev=dev)
    start = [p.clone() for p in ps]
    hp = llmt.hparams(**HP)
    for bits in (32, 8):
        def fresh():
            for p, x in zip(ps, start):
                p.copy_(x)
            return [llmt.adamw_state(p, bits) for p in ps]
        s = fresh()
        lst = llmt.AdamTensors(ps, gs, s)
        for _ in range(3):
            llmt.adamw_update(lst, hp, 4, seed=9)
        want = [p.clone() for p in ps] + [t.clone() for x in s for t in x if t is not None]
        s = fresh()
        lst = llmt.AdamTensors(ps, gs, s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            llmt.adamw_update(lst, hp, 4, seed=9)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
        got = ps + [t for x in s for t in x if t is not None]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        s = fresh()
        lst = llmt.AdamTensors(ps, gs, s)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            llmt.adamw_update(lst, hp, 4, seed=9, stream=side)
        side.synchronize()
        got = ps + [t for x in s for t in x if t is not None]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_gradients_for_the_same_list(dev):
    ps, gs = problem([500, 20], dev=dev)
    other = [g.to(B) * 2 for g in gs]
    a = [p.clone() for p in ps]
    lst = llmt.AdamTensors(a, gs, [llmt.adamw_state(p) for p in a])
    lst.set_grads(other)
    llmt.adamw_update(lst, llmt.hparams(**HP), 1)
    b = [p.clone() for p in ps]
    llmt.adamw_update(llmt.AdamTensors(b, other, [llmt.adamw_state(p) for p in b]),
                      llmt.hparams(**HP), 1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_as_the_contexts_adamw(dev):
    """The formula of llmt_adamw on a context's arena: the same parameters to a few roundings."""
    from helpers import SMALL, small_problem, upload_model
    W, ad, tok, tgt = small_problem()
    ctx = llmt.Context(llmt.make_dims(SMALL), max_batch=tok.shape[0], seq_len=tok.shape[1])
    try:
        upload_model(ctx, W, dev)
        ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
        p = ctx.lora_get("param")
        ctx.step(tok.to(dev), tgt.to(dev), llmt.hparams(), 1)
        g = ctx.lora_get("grad")
        s = llmt.adamw_state(p)
        llmt.adamw_update(llmt.AdamTensors([p], [g], [s]), llmt.hparams(), 1)
        # the context's bias corrections are fp32: 1 - 0.999 to 2^-24 / 0.001, about 6e-5 of the update
        assert (p - ctx.lora_get("param")).abs().max() <= 1e-4 * 3e-4 + 2 ** -23 * p.abs().max()
        assert torch.allclose(s.m, ctx.lora_get("m"), rtol=1e-6, atol=0)
        assert torch.allclose(s.v, ctx.lora_get("v"), rtol=1e-6, atol=0)
    finally:
        ctx.close()
