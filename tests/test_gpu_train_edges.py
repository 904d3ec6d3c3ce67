"""GPU: borders of the operators for training all weights on packed sequences: scores next to the
documented bound in the attention's large tiles, heads of one buffer that lie between one another, rows beyond 2^28;
AdamW's largest moments, its lists of large tensors and of tensors unlike in size; small
gradients with exact inputs; calls beside others."""
import math

import numpy as np
import pytest
import torch

import llmt
import packed_ref as ref
import test_gpu_adamw_list as adamw
from test_gpu_adamw_list import HP, check_p, numpy_step
from test_gpu_packed import offsets, problem

pytestmark = pytest.mark.gpu
F, H, B = torch.float32, torch.float16, torch.bfloat16
LN2 = float(np.float32(math.log(2)))


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (16, 8, 64), (32, 8, 64)])
@pytest.mark.parametrize("T", [1100, 4200])
def test_maxima_of_millions_that_grow_by_small_steps(dev, dtype, nq, nkv, d, T):
    """Scores of 1.6e7 whose tiles' maxima rise by 2 to 14 steps of a base-2 score each, in the
    workgroups of 64 and of 128 rows.  With scale ln 2 the base-2 scores are q k itself (ln 2 log2 e
    is 1 in fp32): 4096 * 5632 + 2 r + s_j, even numbers below 2^25, which fp32 holds exactly in any
    order of the sum.  So a score is exact, a weight 2^(s_j - max) too, and o is off by the rounding
    of P (u), those of the sums and the exponential (2^-16) and its own (u).  lse: five roundings and
    constants of 2^-24."""
    assert np.float32(LN2) * np.float32(1.4426950408889634) == 1
    g = torch.Generator().manual_seed(T + nq + d)
    tiles = -(-T // 64)
    # a tile's maximum: above the last one's by 2 .. 14, at most 500 in all: exact in both types
    rise = 2 * torch.randint(1, 8, (tiles,), generator=g)
    rise[1], rise[2] = 8, 8                       # the first two from an m that is 0 or 2 mod 4
    top = rise.cumsum(0).clamp(max=500)
    s = top.repeat_interleave(64)[:T] - 2 * torch.randint(0, 8, (T,), generator=g)
    first = torch.arange(0, T, 64)
    s[first + torch.randint(0, 64, (tiles,), generator=g).clamp(max=T - 1 - first)] = top
    s = s - top[0]
    q, k = torch.zeros(T, nq, d), torch.zeros(T, nkv, d)
    r = torch.arange(T) // 64 % 2                 # by the token's block: a wave's rows alike
    q[..., 0], q[..., 1], q[..., 2], k[..., 0], k[..., 2] = 4096, 1, r[:, None], 5632, 2
    k[..., 1] = s[:, None]
    v = torch.randn(T, nkv, d, generator=g).to(dtype).to(dev)
    q, k = (x.to(dtype).to(dev) for x in (q, k))
    assert (k[:, 0, 1].cpu() == s).all()
    o, lse = llmt.packed_attention(q, k, v, offsets([T]).to(dev), scale=LN2)
    w = s.double().to(dev)
    see = torch.ones(T, T, dtype=torch.bool, device=dev).tril()
    w = torch.where(see, w[None], -math.inf)
    m = w.amax(1, keepdim=True)
    p = torch.exp2(w - m)
    total = p.sum(1, keepdim=True)
    p = p / total
    base = 4096.0 * 5632 + 2 * r.double().to(dev)
    want = (base + (m + total.log2())[:, 0]) * math.log(2)
    assert ((lse.double() - want[:, None]).abs() <= 5 * 2 ** -24 * want[:, None]).all()
    u = ref.unit(dtype)
    for h in range(nq):
        x = v[:, h // (nq // nkv)].double()
        y, mag = p @ x, p @ x.abs()
        assert ((o[:, h].double() - y).abs() <= (u + 2 ** -16) * mag + u * y.abs() + 2 ** -25).all(), h


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("ql", [[1], [9, 50], [700, 900]])
@pytest.mark.parametrize("nq,nkv,d,parts,turned", [(6, 2, 64, 2, False), (16, 8, 128, 2, False), (8, 4, 128, 2, True),
                                                   (4, 4, 64, 3, False), (4, 4, 128, 3, True)])
def test_heads_between_one_another(dev, dtype, ql, nq, nkv, d, parts, turned):
    """Projections whose rows are [heads, 2, d] (keys and values) or [heads, 3, d] (queries too),
    tokens or heads outermost: the bits of separate tensors, and what lies beside stays."""
    q, k, v, do, qo, _ = problem(dev, dtype, d, nq, nkv, ql)
    T, heads = q.shape[0], (q, k, v)[3 - parts:]

    def buffer():
        x = torch.full((nkv, T, parts, d) if turned else (T, nkv, parts, d + 8), 7.0, dtype=dtype, device=dev)
        return x, [(x.transpose(0, 1) if turned else x)[:, :, i, :d] for i in range(parts)]
    _, inside = buffer()
    for x, y in zip(inside, heads):
        x.copy_(y)
    inside = [q, k, v][:3 - parts] + inside
    o, lse = llmt.packed_attention(q, k, v, qo)
    o2, lse2 = llmt.packed_attention(*inside, qo)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    want = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo)
    buf, out = buffer()
    out = [torch.empty_like(q)][:3 - parts] + out
    got = llmt.packed_attention_bwd(*inside, o, lse, do, qo, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert turned or (buf[..., d:] == 7).all()


def test_gradients_of_more_than_2_28_rows(dev):
    """16 heads of 2^24 tokens and some: 100 tokens with keys behind all the others, which have
    none.  (One row of q, dout and o serves a token's heads; dq alone is 69 GB.)"""
    nq, d, few, T = 16, 128, 100, (1 << 24) + 4096
    if torch.cuda.mem_get_info()[0] < 90e9:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("90 GB of device memory are needed")
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g).to(B).to(dev)
    row = torch.zeros(T, d, dtype=B, device=dev)
    row[-few:] = rnd(few, d)
    x = row[:, None].expand(T, nq, d)
    k, v = rnd(few, nq, d), rnd(few, nq, d)
    qo = torch.tensor([0, T - few, T], dtype=torch.int32, device=dev)
    ko = torch.tensor([0, 0, few], dtype=torch.int32, device=dev)
    tail = x[-few:]
    _, end = llmt.packed_attention(tail, k, v, ko[1:])
    lse = torch.full((T, nq), -math.inf, device=dev)
    lse[-few:] = end
    dq = torch.empty(T, nq, d, dtype=B, device=dev).fill_(math.nan)
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    llmt.packed_attention_bwd(x, k, v, x, lse, x, qo, ko, out=(dq, dk, dv))
    want, bounds = ref.backward(tail, k, v, tail, end, tail, ko[1:], ko[1:], d ** -0.5)
    for name, a, b, bound in zip(("dq", "dk", "dv"), (dq[-few:], dk, dv), want, bounds):
        ref.within(name, a, b, bound)
    for part in dq[:-few].split(1 << 20):
        assert not (part != 0).any()
    del dq, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("beta2", [0.9, 0.99, 0.999])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_gradients(dev, bits, beta2, sign):
    """Second moments in fp32's range whose quotient by 1 - beta2^step is not: the update as for any
    other size, lr in the first step.  (8 bits: the largest block ends below 1.875 2^126.)"""
    n, steps = 1024, 3
    largest = math.sqrt(1.2e38 / (1 - beta2 ** steps))     # v to 1.2e38, codes an eighth more
    g = (sign * largest * 2.0 ** -torch.linspace(0, 12, n)).to(dev)
    hp = dict(HP, beta2=beta2)
    p, s = torch.zeros(n, device=dev), llmt.adamw_state(torch.zeros(n, device=dev), bits)
    lst = llmt.AdamTensors([p], [g], [s])
    m = v = np.zeros(n, np.float32)
    for step in range(1, steps + 1):
        before = p.cpu().numpy()
        llmt.adamw_update(lst, llmt.hparams(**hp), step, seed=4)
        want, up, m, v = numpy_step(before, g.cpu().numpy(), m, v, step, hp=hp)
        assert np.isfinite(v).all()
        if step == 1:
            hat = v.astype(np.float64) / (1 - float(np.float32(beta2)))
            assert (hat > float(np.finfo(np.float32).max)).sum() > 10 and (up > 0.99 * HP["lr"]).all()
        check_p(p, want, up)
        if bits == 32:
            assert np.array_equal(s.m.cpu().numpy(), m) and np.array_equal(s.v.cpu().numpy(), v)
        else:
            m, v = (x.cpu().numpy() for x in llmt.adamw_moments(s))
            assert np.isfinite(v).all()


@pytest.mark.parametrize("sizes", [
    # above 2.1 M elements: pieces of 4096, a search in every launch, more descriptors than one holds
    [1500001, 4095, 4096, 4097, 0, 1, 700003, 257] + [33, 4097] * 40,
    [4096] * 60 + [2500000, 3],
    # below: pieces of 1024, a search where the sizes are unlike
    [3] * 60 + [200001] + [5] * 8, [200001] + [1025, 3] * 20, [1, 0, 1023, 150000, 1024, 0] + [700] * 20])
@pytest.mark.parametrize("gt,ct", [(F, None), (B, B), (H, H)])
@pytest.mark.parametrize("bits", [32, 8])
def test_lists_whose_workgroups_search_their_tensor(dev, sizes, gt, ct, bits):
    adamw.test_steps(dev, sizes, gt, ct, bits)


@pytest.mark.parametrize("dtype,small", [(H, 2.0 ** -10), (B, 2.0 ** -60)])
@pytest.mark.parametrize("ql", [[300, 41], [1500, 900]])
def test_gradients_of_small_and_large_dout_have_the_same_bits(dev, dtype, small, ql):
    """dout of random signs times [0.5, 4], exact in the type times `small` too, so every
    intermediate value is (fp16's dS in part below its smallest normal number, were it not scaled).
    Keys and queries of 2^-6 under a scale of 2^12 leave the weights as they are and raise dq and
    dk, so that most outputs of the small run are normal numbers (of dv, whose late keys have few
    rows, a third): those are compared from twice the smallest on, where the steps are the
    type's."""
    q, k, v, do, qo, ko = problem(dev, dtype, 128, 16, 8, ql)
    g = torch.Generator().manual_seed(9)
    do = torch.randn(do.shape, generator=g).sign() * (0.5 + 3.5 * torch.rand(do.shape, generator=g))
    do = do.to(dtype).to(dev)
    assert ((do * small).double() == do.double() * small).all()
    q, k, scale = q / 64, k / 64, 128 ** -0.5 * 4096
    o, lse = llmt.packed_attention(q, k, v, qo, scale=scale)
    big = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, scale=scale)
    low = llmt.packed_attention_bwd(q, k, v, o, lse, do * small, qo, scale=scale)
    for a, b, share in zip(big, low, (0.9, 0.9, 1 / 3)):
        normal = b.double().abs() >= 2 * torch.finfo(dtype).tiny
        assert a.isfinite().all() and normal.double().mean() > share
        assert torch.equal(a.double()[normal] * small, b.double()[normal])


def test_beside_other_work_the_same_bits(dev):
    """The operators on four streams at once, beside a stream of products, against the same calls
    one after another."""
    A = llmt.packed_attention
    P = [problem(dev, *p) for p in (
        (B, 128, 16, 8, [1500, 700, 33, 2000, 900, 1, 800, 1200, 1058]), (H, 128, 16, 8, [80, 77, 1, 90, 60, 305]),
        (H, 64, 32, 8, [2100, 65, 7]), (B, 128, 16, 8, [1] * 8, [900, 1, 3000, 64, 700, 2000, 50, 9]))]
    tok = torch.randint(-1, 3000, (20000,), dtype=torch.int32, device=dev)
    dx = torch.randn(20000, 264, device=dev).to(B)
    g = [torch.randn(n, device=dev) for n in (3000000, 70001)]

    def calls(i):
        q, k, v, do, qo, ko = P[i]
        o, lse = A(q, k, v, qo, ko)
        grads = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, ko)
        dw = llmt.embedding_bwd(tok, dx, torch.zeros(3000, 264, device=dev))
        p = [torch.ones_like(x) for x in g]
        s = [llmt.adamw_state(x, 8) for x in p]
        llmt.adamw_update(llmt.AdamTensors(p, g, s), llmt.hparams(**HP), 1, seed=i)
        return [o, lse, *grads, dw, *p, *(t for x in s for t in x)]
    want = [calls(i) for i in range(4)]
    noise = torch.randn(4096, 4096, device=dev).to(B)
    streams = [torch.cuda.Stream() for _ in range(5)]
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(streams[4]):
            for _ in range(8):
                noise @ noise
        got = []
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                got.append(calls(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
