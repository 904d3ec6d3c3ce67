"""GPU: llmt.packed_attention and its gradients against float64 (packed_ref.py, which derives
the bounds): lengths from none to several tiles, every kernel, layouts, offsets, masks that leave
rows empty, tokens of no sequence, streams and graphs."""
import ctypes as C
import math

import pytest
import torch

import llmt
import packed_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
INF = math.inf


def offsets(lengths, first=0):
    return torch.tensor([first] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32)


def problem(dev, dtype, d, nq, nkv, ql, kl=None, seed=0, qkv=False, pad=0, scale=1.0):
    """q, k, v, dout and offsets; pad: tokens before the first and behind the last sequence."""
    g = torch.Generator().manual_seed(seed + 7 * sum(ql) + len(ql))
    rnd = lambda *s: torch.randn(*s, generator=g)
    qo, ko = offsets(ql, pad), offsets(ql if kl is None else kl, pad)
    Tq, Tk = int(qo[-1]) + pad, int(ko[-1]) + pad
    if qkv:  # parts of one projection's rows
        x = rnd(Tq, (nq + 2 * nkv) * d).to(dtype).to(dev)
        q = x[:, :nq * d].view(Tq, nq, d)
        k = x[:, nq * d:(nq + nkv) * d].view(Tq, nkv, d)
        v = x[:, (nq + nkv) * d:].view(Tq, nkv, d)
    else:
        q, k, v = (rnd(T, n, d).to(dtype).to(dev) for T, n in ((Tq, nq), (Tk, nkv), (Tk, nkv)))
    do = (scale * rnd(Tq, nq, d)).to(dtype).to(dev)
    return q, k, v, do, qo.to(dev), ko.to(dev)


def check(q, k, v, do, qo, ko, scale=None, same=False, backward=True):
    s = q.shape[2] ** -0.5 if scale is None else scale
    kk = None if same else ko
    o, lse = llmt.packed_attention(q, k, v, qo, kk, scale=scale)
    want, wl, bo, bl = ref.forward(q, k, v, qo, ko, s)
    ref.within("lse", lse, wl, bl)
    ref.within("o", o, want, bo)
    if not backward:
        return o, lse
    got = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, kk, scale=scale)
    want, bounds = ref.backward(q, k, v, o, lse, do, qo, ko, s)
    for name, a, b, bound in zip(("dq", "dk", "dv"), got, want, bounds):
        ref.within(name, a, b, bound)
    return o, lse, *got


HEADS = [(16, 8, 128), (4, 4, 64), (6, 2, 128), (7, 1, 64), (1, 1, 128), (10, 2, 64)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("ql", [[1], [2], [3, 1, 2], [15, 16, 17], [31, 33], [63, 64, 65], [0, 5, 0],
                                [127, 129, 1], [200, 0, 331]])
def test_sequences_of_their_own(dev, dtype, nq, nkv, d, ql):
    check(*problem(dev, dtype, d, nq, nkv, ql, qkv=True), same=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("ql,kl", [
    ([1], [1]), ([1], [500]), ([1, 1, 1], [1, 33, 700]), ([5, 0, 40], [64, 90, 40]),
    # more queries than keys: the first ones see none
    ([10], [3]), ([70, 4], [5, 0]), ([130], [64]), ([3], [0]), ([200, 1], [1, 1])])
def test_keys_of_another_length(dev, dtype, nq, nkv, d, ql, kl):
    p = problem(dev, dtype, d, nq, nkv, ql, kl)
    o, lse, dq, dk, dv = check(*p)
    at = 0
    for a, b in zip(ql, kl):
        none = max(0, a - b) if b else a
        assert not o[at:at + none].any() and (lse[at:at + none] == -INF).all()
        assert not dq[at:at + none].any()
        at += a


# enough rows for 64- and 128-row tiles, lengths across tile borders
@pytest.mark.parametrize("dtype,nq,nkv,d,ql", [
    (BF, 16, 8, 128, [700, 1, 513, 64, 1000]), (HF, 16, 8, 128, [2049, 31, 900, 1200]),
    (BF, 32, 8, 64, [1300, 777]), (HF, 6, 2, 128, [3000]), (BF, 5, 1, 64, [4100, 3]),
    (BF, 16, 8, 128, [4099, 130]), (HF, 32, 8, 64, [2100, 65, 7]),
    # keys enough for workgroups of 64 in one piece
    (BF, 16, 16, 128, [3300, 50]), (HF, 16, 16, 128, [1, 2700]), (HF, 32, 32, 64, [3310]),
    (BF, 40, 40, 64, [2500, 131])])
def test_many_rows(dev, dtype, nq, nkv, d, ql):
    check(*problem(dev, dtype, d, nq, nkv, ql, qkv=True), same=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [62, 63, 65, 300])
def test_many_sequences(dev, dtype, n):
    """More sequences than one search step sees, some of them empty."""
    g = torch.Generator().manual_seed(n)
    ql = torch.randint(0, 4, (n,), generator=g).tolist()
    kl = [a + b for a, b in zip(ql, torch.randint(0, 9, (n,), generator=g).tolist())]
    q, k, v, do, qo, ko = problem(dev, dtype, 64, 2, 1, ql, kl)
    check(q, k, v, do, qo, ko)


# few or many rows against few or many keys: the blocks of rows and of keys that the others do not
# bring together
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d,ql,kl", [
    (16, 8, 128, [77] * 8, None), (32, 8, 64, [60] * 9, None), (32, 1, 128, [7] * 157, None),
    (16, 8, 128, [300, 30, 250], [3000, 2350, 250]), (32, 8, 64, [300, 30, 250], [3000, 2900, 250]),
    (32, 1, 128, [1100], None), (32, 1, 64, [600, 600], [500, 700]), (32, 8, 64, [1, 1, 1], [5000, 2000, 3001]),
    (16, 8, 128, [600], [90]), (4, 4, 128, [500, 500], None), (1, 1, 64, [1900], None), (1, 1, 128, [4000], None),
    (16, 8, 128, [100, 28], [900, 1020]), (8, 1, 64, [64], [4000]), (2, 1, 128, [33, 0, 7], [2500, 10, 2]),
    (1, 1, 64, [4090], None)])
def test_rows_and_keys_of_other_numbers(dev, dtype, nq, nkv, d, ql, kl):
    check(*problem(dev, dtype, d, nq, nkv, ql, kl))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d", [(33, 1, 64), (64, 1, 128), (128, 2, 64)])
@pytest.mark.parametrize("ql,kl", [([1], [1]), ([2, 63, 17], None), ([300, 5], None), ([1, 3], [700, 2])])
def test_large_groups(dev, dtype, nq, nkv, d, ql, kl):
    """Up to 64 query heads share a KV head: a token is a whole tile."""
    check(*problem(dev, dtype, d, nq, nkv, ql, kl))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [253, 254, 255])
@pytest.mark.parametrize("most", [3, 70])
def test_as_many_sequences_as_are_ordered(dev, dtype, n, most):
    g = torch.Generator().manual_seed(n + most)
    ql = torch.randint(0, most, (n,), generator=g).tolist()
    check(*problem(dev, dtype, 64, 4, 4, ql, pad=5))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ql,kl", [([40, 33, 70], None), ([700, 900, 1100], None), ([1, 1, 1], [90, 900, 2000])])
def test_a_sequence_of_nan_stays_alone(dev, dtype, ql, kl):
    """NaN and infinities in one sequence leave its neighbours' bits as they were, in tiles that
    both have rows in."""
    q, k, v, do, qo, ko = problem(dev, dtype, 128, 16, 8, ql, kl)
    o, lse = llmt.packed_attention(q, k, v, qo, ko)
    want = (o, lse, *llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, ko))
    a, b, c, e = int(qo[1]), int(qo[2]), int(ko[1]), int(ko[2])
    for bad in (math.nan, INF):
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        q2[a:b], do2[a:b], k2[c:e], v2[c:e] = bad, bad, bad, bad
        o, lse = llmt.packed_attention(q2, k2, v2, qo, ko)
        got = (o, lse, *llmt.packed_attention_bwd(q2, k2, v2, o, lse, do2, qo, ko))
        for x, y, i, j in zip(got, want, (a, a, a, c, c), (b, b, b, e, e)):
            assert torch.equal(x[:i], y[:i]) and torch.equal(x[j:], y[j:])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (6, 2, 64)])
@pytest.mark.parametrize("kl", [[5000], [1, 3000, 64, 129], [2000] * 7 + [0], [700], [300, 0, 33, 1000], [9000],
                                [16000, 4, 300]])
def test_single_tokens_of_long_keys(dev, dtype, nq, nkv, d, kl):
    """One new token a sequence: the keys are split over workgroups and joined."""
    check(*problem(dev, dtype, d, nq, nkv, [1] * len(kl), kl))


def test_keys_are_split_over_workgroups():
    """The cases above do take the split: a workspace is asked for."""
    for tq, tk, n, nq, nkv, d in ((1, 5000, 1, 16, 8, 128), (8, 14000, 8, 16, 8, 128),
                                  (1, 5000, 1, 6, 2, 64)):
        dims = llmt.PackedDims(2, nq, nkv, d, n, tq, tk, 1.0, 16, 16)
        assert llmt.lib().llmt_packed_attention_workspace(C.byref(dims)) > 0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ql,kl", [([40, 70], None), ([300, 1500], None), ([1, 1], [900, 2000])])
def test_tokens_of_no_sequence(dev, dtype, ql, kl):
    """Padding before and behind the sequences holds NaN: it reaches nothing, and its own outputs
    are 0 (lse -inf)."""
    q, k, v, do, qo, ko = problem(dev, dtype, 128, 16, 8, ql, kl, pad=37)
    for t, off in ((q, qo), (do, qo), (k, ko), (v, ko)):
        t[:int(off[0])] = math.nan
        t[int(off[-1]):] = math.nan
    o, lse = llmt.packed_attention(q, k, v, qo, ko)
    a, b = int(qo[0]), int(qo[-1])
    for x in (o[:a], o[b:]):
        assert not x.any()
    assert (lse[:a] == -INF).all() and (lse[b:] == -INF).all()
    dq, dk, dv = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, ko)
    ka, kb = int(ko[0]), int(ko[-1])
    for x, i, j in ((dq, a, b), (dk, ka, kb), (dv, ka, kb)):
        assert not x[:i].any() and not x[j:].any() and x.isfinite().all()
    # the sequences themselves, against the oracle on their tokens alone (another number of tokens
    # may take another split of the keys: not the same bits)
    q, do, o, lse, dq = (t[a:b] for t in (q, do, o, lse, dq))
    k, v, dk, dv = (t[ka:kb] for t in (k, v, dk, dv))
    want, wl, bo, bl = ref.forward(q, k, v, qo - a, ko - ka, 128 ** -0.5)
    ref.within("lse", lse, wl, bl)
    ref.within("o", o, want, bo)
    want, bounds = ref.backward(q, k, v, o, lse, do, qo - a, ko - ka, 128 ** -0.5)
    for x, y, z in zip((dq, dk, dv), want, bounds):
        ref.within("gradients", x, y, z)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ql", [[9, 50], [700, 900]])
def test_layouts_and_given_outputs(dev, dtype, ql):
    """[heads, T, d] inputs, and outputs that are parts of one buffer whose rest stays."""
    nq, nkv, d = 6, 2, 64
    q, k, v, do, qo, ko = problem(dev, dtype, d, nq, nkv, ql)
    o, lse, *grads = check(q, k, v, do, qo, ko)
    T = q.shape[0]
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]
    buf = torch.full((T, (nq + 2 * nkv) * d + 24), 7.0, dtype=dtype, device=dev)
    parts = [buf[:, a * d:b * d].view(T, b - a, d) for a, b in
             ((0, nq), (nq, nq + nkv), (nq + nkv, nq + 2 * nkv))]
    wide = torch.full((T, nq, d + 8), 7.0, dtype=dtype, device=dev)
    o2, lse2 = llmt.packed_attention(*turned[:3], qo, out=wide[..., :d])
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and (wide[..., d:] == 7).all()
    got = llmt.packed_attention_bwd(*turned[:3], o2, lse2, turned[3], qo, out=parts)
    for a, b in zip(got, grads):
        assert torch.equal(a, b)
    assert (buf[:, (nq + 2 * nkv) * d:] == 7).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scale_and_large_scores(dev, dtype):
    """Scores of hundreds: one key takes all; a scale of one's own."""
    q, k, v, do, qo, ko = problem(dev, dtype, 128, 4, 2, [90, 200])
    check(q, k, v, do, qo, ko, scale=0.3)
    o, lse = llmt.packed_attention(q * 8, k * 8, v, qo)
    s = (q.double() * 8)[-1, 0] @ (k.double() * 8)[90:, 0].t() * 128 ** -0.5
    assert abs(lse[-1, 0].item() - torch.logsumexp(s, 0).item()) < 1e-3
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ql", [[200], [3000]])
def test_scores_of_millions(dev, dtype, ql):
    """Scores up to 2^24: one key has all of a row's weight.  A row of q is the row of a key that it
    sees: their product is 2^23, those with the other keys (signs drawn apart) less than 2^22, and
    what fp32 leaves out of a score is below 2.  o is then v's row: off by one rounding of P and its
    own.  lse: five roundings and constants of 2^-24."""
    g = torch.Generator().manual_seed(1)
    T = ql[0]
    k = torch.where(torch.rand(T, 1, 128, generator=g) < 0.5, -1.0, 1.0) * 256
    pick = torch.tensor([int(torch.randint(0, t + 1, (1,), generator=g)) for t in range(T)])
    q = k[pick].repeat(1, 2, 1)
    v, do = torch.randn(T, 1, 128, generator=g), torch.randn(T, 2, 128, generator=g)
    q, k, v, do = (t.to(dtype).to(dev) for t in (q, k, v, do))
    off = offsets(ql).to(dev)
    o, lse = llmt.packed_attention(q, k, v, off, scale=1.9)
    want = v[pick.to(dev)].repeat(1, 2, 1).double()
    assert ((o.double() - want).abs() <= 2.02 * ref.unit(dtype) * want.abs()).all()
    assert torch.allclose(lse, torch.full_like(lse, 1.9 * 2 ** 23), rtol=2 ** -21, atol=0)
    dq, dk, dv = llmt.packed_attention_bwd(q, k, v, o, lse, do, off, scale=1.9)
    assert all(t.isfinite().all() for t in (dq, dk, dv))


@pytest.mark.parametrize("dtype,small", [(HF, 2.0 ** -13), (BF, 2.0 ** -60)])
@pytest.mark.parametrize("ql", [[300, 41], [1500, 900]])
def test_small_gradients_keep_their_bits(dev, dtype, small, ql):
    """dout times a power of two gives the same gradients times it: none of the intermediate
    products underflows.  (2^-13 of values near 1 are normal fp16 numbers; the outputs are compared
    where those of the small run are normal too.)"""
    q, k, v, do, qo, ko = problem(dev, dtype, 128, 16, 8, ql)
    do = do.clamp(-4, 4) + 0.5
    o, lse = llmt.packed_attention(q, k, v, qo)
    big = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo)
    low = llmt.packed_attention_bwd(q, k, v, o, lse, do * small, qo)
    exact = (do * small).double() == do.double() * small
    assert exact.all() or dtype == HF
    if exact.all():
        for a, b in zip(big, low):
            normal = b.double().abs() >= torch.finfo(dtype).tiny
            assert torch.equal(a.double()[normal] * small, b.double()[normal])


def test_running_twice_and_in_any_company_gives_the_same_bits(dev):
    q, k, v, do, qo, ko = problem(dev, BF, 128, 16, 8, [400, 33, 800])
    o, lse = llmt.packed_attention(q, k, v, qo)
    g = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo)
    o2, lse2 = llmt.packed_attention(q, k, v, qo)
    g2 = llmt.packed_attention_bwd(q, k, v, o2, lse2, do, qo)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    assert all(torch.equal(a, b) for a, b in zip(g, g2))


@pytest.mark.parametrize("ql,kl", [([30, 90], None), ([900, 1400], None), ([1, 1], [3000, 100])])
def test_captured_and_replayed(dev, ql, kl):
    q, k, v, do, qo, ko = problem(dev, BF, 128, 16, 8, ql, kl)
    def both():
        o, lse = llmt.packed_attention(q, k, v, qo, ko)
        return (o, lse, *llmt.packed_attention_bwd(q, k, v, o, lse, do, qo, ko))
    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        q.copy_(torch.randn_like(q))
        v.mul_(1.25)
        want = both()
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_on_another_stream(dev):
    q, k, v, do, qo, ko = problem(dev, HF, 64, 4, 2, [200, 31])
    o, lse, *g = check(q, k, v, do, qo, ko)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    o2, lse2 = llmt.packed_attention(q, k, v, qo, stream=s)
    g2 = llmt.packed_attention_bwd(q, k, v, o2, lse2, do, qo, stream=s)
    s.synchronize()
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(g, g2))


@pytest.mark.parametrize("off", [[0, 50, 30, 80], [-5, 40, 300, 60], [90, 10, 5, 2], [0, 80, 80, 2 ** 31 - 1]])
def test_malformed_offsets_stay_inside_the_arrays(dev, off):
    """Offsets that descend or leave the arrays: outputs are of no account, memory around them is
    untouched."""
    nq, nkv, d, T = 4, 2, 64, 80
    room = lambda n, dt=BF: torch.full((3 * T, n, d), 3.0, dtype=dt, device=dev)
    q, o, do, dq = (room(nq) for _ in range(4))
    k, v, dk, dv = (room(nkv) for _ in range(4))
    cut = lambda t: t[T:2 * T]
    bad = torch.tensor(off, dtype=torch.int32, device=dev)
    good = torch.tensor([0, 20, 60, 80], dtype=torch.int32, device=dev)
    for qo, ko in ((bad, good), (good, bad), (bad, bad)):
        _, lse = llmt.packed_attention(cut(q), cut(k), cut(v), qo, ko, out=cut(o))
        llmt.packed_attention_bwd(cut(q), cut(k), cut(v), cut(o), lse, cut(do), qo, ko,
                                  out=(cut(dq), cut(dk), cut(dv)))
        torch.cuda.synchronize()
        for t in (o, dq, dk, dv):
            assert (t[:T] == 3).all() and (t[2 * T:] == 3).all()


def test_gradients_against_differences(dev):
    """Central differences of sum(o dout) in float64 on a small problem, through the kernel's own
    gradients (bf16: 2^-8 a factor, so a direction's derivative to about 1%)."""
    q, k, v, do, qo, ko = problem(dev, HF, 64, 2, 1, [12, 20])
    o, lse = llmt.packed_attention(q, k, v, qo)
    grads = llmt.packed_attention_bwd(q, k, v, o, lse, do, qo)
    g = torch.Generator().manual_seed(3)
    for i, (t, grad) in enumerate(zip((q, k, v), grads)):
        way = torch.randn(t.shape, generator=g).double().to(dev)
        f = []
        for h in (1e-4, -1e-4):
            x = [y.double() for y in (q, k, v)]
            x[i] = x[i] + h * way
            f.append(float((ref.forward64(*x, qo, ko, 0.125) * do.double()).sum()))
        slope = (f[0] - f[1]) / 2e-4
        got = float((grad.double() * way).sum())
        # fp16 roundings of P, dS and the result: about 2^-10 of the sum of magnitudes' root
        room = 2 ** -9 * float((grad.double() * way).abs().sum()) / 8
        assert abs(got - slope) <= room, (i, got, slope, room)


def test_no_tokens(dev):
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    e = torch.empty(0, 2, 64, dtype=BF, device=dev)
    o, lse = llmt.packed_attention(e, e, e, off)
    assert o.shape == e.shape and lse.shape == (0, 2)
    k = torch.ones(5, 2, 64, dtype=BF, device=dev)
    ko = torch.tensor([0, 2, 5], dtype=torch.int32, device=dev)
    dq, dk, dv = llmt.packed_attention_bwd(e, k, k, e, lse, e, off, ko)
    assert not dk.any() and not dv.any()
    o, lse = llmt.packed_attention(k, e, e, ko, off)
    assert not o.any() and (lse == -INF).all()
    dq, dk, dv = llmt.packed_attention_bwd(k, e, e, o, lse, k, ko, off)
    assert not dq.any()
