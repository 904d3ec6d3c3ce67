"""GPU: the preference loss and the clipped policy loss against float64 on the CPU.

The kernels compute in fp64 and round each output once to fp32 (half a step, 2^-24 of
itself); the mean preference loss is a mean of rounded losses, one more half step.  The
reference sums in another order: 1e-12 of the terms' size."""
import math

import pytest
import torch
import torch.nn.functional as F

import llmt

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def close(got, want, size=1.0, steps=1):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    assert ((got - want).abs() <= steps * U * want.abs() + 1e-12 * size + 2.0 ** -126).all(), \
        float((got - want).abs().max())


def ragged(g, count, S, gap=(0, 0), empty=()):
    n = torch.randint(1, S + 1, (count,), generator=g)
    for i in empty:
        n[i % count] = 0
    off = torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]) + gap[0]
    return off.to(torch.int32), int(off[-1]) + gap[1]


def pref64(lp, ref, off, mask, kind, beta, smooth, margin, average):
    """losses, rewards by the definition, a Python loop over the sequences (autograd tensors)."""
    r = []
    for s in range(len(off) - 1):
        sl = slice(int(off[s]), int(off[s + 1]))
        k = mask[sl]
        d = (lp[sl] - ref[sl])[k]
        v = d.sum()
        r.append(f32(beta) * (v / max(1, int(k.sum())) if average else v))
    r = torch.stack(r)
    z = r[0::2] - r[1::2] - f32(margin)
    f = {"sigmoid": lambda v: F.softplus(-v, threshold=1e9), "hinge": lambda v: F.relu(1 - v),
         "square": lambda v: (v - 0.5) ** 2}[kind]
    e = f32(smooth)
    return (1 - e) * f(z) + e * f(-z), r


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
@pytest.mark.parametrize("n,S,average,smooth,use_ref,use_mask", [
    (1, 1, False, 0.0, True, False), (1, 5000, True, 0.1, True, True), (2, 40000, False, 0.0, True, True),
    (5, 3, True, 0.0, False, True), (40, 77, False, 0.2, True, True), (300, 200, True, 0.0, True, False),
    (2500, 9, False, 0.0, False, True)])
def test_preference_loss(dev, kind, n, S, average, smooth, use_ref, use_mask):
    g = torch.Generator().manual_seed(n * 31 + S)
    gap = (0, 0) if n % 2 else (5, 37)
    off, T = ragged(g, 2 * n, S, gap, empty=() if n < 5 else (1, 4, 9))
    lp = -torch.rand(T, generator=g) * 3
    ref = lp + 0.1 * torch.randn(T, generator=g) if use_ref else torch.zeros(T)
    mask = torch.rand(T, generator=g) < 0.7 if use_mask else torch.ones(T, dtype=torch.bool)
    if n >= 5 and use_mask:
        mask[int(off[6]):int(off[7])] = False          # a sequence without any kept token
    beta, margin = 0.3 if average else 0.05, 0.2
    x = lp.double().requires_grad_()
    losses, r = pref64(x, ref.double(), off, mask, kind, beta, smooth, margin, average)
    losses.mean().backward()
    junk = lp.clone()
    junk[~mask] = math.nan                             # left out: not read
    junk[:gap[0]] = math.nan
    junk[T - gap[1]:] = math.inf
    mean, got, rew, d = llmt.preference_loss(
        junk.to(dev), ref.to(dev) if use_ref else None, off.to(dev), loss=kind, beta=beta,
        label_smoothing=smooth, margin=margin, average=average,
        mask=mask.to(dev))
    close(got, losses.detach(), size=S)
    close(rew, r.detach(), size=S)
    close(mean, losses.detach().mean().reshape(1), size=S, steps=2)
    close(d, x.grad)
    outside = torch.ones(T, dtype=torch.bool)
    outside[int(off[0]):int(off[-1])] = False
    assert (d.cpu()[outside] == 0).all() and (d.cpu()[~mask] == 0).all()
    if not use_mask:
        again = llmt.preference_loss(lp.to(dev), ref.to(dev) if use_ref else None, off.to(dev),
                                     loss=kind, beta=beta, label_smoothing=smooth, margin=margin,
                                     average=average, want_grad=False)
        assert torch.equal(again[1], got) and torch.equal(again[0], mean) and again[3] is None


def test_preference_gradient_against_differences(dev):
    """Central differences of the mean loss: values rounded to 2^-24, steps of 2^-5, so a
    difference is off by 2^-24 / 2^-5 = 2^-19 and h^2 / 6 times the third derivative."""
    g = torch.Generator().manual_seed(5)
    off, T = ragged(g, 6, 4)
    lp, ref = -torch.rand(T, generator=g).to(dev), -torch.rand(T, generator=g).to(dev)
    call = lambda x: llmt.preference_loss(x, ref, off.to(dev), beta=0.5)
    d = call(lp)[3]
    for t in range(T):
        e = torch.zeros(T, device=dev)
        e[t] = 2.0 ** -5
        diff = (float(call(lp + e)[0]) - float(call(lp - e)[0])) / 2.0 ** -4
        assert abs(diff - float(d[t])) <= 2.0 ** -18 + 1e-4 * 0.5 ** 3


def test_preference_extremes(dev):
    """Differences far beyond exp's range, and a log-probability of -inf."""
    off = torch.tensor([0, 1, 2, 3, 4, 5, 6], dtype=torch.int32, device=dev)
    lp = torch.tensor([1e6, 0.0, 0.0, 1e6, -math.inf, 0.0], device=dev)
    mean, losses, r, d = llmt.preference_loss(lp, None, off, beta=1.0)
    assert losses.tolist() == [0.0, 1e6, math.inf] and mean.item() == math.inf
    close(d, torch.tensor([0.0, 0.0, -1 / 3, 1 / 3, -1 / 3, 1 / 3], dtype=torch.float64))


def test_offsets_out_of_range_stay_in_the_arrays(dev):
    """Offsets beyond T or below 0 are clamped (the arrays' own memory, guarded on both
    sides, is all that is touched)."""
    T = 50
    lp, adv = torch.zeros(T, device=dev), torch.ones(T, device=dev)
    off = torch.tensor([-7, 20, 10 ** 9, 2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    mean, losses, r, d = llmt.preference_loss(lp, None, off, beta=1.0)
    close(losses, torch.full((2,), math.log(2.0), dtype=torch.float64))
    p = llmt.policy_loss(lp, None, adv, off)
    assert p.loss.item() == -1.0 and (p.dlogp == -f32(1 / T)).all()


def policy64(lp, old, ref, adv, ent, off, mask, mean, low, high, kl, ec):
    n, T = len(off) - 1, len(lp)
    lens = (off[1:] - off[:-1]).long()
    seq = torch.full((T,), -1)
    seq[int(off[0]):int(off[-1])] = torch.repeat_interleave(torch.arange(n), lens)
    inside = (seq >= 0) & mask
    s = seq.clamp(min=0)
    if mean == "token":
        w = inside.double() / max(1, int(inside.sum()))
    else:
        kept = torch.zeros(n, dtype=torch.double).index_add(0, s, inside.double())
        w = inside.double() / (kept.clamp(min=1)[s] * n)
    A = adv.double()[s] if adv.shape[0] == n and adv.shape[0] != T else adv.double()
    ratio = (lp - old).exp()
    lo, hi = 1 - f32(low), 1 + f32(high)
    s1, s2 = ratio * A, ratio.clamp(lo, hi) * A
    pg = -torch.minimum(s1, s2)
    d = ref - lp
    k = torch.expm1(d) - d
    l = pg + f32(kl) * k - f32(ec) * ent
    return (l * w).sum(), torch.stack([(pg * w).sum(), (k * w).sum(), ((s1 > s2) * w).sum()])


@pytest.mark.parametrize("mean", ["token", "sequence"])
@pytest.mark.parametrize("n,S,per_seq,use_old,use_ref,use_ent,use_mask", [
    (1, 1, False, True, True, True, False), (1, 30000, True, True, True, False, True),
    (3, 2, False, False, True, True, True), (8, 200, True, True, True, False, True),
    (60, 700, False, True, False, True, True), (700, 90, True, True, True, True, False),
    (3000, 5, False, True, True, False, True)])
def test_policy_loss(dev, n, S, per_seq, use_old, use_ref, use_ent, use_mask, mean):
    g = torch.Generator().manual_seed(n * 17 + S)
    gap = (3, 1500) if n in (8, 60) else (0, 0)
    off, T = ragged(g, n, S, gap, empty=() if n < 8 else (2, 7))
    lp = -torch.rand(T, generator=g) * 3
    old = lp + 0.3 * torch.randn(T, generator=g)
    ref = lp + 0.3 * torch.randn(T, generator=g)
    adv = torch.randn(n if per_seq else T, generator=g)
    ent = torch.rand(T, generator=g)
    mask = torch.rand(T, generator=g) < 0.7 if use_mask else torch.ones(T, dtype=torch.bool)
    if n >= 8 and use_mask:
        mask[int(off[4]):int(off[5])] = False
    kl, ec = 0.05, 0.02
    x, e = lp.double().requires_grad_(), ent.double().requires_grad_()
    want, stats = policy64(x, old.double() if use_old else x.detach(),
                           ref.double() if use_ref else x.detach(), adv, e if use_ent else 0 * e,
                           off, mask, mean, 0.2, 0.28, kl if use_ref else 0.0, ec)
    want.backward()
    bad = lambda v: torch.where(mask, v, torch.full_like(v, math.nan)).to(dev)
    p = llmt.policy_loss(bad(lp), bad(old) if use_old else None,
                         adv.to(dev) if per_seq else bad(adv), off.to(dev),
                         ref_logp=bad(ref) if use_ref else None,
                         entropy=bad(ent) if use_ent else None,
                         mask=mask.to(dev) if use_mask else None, clip_low=0.2, clip_high=0.28,
                         kl_coef=kl, entropy_coef=ec, mean=mean, per_sequence=per_seq)
    close(p.loss, want.detach().reshape(1))
    close(p.stats, stats.detach())
    close(p.dlogp, x.grad)
    if use_ent:
        close(p.dentropy, e.grad)
    else:
        assert p.dentropy is None


@pytest.mark.parametrize("n,S", [(120, 1000), (140, 2000)])
def test_policy_loss_of_many_masked_tokens(dev, n, S):
    """About 60000 and 140000 tokens: the kept ones are counted by every workgroup, and by
    a launch of their own."""
    test_policy_loss(dev, n, S, False, True, True, True, True, "token")


def test_policy_gradient_against_differences(dev):
    """As for the preference loss: 2^-24 rounded values over steps of 2^-6 (away from the
    clip borders, where the loss has a corner)."""
    g = torch.Generator().manual_seed(9)
    T = 12
    off = torch.tensor([0, 5, 5, 12], dtype=torch.int32, device=dev)
    lp = -torch.rand(T, generator=g).to(dev)
    old = lp + torch.tensor([-0.5, 0.05, 0.5, 0.0], device=dev).repeat(3)
    ref = lp + torch.randn(T, generator=g).to(dev)
    adv = torch.randn(T, generator=g).to(dev)
    for mean in ("token", "sequence"):
        call = lambda x: llmt.policy_loss(x, old, adv, off, ref_logp=ref, kl_coef=0.5, mean=mean)
        d = call(lp).dlogp
        for t in range(T):
            e = torch.zeros(T, device=dev)
            e[t] = 2.0 ** -6
            diff = (float(call(lp + e).loss) - float(call(lp - e).loss)) / 2.0 ** -5
            assert abs(diff - float(d[t])) <= 2.0 ** -16 + 2.0 ** -12 / 6 * 4, t


def test_policy_nothing_kept(dev):
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device=dev)
    x = torch.full((8,), math.nan, device=dev)
    for mean in ("token", "sequence"):
        p = llmt.policy_loss(x, x, x, off, ref_logp=x, entropy=x, mean=mean,
                             mask=torch.zeros(8, dtype=torch.bool, device=dev))
        assert p.loss.item() == 0 and (p.stats == 0).all()
        assert (p.dlogp == 0).all() and (p.dentropy == 0).all()


def test_no_tokens(dev):
    e = torch.empty(0, device=dev)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    mean, losses, r, d = llmt.preference_loss(e, e, off)
    close(mean, torch.tensor([math.log(2.0)], dtype=torch.float64))
    p = llmt.policy_loss(e, e, e, off)
    assert p.loss.item() == 0 and p.dlogp.shape == (0,)


def test_losses_repeat_in_a_graph_and_on_a_side_stream(dev):
    g = torch.Generator().manual_seed(2)
    off, T = ragged(g, 60, 900)
    lp, old = -torch.rand(T, generator=g).to(dev), -torch.rand(T, generator=g).to(dev)
    mask = (torch.rand(T, generator=g) < 0.5).to(dev)
    off = off.to(dev)

    def both(stream=None):
        return (*llmt.preference_loss(lp, old, off, mask=mask, stream=stream),
                *llmt.policy_loss(lp, old, old, off, ref_logp=old, entropy=old, mask=mask,
                                  kl_coef=0.1, entropy_coef=0.1, stream=stream))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):                    # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    for _ in range(3):
        lp.mul_(0.9)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = both()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_the_binding_refuses_wrong_types_and_shapes(dev):
    x, t = torch.zeros(4, 8, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    off, v = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev), torch.zeros(4, device=dev)
    st = torch.zeros(4, 2, device=dev)
    for call in (lambda: llmt.token_logprobs(x.double(), t),
                 lambda: llmt.token_logprobs(x, t, temperature=0.0),
                 lambda: llmt.token_logprobs(x, t, temperature=-1.0),
                 lambda: llmt.token_logprobs(x, t, temperature=float("nan")),
                 lambda: llmt.token_logprobs(x.t(), t),
                 lambda: llmt.token_logprobs(x, t.long()),
                 lambda: llmt.token_logprobs(x, t[:3]),
                 lambda: llmt.token_logprobs(x[:, :4], t.cpu()),
                 lambda: llmt.token_logprobs_bwd(x, t, st[:, :1], v),
                 lambda: llmt.token_logprobs_bwd(x, t, st, v.double()),
                 lambda: llmt.token_logprobs_bwd(x, t, st, v, out=x.half()),
                 lambda: llmt.token_logprobs_bwd(x, t, st, v, out=x[:3]),
                 lambda: llmt.token_logprobs_bwd(x, t, st, v, dentropy=v),
                 lambda: llmt.preference_loss(v, None, off[:2]),
                 lambda: llmt.preference_loss(v.half(), None, off),
                 lambda: llmt.preference_loss(v, v[:3], off),
                 lambda: llmt.preference_loss(v, None, off.long()),
                 lambda: llmt.preference_loss(v, None, off, mask=v),
                 lambda: llmt.preference_loss(x[:, 0], None, off),
                 lambda: llmt.policy_loss(v, v, v, off[:1]),
                 lambda: llmt.policy_loss(v, v, v[:2], off),
                 lambda: llmt.policy_loss(v, v, v, off, per_sequence=True),
                 lambda: llmt.policy_loss(v, v, v, off, mask=t)):
        with pytest.raises(llmt.LlmtError):
            call()


def test_two_streams_at_once(dev):
    """Calls that run beside one another on two streams share nothing."""
    g = torch.Generator().manual_seed(13)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    data = []
    for k in range(2):
        off, T = ragged(g, 40, 700)
        data.append(dict(off=off.to(dev), lp=-torch.rand(T, generator=g).to(dev),
                         old=-torch.rand(T, generator=g).to(dev),
                         mask=(torch.rand(T, generator=g) < 0.5).to(dev),
                         x=torch.randn(5, 60000, generator=g).to(dev),
                         t=torch.randint(0, 60000, (5,), generator=g, dtype=torch.int32).to(dev),
                         u=torch.randn(3, 30, 500, generator=g).to(dev)))

    def all_of(d, stream):
        p = llmt.policy_loss(d["lp"], d["old"], d["old"], d["off"], ref_logp=d["old"],
                             mask=d["mask"], kl_coef=0.1, stream=stream)
        q = llmt.preference_loss(d["lp"], d["old"], d["off"], mask=d["mask"], stream=stream)
        lp, st, _ = llmt.token_logprobs(d["x"], d["t"], stream=stream)
        return (p.loss, p.stats, p.dlogp, *q, lp, st,
                llmt.token_logprobs_bwd(d["x"], d["t"], st, lp, stream=stream),
                llmt.orthogonalize(d["u"], stream=stream))

    want = [all_of(d, None) for d in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            got[k].append(all_of(data[k], sides[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
